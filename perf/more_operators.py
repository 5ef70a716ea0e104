"""Cases and plain forms of the serving-attention operators: rotary positions, the paged cache, single-token attention.

Four entry points are measured:

* ``rotary_fwd``  RotaryEmbeddingFwdOp: queries and keys rotated by their positions;
* ``rotary_bwd``  RotaryEmbeddingBwdOp: its gradients;
* ``append``      PagedKVAppendOp: new keys (rotated) and values into a paged cache, the queries rotated beside them;
* ``attend``      PagedAttentionDecodeOp: one new token of every sequence over the paged cache.

``run`` computes them in elementary torch operations where ``own`` is false and through the package where it is true;
``exact`` computes them in 64 bits by another route (complex numbers, sequence after sequence).
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BASE = 10000.0
# The scaled frequencies: pairs that turn less than SLOW times over ORIGINAL tokens are slowed down by FACTOR, those of
# more than FAST turns stay, a ramp between.
FACTOR, ORIGINAL, SLOW, FAST = 8.0, 8192, 1.0, 32.0


def listed():
    return [
        # One token of one user over a short conversation: launch latency.
        {"name": "attend one short", "op": "attend", "batch": 1, "max_len": 1000, "lens": "full", "heads": 32,
         "heads_kv": 8, "dim": 128, "page_size": 16, "window": 0, "layout": "token", "dtype": "bfloat16"},
        # One token of one user over a long document: few rows, the cache's length has to be split.
        {"name": "attend one long", "op": "attend", "batch": 1, "max_len": 131072, "lens": "full", "heads": 32,
         "heads_kv": 8, "dim": 128, "page_size": 64, "window": 0, "layout": "token", "dtype": "bfloat16"},
        # A serving batch of conversations of all lengths, some slots idle.
        {"name": "attend batch ragged", "op": "attend", "batch": 64, "max_len": 8192, "lens": "ragged", "heads": 32,
         "heads_kv": 8, "dim": 128, "page_size": 16, "window": 0, "layout": "token", "dtype": "bfloat16"},
        # The attention benchmark's heads (as many key heads as query heads), pages laid out head by head.
        {"name": "attend mha f16", "op": "attend", "batch": 8, "max_len": 4096, "lens": "ragged", "heads": 32,
         "heads_kv": 32, "dim": 128, "page_size": 32, "window": 0, "layout": "head", "dtype": "float16"},
        # Odd everything: six query heads a key head, 80 channels, pages of seven tokens, a sliding window.
        {"name": "attend odd window f16", "op": "attend", "batch": 37, "max_len": 5000, "lens": "ragged", "heads": 12,
         "heads_kv": 2, "dim": 80, "page_size": 7, "window": 1000, "layout": "head", "dtype": "float16"},
        # The step before the first of these: one token of one user into the cache.
        {"name": "append step one", "op": "append", "batch": 1, "tokens": 1, "packed": False, "max_len": 1000,
         "heads": 32, "heads_kv": 8, "dim": 128, "rotary_dim": 128, "interleaved": False, "scaled": False,
         "page_size": 16, "layout": "token", "dtype": "bfloat16"},
        # One token of every sequence of a large serving batch.
        {"name": "append step batch", "op": "append", "batch": 256, "tokens": 1, "packed": False, "max_len": 8192,
         "heads": 32, "heads_kv": 8, "dim": 128, "rotary_dim": 128, "interleaved": False, "scaled": True,
         "page_size": 16, "layout": "token", "dtype": "bfloat16"},
        # Prompts of many lengths packed on one axis, behind prefixes that are in the cache already.
        {"name": "append prefill packed", "op": "append", "batch": 9, "tokens": 16384, "packed": True, "max_len": 8192,
         "heads": 32, "heads_kv": 8, "dim": 128, "rotary_dim": 64, "interleaved": True, "scaled": False,
         "page_size": 64, "layout": "head", "dtype": "float16"},
        # A training step's queries and keys, at the attention benchmark's tokens and heads.
        {"name": "rotary train", "op": "rotary_fwd", "batch": 8, "seq_len": 4096, "heads": 32, "heads_kv": 32,
         "dim": 128, "rotary_dim": 128, "interleaved": False, "scaled": False, "positions": "none", "sliced": False,
         "dtype": "bfloat16"},
        # A short prompt at far positions; q and k are column slices of one projection's output; full precision.
        {"name": "rotary odd far f32", "op": "rotary_fwd", "batch": 3, "seq_len": 1001, "heads": 5, "heads_kv": 1,
         "dim": 72, "rotary_dim": 36, "interleaved": True, "scaled": True, "positions": "batch", "sliced": True,
         "dtype": "float32"},
        # The backward pass of a training step with few key heads.
        {"name": "rotary bwd train", "op": "rotary_bwd", "batch": 8, "seq_len": 4096, "heads": 32, "heads_kv": 8,
         "dim": 128, "rotary_dim": 128, "interleaved": False, "scaled": True, "positions": "row", "sliced": False,
         "dtype": "bfloat16"},
        # The same of a small model with part of the head rotated, in half precision.
        {"name": "rotary bwd part f16", "op": "rotary_bwd", "batch": 2, "seq_len": 777, "heads": 12, "heads_kv": 12,
         "dim": 64, "rotary_dim": 24, "interleaved": False, "scaled": False, "positions": "none", "sliced": True,
         "dtype": "float16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rotation(rng, dim):
    """Of a head: all of it, half of it, or any even part."""
    part = rng.choice([dim, dim, dim // 2 // 2 * 2, 2 * rng.randint(1, dim // 2)])
    return {"rotary_dim": max(2, part), "interleaved": rng.random() < 0.4, "scaled": rng.random() < 0.4}


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "rotary_fwd", "rotary_bwd"])
    heads_kv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    heads = heads_kv * rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16, 24) if heads_kv * g <= 64])
    dim = rng.choice([64, 128, 128, 128, 80, 96, 192, 256, 40])
    case = {"op": op, "heads": heads, "heads_kv": heads_kv, "dim": dim}
    if op.startswith("rotary"):
        if rng.random() < 0.2:
            case["dim"] = dim = 2 * rng.randint(8, 100)
        batch = _log_int(rng, 1, 16)
        most = max(1, (1 << 27) // (batch * (heads + heads_kv) * dim))
        case.update(batch=batch, seq_len=_log_int(rng, 1, min(32768, most)), **_rotation(rng, dim),
                    positions=rng.choice(["none", "row", "batch"]), sliced=rng.random() < 0.4,
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
        return case
    case.update(page_size=rng.choice([16, 16, 32, 64, 128, 256, 7, 1]), layout=rng.choice(["token", "token", "head"]))
    if op == "append":
        batch = _log_int(rng, 1, 256)
        packed = rng.random() < 0.5
        most = (1 << 27) // ((heads + 2 * heads_kv) * dim)
        tokens = _log_int(rng, batch, min(16384, most)) if packed else _log_int(rng, 1, max(1, min(2048, most // batch)))
        case.update(batch=batch, tokens=tokens, packed=packed, max_len=_log_int(rng, 2048, 65536), **_rotation(rng, dim),
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
        return case
    batch = _log_int(rng, 1, 256)
    most = max(1, (1 << 28) // (batch * heads_kv * dim))
    case.update(batch=batch, max_len=_log_int(rng, 1, min(131072, most)), lens=rng.choice(["full", "ragged", "ragged"]),
                window=rng.choice([0, 0, 0, _log_int(rng, 1, 8192)]), dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    return case


def _lengths(case):
    """The sequences' lengths, of the case alone: all at the longest, or spread over the logarithm with idle slots."""
    B, L = case["batch"], case["max_len"]
    if case.get("lens", "ragged") == "full":
        return [L] * B
    rng = random.Random(1000003 * B + L)
    return [0 if rng.random() < 0.05 else _log_int(rng, max(1, L // 64), L) for _ in range(B)]


def _new_tokens(case):
    """How many tokens each sequence of an append brings, and its length after it."""
    B, T, L = case["batch"], case["tokens"], case["max_len"]
    rng = random.Random(1000003 * B + T)
    if case["packed"]:
        cuts = sorted(rng.randint(0, T) for _ in range(B - 1))
        new = [b - a for a, b in zip([0, *cuts], [*cuts, T])]
    else:
        new = [T] * B
    return new, [n + rng.randint(0, L) for n in new]


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    H, Hkv, D = case["heads"], case["heads_kv"], case["dim"]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    state = {"case": dict(case)}
    if case["op"].startswith("rotary"):
        B, S = case["batch"], case["seq_len"]
        if case["sliced"]:
            both = randn(B, S, (H + 2 * Hkv) * D)
            state["q"] = both[..., : H * D].view(B, S, H, D)
            state["k"] = both[..., H * D : (H + Hkv) * D].view(B, S, Hkv, D)
        else:
            state["q"], state["k"] = randn(B, S, H, D), randn(B, S, Hkv, D)
        at = torch.arange(S, device="cuda", dtype=torch.int32)
        state["positions"] = None
        if case["positions"] == "row":
            state["positions"] = at + 4096
        elif case["positions"] == "batch":
            state["positions"] = at + torch.randint(0, 1 << 20, (B, 1), generator=g, device="cuda", dtype=torch.int32)
        return state

    B, P = case["batch"], case["page_size"]
    if case["op"] == "append":
        new, lens = _new_tokens(case)
        first = [(n_all - n) // P for n, n_all in zip(new, lens)]  # pages before it are a prefix that all share
    else:
        lens, first = _lengths(case), [0] * B
    width = max(1, max(-(-n // P) for n in lens))
    lens_t = torch.tensor(lens, device="cuda", dtype=torch.int32)
    first_t = torch.tensor(first, device="cuda")
    column = torch.arange(width, device="cuda")
    has = (column < (lens_t[:, None] + P - 1) // P) & (column >= first_t[:, None])
    pages = int(sum(-(-n // P) - f for n, f in zip(lens, first))) + 1  # page 0 is the shared prefix, or no one's
    order = 1 + torch.randperm(pages - 1, generator=g, device="cuda")
    table = torch.zeros(B, width, device="cuda", dtype=torch.int32)
    table[has] = order.to(torch.int32)
    table[column >= (lens_t[:, None] + P - 1) // P] = -1  # behind the sequence's end
    state["page_table"], state["seq_lens"] = table, lens_t
    shape = (pages, P, Hkv, D) if case["layout"] == "token" else (pages, Hkv, P, D)
    for name in ("k_cache", "v_cache"):
        cache = randn(*shape)
        state[name] = cache if case["layout"] == "token" else cache.transpose(1, 2)
    if case["op"] == "attend":
        state["q"] = randn(B, H, D, scale=2.0)
        return state
    T = case["tokens"]
    rows = (T,) if case["packed"] else (B,) if T == 1 else (B, T)
    state["q"], state["k"], state["v"] = randn(*rows, H, D), randn(*rows, Hkv, D), randn(*rows, Hkv, D)
    state["cu_seqlens"] = None
    if case["packed"]:
        state["cu_seqlens"] = torch.tensor([0, *new], device="cuda").cumsum(0).to(torch.int32)
    return state


# ------------------------------------------------------- plain forms, 32 bits
def _frequencies(case):
    """Angles a token of the pairs, in 64 bits, and the factor on the rotated channels."""
    r = case["rotary_dim"]
    f = BASE ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if not case["scaled"]:
        return f, 1.0
    turns = ORIGINAL * f / (2.0 * math.pi)
    keep = ((turns - SLOW) / (FAST - SLOW)).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / FACTOR), 1.0 + 0.1 * math.log(FACTOR)


def _plain_rotate(x, positions, case, back=False):
    """x (..., heads, dim) at positions (...)."""
    f, amplitude = _frequencies(case)
    angle = positions.double()[..., None, None] * f
    c, s = (amplitude * torch.cos(angle)).float(), (amplitude * torch.sin(angle)).float()
    if back:
        s = -s
    r, wide = case["rotary_dim"], x.float()
    if case["interleaved"]:
        a, b = wide[..., 0:r:2], wide[..., 1:r:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    else:
        a, b = wide[..., : r // 2], wide[..., r // 2 : r]
        turned = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    return torch.cat([turned, wide[..., r:]], dim=-1).to(x.dtype)


def _plain_rotary(st):
    c = st["case"]
    positions = st["positions"]
    if positions is None:
        positions = torch.arange(c["seq_len"], device="cuda")
    back = c["op"] == "rotary_bwd"
    return tuple(_plain_rotate(st[n], positions, c, back) for n in ("q", "k"))


def _plain_append(st):
    c, lens = st["case"], st["seq_lens"].long()
    P = c["page_size"]
    if c["packed"]:
        cu = st["cu_seqlens"].long()
        t = torch.arange(c["tokens"], device="cuda")
        seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
        positions = lens[seq] - cu[seq + 1] + t
    else:
        seq = torch.arange(c["batch"], device="cuda")
        positions = lens - 1
        if c["tokens"] > 1:
            seq = seq[:, None]
            positions = lens[:, None] - c["tokens"] + torch.arange(c["tokens"], device="cuda")
    page, slot = st["page_table"][seq, positions // P].long(), positions % P
    st["k_cache"][page, slot] = _plain_rotate(st["k"], positions, c)
    st["v_cache"][page, slot] = st["v"]
    return _plain_rotate(st["q"], positions, c), st["k_cache"], st["v_cache"]


def _plain_attend(st):
    c, lens = st["case"], st["seq_lens"]
    B, H, Hkv, D, P = c["batch"], c["heads"], c["heads_kv"], c["dim"], c["page_size"]
    table = st["page_table"].clamp(min=0).long()
    L = table.shape[1] * P
    keys = st["k_cache"][table].reshape(B, L, Hkv, D).permute(0, 2, 3, 1).float()
    q = st["q"].float().view(B, Hkv, H // Hkv, D)
    s = torch.matmul(q, keys) * (D**-0.5 * math.log2(math.e))
    del keys
    j = torch.arange(L, device="cuda")
    seen = j < lens[:, None]
    if c["window"]:
        seen = seen & (j >= lens[:, None] - c["window"])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp2(s - m)
    total = p.sum(dim=-1, keepdim=True)
    values = st["v_cache"][table].reshape(B, L, Hkv, D).transpose(1, 2).float()
    o = torch.matmul(p, values) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log2(total)).view(B, H)
    return o.view(B, H, D).to(st["q"].dtype), lse


# ------------------------------------------------------------ one pass
def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tile-ascendnpu-ops_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import tileops.ops.attention as attention
    return attention


def _own_op(st):
    """The op object of a case, built on its first pass and kept, as a program keeps it."""
    if "op" not in st:
        att, c, dt = _package(), st["case"], st["q"].dtype
        heads = {"heads": c["heads"], "heads_kv": c["heads_kv"], "dim": c["dim"], "dtype": dt}
        if c["op"] == "attend":
            st["op"] = att.PagedAttentionDecodeOp(page_size=c["page_size"], window=c["window"] or None, **heads)
            return st["op"]
        turn = {"rotary_dim": c["rotary_dim"], "interleaved": c["interleaved"]}
        if c["scaled"]:
            turn["frequencies"] = att.rotary_frequencies(c["rotary_dim"], BASE, factor=FACTOR, original_length=ORIGINAL,
                                                         slow_turns=SLOW, fast_turns=FAST)
            turn["amplitude"] = 1.0 + 0.1 * math.log(FACTOR)
        if c["op"] == "append":
            st["op"] = att.PagedKVAppendOp(page_size=c["page_size"], **heads, **turn)
        else:
            op = att.RotaryEmbeddingFwdOp if c["op"] == "rotary_fwd" else att.RotaryEmbeddingBwdOp
            st["op"] = op(batch=c["batch"], seq_len=c["seq_len"], **heads, **turn)
    return st["op"]


def run(state):
    st, op = state, state["case"]["op"]
    if own:
        call = _own_op(st)
        if op == "attend":
            return call(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["seq_lens"])
        if op == "append":
            q = call(st["k"], st["v"], st["k_cache"], st["v_cache"], st["page_table"], st["seq_lens"], st["q"],
                     st["cu_seqlens"])
            return q, st["k_cache"], st["v_cache"]
        return call(st["q"], st["k"], st["positions"])
    if op == "attend":
        return _plain_attend(st)
    if op == "append":
        return _plain_append(st)
    return _plain_rotary(st)


def work(case):
    eb, H, Hkv, D = DTYPES[case["dtype"]].itemsize, case["heads"], case["heads_kv"], case["dim"]
    if case["op"].startswith("rotary"):
        tokens = case["batch"] * case["seq_len"]
        told = {"none": 0, "row": case["seq_len"], "batch": tokens}[case["positions"]]
        return {"bytes": 2 * tokens * (H + Hkv) * D * eb + 4 * told,
                "flops": 3 * tokens * (H + Hkv) * case["rotary_dim"]}
    B, P = case["batch"], case["page_size"]
    if case["op"] == "append":
        tokens = case["tokens"] * (1 if case["packed"] else B)
        return {"bytes": 2 * tokens * (H + 2 * Hkv) * D * eb + 4 * B + 4 * tokens // P,
                "flops": 3 * tokens * (H + Hkv) * case["rotary_dim"]}
    seen = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
    return {"bytes": 2 * seen * Hkv * D * eb + 2 * B * H * D * eb + 4 * B * H + 4 * B + 4 * seen // P,
            "flops": max(1, 4 * seen * H * D)}


# ------------------------------------------------- 64 bits, by another route
def _exact_turns(case):
    """Angles a token, pair by pair."""
    r, out = case["rotary_dim"], []
    for i in range(r // 2):
        f = math.exp(-2.0 * i / r * math.log(BASE))
        if case["scaled"]:
            turns = ORIGINAL * f / math.tau
            keep = min(1.0, max(0.0, (turns - SLOW) / (FAST - SLOW)))
            f = f * keep + f / FACTOR * (1.0 - keep)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _exact_rotate(x, positions, case, sign=1.0):
    r, wide = case["rotary_dim"], x.double().contiguous()
    size = torch.tensor(1.0 + (0.1 * math.log(FACTOR) if case["scaled"] else 0.0), dtype=torch.float64, device="cuda")
    turn = torch.polar(size, sign * positions.double()[..., None] * _exact_turns(case))[..., None, :]
    out = wide.clone()
    if case["interleaved"]:
        pairs = torch.view_as_complex(wide[..., :r].unflatten(-1, (r // 2, 2)).contiguous())
        out[..., :r] = torch.view_as_real(pairs * turn).flatten(-2)
    else:
        pairs = torch.complex(wide[..., : r // 2].contiguous(), wide[..., r // 2 : r].contiguous()) * turn
        out[..., : r // 2], out[..., r // 2 : r] = pairs.real, pairs.imag
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"].startswith("rotary"):
        positions = st["positions"]
        if positions is None:
            positions = torch.arange(case["seq_len"], device="cuda")
        sign = 1.0 if case["op"] == "rotary_fwd" else -1.0
        return tuple(_exact_rotate(st[n], positions, case, sign) for n in ("q", "k"))
    P, table = case["page_size"], st["page_table"].tolist()
    if case["op"] == "attend":
        return _exact_attend(case, st)
    new, lens = _new_tokens(case)
    q_out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    caches = st["k_cache"].double(), st["v_cache"].double()
    begin = 0
    for b, (n, end) in enumerate(zip(new, lens)):
        if case["packed"]:
            rows = slice(begin, begin + n)
            begin += n
        else:
            rows = slice(b, b + 1) if case["tokens"] == 1 else b
        at = list(range(end - n, end))
        if not n:
            continue
        positions = torch.tensor(at, device="cuda")
        pages = torch.tensor([table[b][p // P] for p in at], device="cuda")
        slots = torch.tensor([p % P for p in at], device="cuda")
        caches[0][pages, slots] = _exact_rotate(st["k"][rows], positions, case)
        caches[1][pages, slots] = st["v"][rows].double()
        q_out[rows] = _exact_rotate(st["q"][rows], positions, case)
    return q_out, *caches


def _exact_attend(case, st):
    B, H, Hkv, D, P = case["batch"], case["heads"], case["heads_kv"], case["dim"], case["page_size"]
    G = H // Hkv
    o = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        pages = st["page_table"][b, first // P : -(-n // P)].long()
        inside = slice(first % P, first % P + n - first)
        keys, values = (st[c][pages].flatten(0, 1)[inside].double() for c in ("k_cache", "v_cache"))
        for h in range(Hkv):
            score = st["q"][b, h * G : (h + 1) * G].double() @ keys[:, h].T / math.sqrt(D)
            total = torch.logsumexp(score, dim=-1)
            o[b, h * G : (h + 1) * G] = torch.exp(score - total[:, None]) @ values[:, h]
            lse[b, h * G : (h + 1) * G] = total / math.log(2.0)
    return o, lse
