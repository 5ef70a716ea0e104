"""Cases and plain forms of the recurrent-block operators.

Five entry points are measured:

* ``rec_fwd``   GatedLinearRecurrenceFwdOp: prefill over a whole sequence or over packed sequences;
* ``rec_train`` the same forward with its saved states, followed by GatedLinearRecurrenceBwdOp;
* ``rec_step``  GatedLinearRecurrenceDecodeOp: one token of every sequence of a batch;
* ``norm_fwd``  FusedSandwichNormFwdOp: the norm after a block, its gate, the scaled residual, the next block's norm;
* ``norm_bwd``  FusedSandwichNormBwdOp: its gradients.

``run`` computes them in elementary torch operations where ``own`` is false and through the package where it is true;
``exact`` computes them in 64 bits by another route (token after token, gradients by automatic differentiation).
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
DECAY_SCALE = 8.0  # c in log a = -c softplus(lambda) sigmoid(decay gate)
EPS = 1e-6


def listed():
    return [
        # A short prompt of one user; the three inputs are column slices of one projection's output.
        {"name": "rec prefill short", "op": "rec_fwd", "batch": 1, "seq_len": 257, "dim": 2560, "dtype": "bfloat16",
         "seqs": 0, "sliced": True},
        # One long document, the case the time axis is split for.
        {"name": "rec prefill long", "op": "rec_fwd", "batch": 1, "seq_len": 65536, "dim": 4096, "dtype": "bfloat16",
         "seqs": 0, "sliced": False},
        # Requests of many lengths packed on one axis, some of them empty.
        {"name": "rec prefill packed", "op": "rec_fwd", "batch": 1, "seq_len": 12345, "dim": 1600, "dtype": "float16",
         "seqs": 37, "sliced": False},
        # A training step's batch.
        {"name": "rec train", "op": "rec_train", "batch": 8, "seq_len": 4096, "dim": 4096, "dtype": "bfloat16",
         "seqs": 0, "sliced": False},
        # Odd sizes in full precision, as in a numerics check of a small model.
        {"name": "rec train odd f32", "op": "rec_train", "batch": 3, "seq_len": 1001, "dim": 1111, "dtype": "float32",
         "seqs": 0, "sliced": False},
        # Documents packed into one training row.
        {"name": "rec train packed", "op": "rec_train", "batch": 1, "seq_len": 16384, "dim": 2048, "dtype": "bfloat16",
         "seqs": 23, "sliced": False},
        # One token of one user: launch latency.
        {"name": "rec step one", "op": "rec_step", "batch": 1, "dim": 2560, "dtype": "bfloat16"},
        # One token of a large serving batch.
        {"name": "rec step batch", "op": "rec_step", "batch": 512, "dim": 4096, "dtype": "bfloat16"},
        # Between two blocks while decoding for one user.
        {"name": "norm fwd one", "op": "norm_fwd", "rows": 1, "n": 4096, "groups": 1, "norm": "rms", "bias": False,
         "dtype": "bfloat16", "affine": "bfloat16"},
        # The FusedAddLayerNorm benchmark's shape, with a gate per sample and affine parameters in fp32.
        {"name": "norm fwd layer", "op": "norm_fwd", "rows": 8192, "n": 4096, "groups": 8, "norm": "layer", "bias": True,
         "dtype": "bfloat16", "affine": "float32"},
        # A training batch between two blocks, backwards.
        {"name": "norm bwd rms", "op": "norm_bwd", "rows": 16384, "n": 4096, "groups": 1, "norm": "rms", "bias": False,
         "dtype": "bfloat16", "affine": "float32"},
        # Odd row length, few rows, biases and a gate per sample, in full precision.
        {"name": "norm bwd odd layer f32", "op": "norm_bwd", "rows": 1025, "n": 1155, "groups": 5, "norm": "layer",
         "bias": True, "dtype": "float32", "affine": "float32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 64, at times one of 8, at times any number."""
    n = _log_int(rng, lo, hi)
    q = rng.choice([64, 64, 64, 8, 1])
    return max(q, n // q * q)


def draw(rng):
    op = rng.choice(["rec_fwd", "rec_fwd", "rec_train", "rec_train", "rec_step", "norm_fwd", "norm_bwd"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "rec_step":
        return {"op": op, "batch": _log_int(rng, 1, 512), "dim": _width(rng, 256, 8192), "dtype": dtype}
    if op in ("rec_fwd", "rec_train"):
        dim = _width(rng, 256, 8192)
        most = (1 << (26 if op == "rec_fwd" else 25)) // dim  # tokens
        if rng.random() < 0.4:
            batch, seq_len = 1, _log_int(rng, 64, min(65536, most))
            seqs = _log_int(rng, 1, 64)
        else:
            batch = _log_int(rng, 1, 16)
            seq_len, seqs = _log_int(rng, 1, min(65536, most // batch)), 0
        return {"op": op, "batch": batch, "seq_len": seq_len, "dim": dim, "dtype": dtype, "seqs": seqs,
                "sliced": rng.random() < 0.3}
    n = _width(rng, 256, 16384)
    rows = _log_int(rng, 1, min(16384, (1 << 25) // n))
    groups = rng.choice([g for g in (1, 1, 2, 3, 4, 8) if rows % g == 0])
    return {"op": op, "rows": rows, "n": n, "groups": groups, "norm": rng.choice(["rms", "layer"]),
            "bias": rng.random() < 0.5, "dtype": dtype, "affine": rng.choice([dtype, "float32"])}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, to=dtype, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda")).to(to)

    state = {"case": dict(case)}
    if case["op"].startswith("rec"):
        D = case["dim"]
        # softplus(lambda) such that a gate fully open decays by 0.9 to 0.999 a token.
        a = 0.9 + 0.099 * torch.rand(D, generator=g, device="cuda")
        state["decay_param"] = torch.log(torch.expm1(-torch.log(a) / DECAY_SCALE))
        if case["op"] == "rec_step":
            B = case["batch"]
            shape, nseq = (B, D), B
        else:
            B, T = case["batch"], case["seq_len"]
            shape, nseq = (B, T, D), case["seqs"] or B
            if case["seqs"]:
                cuts = torch.randint(0, T + 1, (case["seqs"] - 1,), generator=g, device="cuda")
                cuts[: len(cuts) // 8] = cuts[-1] if len(cuts) else 0  # some sequences are empty
                ends = torch.tensor([0, T], device="cuda")
                state["cu_seqlens"] = torch.cat([ends, cuts]).sort().values.to(torch.int32)
        if case.get("sliced"):
            both = randn(*shape[:-1], 3 * D)
            state["x"], state["input_gate"], state["decay_gate"] = both.split(D, dim=-1)
        else:
            for name in ("x", "input_gate", "decay_gate"):
                state[name] = randn(*shape)
        state["initial_state"] = randn(nseq, D, to=torch.float32)
        if case["op"] == "rec_train":
            state["dy"] = randn(*shape)
            state["d_final_state"] = randn(nseq, D, to=torch.float32)
    else:
        M, N, G, affine = case["rows"], case["n"], case["groups"], DTYPES[case["affine"]]
        state["x"] = randn(M, N)
        state["residual"] = randn(M, N, scale=2.0)  # forward: the stream before; backward: the one after
        for name in ("post", "pre"):
            state[name + "_weight"] = (1.0 + 0.1 * randn(N, to=torch.float32)).to(affine)
            state[name + "_bias"] = randn(N, to=affine, scale=0.1) if case["bias"] else None
        state["gate"] = (0.5 + 0.3 * randn(G, N, to=torch.float32)).to(affine)
        state["residual_scale"] = 0.875
        if case["op"] == "norm_bwd":
            state["dy"], state["d_residual"] = randn(M, N), randn(M, N)
    return state


# ------------------------------------------------------- plain forms, 32 bits
def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1 from h = 0: neighbours joined in pairs, the half as long scan, then the tokens
    between."""
    n = a.shape[1]
    if n == 1:
        return u.clone()
    half = n // 2 * 2
    odd = a[:, 1:half:2]
    h_odd = _scan(a[:, 0:half:2] * odd, odd * u[:, 0:half:2] + u[:, 1:half:2])
    h = torch.empty_like(u)
    h[:, 1:half:2] = h_odd
    h[:, 0] = u[:, 0]
    h[:, 2::2] = a[:, 2::2] * h_odd[:, : (n - 1) // 2] + u[:, 2::2]
    return h


def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _gates(x, input_gate, decay_gate, decay_param):
    lam = decay_param.float()
    k = DECAY_SCALE * (lam.clamp(min=0) + torch.log1p(torch.exp(-lam.abs())))
    si, sr = _sigmoid(input_gate.float()), _sigmoid(decay_gate.float())
    log_a = -k * sr
    m = torch.sqrt(-torch.expm1(2.0 * log_a))
    return k, si, sr, torch.exp(log_a), m, m * si * x.float()


def _bounds(st):
    """Per token: its sequence, whether it is that one's first and its last; per sequence: its first and last token and
    whether it has none."""
    c = st["case"]
    T = c["seq_len"]
    t = torch.arange(T, device="cuda")
    if not c["seqs"]:
        return None, (t == 0)[None, :, None], (t == T - 1)[None, :, None], None, None, None
    cu = st["cu_seqlens"].long()
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return (seq, (t == cu[seq])[None, :, None], (t == cu[seq + 1] - 1)[None, :, None], cu[:-1].clamp(max=T - 1),
            (cu[1:] - 1).clamp(min=0), (cu[1:] == cu[:-1])[:, None])


def _per_token(v, seq):
    """A value of each sequence, at each of its tokens."""
    return v[:, None, :] if seq is None else v[seq][None]


def _plain_rec_fwd(st):
    seq, first, _, _, last_at, empty = _bounds(st)
    k, si, sr, a, m, u = _gates(st["x"], st["input_gate"], st["decay_gate"], st["decay_param"])
    h0 = _per_token(st["initial_state"], seq)
    h = _scan(torch.where(first, 0.0, a), torch.where(first, u + a * h0, u))
    final = h[:, -1] if seq is None else torch.where(empty, st["initial_state"], h[0, last_at])
    return (k, si, sr, a, m, h), h.to(st["x"].dtype), final.clone()


def _plain_rec_bwd(st, saved):
    k, si, sr, a, m, h = saved
    seq, first, last, first_at, _, empty = _bounds(st)
    x, dt = st["x"].float(), st["x"].dtype
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    into = torch.where(last, st["dy"].float() + _per_token(st["d_final_state"], seq), st["dy"].float())
    G = _scan(torch.where(last, 0.0, after).flip(1), into.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], dim=1)
    before = torch.where(first, _per_token(st["initial_state"], seq), before)
    dx = G * m * si
    d_input = dx * x * (1.0 - si)
    over_m = torch.where(m > 0, 1.0 / m, 0.0)
    d_log_a = a * G * (before - a * si * x * over_m)
    d_decay = -k * sr * (1.0 - sr) * d_log_a
    d_param = DECAY_SCALE * _sigmoid(st["decay_param"]) * -(sr * d_log_a).sum(dim=(0, 1))
    back = a * G
    d_initial = back[:, 0] if seq is None else torch.where(empty, st["d_final_state"], back[0, first_at])
    return dx.to(dt), d_input.to(dt), d_decay.to(dt), d_param, d_initial.clone()


def _plain_step(st):
    _, _, _, a, _, u = _gates(st["x"], st["input_gate"], st["decay_gate"], st["decay_param"])
    h = a * st["initial_state"] + u
    return h.to(st["x"].dtype), h


def _normed(x, kind):
    """(x - mean) rstd and rstd; RMS takes no mean."""
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    return x * rstd, rstd


def _rows(gate, M):
    return gate.float().repeat_interleave(M // gate.shape[0], dim=0)


def _plain_norm_fwd(st):
    kind, dt = st["case"]["norm"], st["x"].dtype
    p = _normed(st["x"].float(), kind)[0] * st["post_weight"].float()
    if st["post_bias"] is not None:
        p = p + st["post_bias"].float()
    s = (st["residual_scale"] * st["residual"].float() + _rows(st["gate"], p.shape[0]) * p).to(dt)
    y = _normed(s.float(), kind)[0] * st["pre_weight"].float()
    if st["pre_bias"] is not None:
        y = y + st["pre_bias"].float()
    return y.to(dt), s


def _plain_norm_grad(e, hat, rstd, kind):
    e = e - hat * (e * hat).mean(dim=-1, keepdim=True) - (e.mean(dim=-1, keepdim=True) if kind == "layer" else 0.0)
    return rstd * e


def _plain_norm_bwd(st):
    kind, dt, at = st["case"]["norm"], st["x"].dtype, st["gate"].dtype
    M, N = st["x"].shape
    G = st["gate"].shape[0]
    dy = st["dy"].float()
    s_hat, s_rstd = _normed(st["residual"].float(), kind)
    x_hat, x_rstd = _normed(st["x"].float(), kind)
    ds = st["d_residual"].float() + _plain_norm_grad(dy * st["pre_weight"].float(), s_hat, s_rstd, kind)
    w1 = st["post_weight"].float()
    dx = _plain_norm_grad(ds * _rows(st["gate"], M) * w1, x_hat, x_rstd, kind)
    P = (ds * x_hat).view(G, M // G, N).sum(dim=1)
    d_post, d_pre, d_gate = (st["gate"].float() * P).sum(dim=0), (dy * s_hat).sum(dim=0), w1 * P
    out = [dx.to(dt), (st["residual_scale"] * ds).to(dt), d_post.to(at), d_pre.to(at)]
    if st["post_bias"] is None:
        return out + [d_gate.to(at)]
    Q = ds.view(G, M // G, N).sum(dim=1)
    d_gate = d_gate + st["post_bias"].float() * Q
    return out + [d_gate.to(at), (st["gate"].float() * Q).sum(dim=0).to(at), dy.sum(dim=0).to(at)]


# ------------------------------------------------------------ one pass
def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tile-ascendnpu-ops_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import tileops.ops.linear_attention as rec
    import tileops.ops.norm as norm
    return rec, norm


def _own_ops(st):
    """The op objects of a case, built on its first pass and kept, as a program keeps them."""
    if "ops" not in st:
        rec, norm = _package()
        c, dt = st["case"], st["x"].dtype
        if c["op"] == "rec_step":
            st["ops"] = [rec.GatedLinearRecurrenceDecodeOp(c["batch"], c["dim"], DECAY_SCALE, dt)]
        elif c["op"] == "rec_fwd":
            st["ops"] = [rec.GatedLinearRecurrenceFwdOp(c["batch"], c["seq_len"], c["dim"], DECAY_SCALE, dt)]
        elif c["op"] == "rec_train":
            size = (c["batch"], c["seq_len"], c["dim"], DECAY_SCALE, dt)
            st["ops"] = [rec.GatedLinearRecurrenceFwdOp(*size, save_states=True),
                         rec.GatedLinearRecurrenceBwdOp(*size)]
        else:
            op = norm.FusedSandwichNormFwdOp if c["op"] == "norm_fwd" else norm.FusedSandwichNormBwdOp
            st["ops"] = [op(dtype=dt, norm=c["norm"], eps=EPS, residual_scale=st["residual_scale"])]
    return st["ops"]


def run(state):
    st, op = state, state["case"]["op"]
    if own:
        ops = _own_ops(st)
        if op == "norm_fwd":
            return ops[0](st["x"], st["residual"], st["post_weight"], st["pre_weight"], st["gate"], st["post_bias"],
                          st["pre_bias"])
        if op == "norm_bwd":
            got = ops[0](st["dy"], st["d_residual"], st["x"], st["residual"], st["post_weight"], st["pre_weight"],
                         st["gate"], st["post_bias"], st["pre_bias"])
            return [t for t in got if t is not None]
        gates = st["x"], st["input_gate"], st["decay_gate"], st["decay_param"]
        if op == "rec_step":
            return ops[0](*gates, st["initial_state"])
        if op == "rec_fwd":
            return ops[0](*gates, st["initial_state"], st.get("cu_seqlens"))
        y, final, states = ops[0](*gates, st["initial_state"], st.get("cu_seqlens"))
        return y, final, *ops[1](st["dy"], *gates, states, st["initial_state"], st["d_final_state"],
                                 st.get("cu_seqlens"))
    if op == "norm_fwd":
        return _plain_norm_fwd(st)
    if op == "norm_bwd":
        return _plain_norm_bwd(st)
    if op == "rec_step":
        return _plain_step(st)
    saved, y, final = _plain_rec_fwd(st)
    if op == "rec_fwd":
        return y, final
    return y, final, *_plain_rec_bwd(st, saved)


def work(case):
    eb = DTYPES[case["dtype"]].itemsize
    if case["op"].startswith("norm"):
        M, N, G, ab = case["rows"], case["n"], case["groups"], DTYPES[case["affine"]].itemsize
        params = (2 + G + (2 if case["bias"] else 0)) * N * ab
        if case["op"] == "norm_fwd":
            return {"bytes": 4 * M * N * eb + params, "flops": 14 * M * N}
        return {"bytes": 6 * M * N * eb + 2 * params, "flops": 30 * M * N}
    D = case["dim"]
    if case["op"] == "rec_step":
        return {"bytes": case["batch"] * D * (4 * eb + 8) + 4 * D, "flops": 20 * case["batch"] * D}
    elems = case["batch"] * case["seq_len"] * D
    states = 4 * D * (case["seqs"] or case["batch"])
    if case["op"] == "rec_fwd":
        return {"bytes": 4 * elems * eb + 2 * states + 4 * D, "flops": 20 * elems}
    return {"bytes": 8 * elems * eb + 4 * states + 8 * D, "flops": 50 * elems}


# ------------------------------------------------- 64 bits, by another route
def _exact_gates(x, i, r, lam):
    k = DECAY_SCALE * torch.nn.functional.softplus(lam, threshold=60)
    log_a = -k * torch.sigmoid(r)
    return torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a)) * torch.sigmoid(i) * x


def exact(case, seed):
    st = prepare(case, seed)
    wide = {n: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for n, v in st.items()}
    if case["op"].startswith("norm"):
        return _exact_norm(case, st, wide)
    x, i, r, lam = (wide[n].detach().requires_grad_() for n in ("x", "input_gate", "decay_gate", "decay_param"))
    train = case["op"] == "rec_train"
    with torch.set_grad_enabled(train):
        a_graph, u_graph = _exact_gates(x, i, r, lam)
    a, u = a_graph.detach(), u_graph.detach()
    h0 = wide["initial_state"]
    if case["op"] == "rec_step":
        h = a * h0 + u
        return h, h
    # Token after token, for all samples of the batch at once, or one sequence of a packed row after another.
    T, packed = case["seq_len"], bool(case["seqs"])
    cu = st["cu_seqlens"].tolist() if packed else [0, T]
    y, before = torch.empty_like(u), torch.empty_like(u) if train else None
    final = h0.clone()
    for n in range(len(cu) - 1):
        h = h0[n : n + 1] if packed else h0
        for t in range(cu[n], cu[n + 1]):
            if train:
                before[:, t] = h
            h = torch.addcmul(u[:, t], a[:, t], h)
            y[:, t] = h
        final[n : n + 1 if packed else None] = h
    if not train:
        return y, final
    dy, d_final = wide["dy"], wide["d_final_state"]
    grad, d_initial = torch.empty_like(u), d_final.clone()
    for n in range(len(cu) - 1):
        back = d_final[n : n + 1] if packed else d_final
        for t in reversed(range(cu[n], cu[n + 1])):
            G = dy[:, t] + back
            grad[:, t] = G
            back = a[:, t] * G
        d_initial[n : n + 1 if packed else None] = back
    dx, di, dr, dlam = torch.autograd.grad((a_graph, u_graph), (x, i, r, lam), (before.mul_(grad), grad))
    return y, final, dx, di, dr, dlam, d_initial


def _exact_rows(x, w, b, kind):
    centre = x - x.mean(dim=-1, keepdim=True) if kind == "layer" else x
    out = centre * torch.rsqrt(centre.square().mean(dim=-1, keepdim=True) + EPS) * w
    return out if b is None else out + b


def _exact_norm(case, st, wide):
    kind, M, N, G = case["norm"], case["rows"], case["n"], case["groups"]

    def joined(x, residual, w, b, gate):
        p = _exact_rows(x, w, b, kind).view(G, M // G, N)
        return st["residual_scale"] * residual + (gate[:, None, :] * p).view(M, N)

    if case["op"] == "norm_fwd":
        s = joined(wide["x"], wide["residual"], wide["post_weight"], wide["post_bias"], wide["gate"])
        # The stream between two blocks is kept in the inputs' type, and the next norm reads what is kept.
        kept = s.to(st["x"].dtype).double()
        return _exact_rows(kept, wide["pre_weight"], wide["pre_bias"], kind), s
    leaf = {n: v.detach().requires_grad_() for n, v in wide.items() if isinstance(v, torch.Tensor)}
    bias = case["bias"]
    y = _exact_rows(leaf["residual"], leaf["pre_weight"], leaf.get("pre_bias"), kind)
    into = [leaf["residual"], leaf["pre_weight"]] + ([leaf["pre_bias"]] if bias else [])
    ds, d_pre, *d_pre_bias = torch.autograd.grad(y, into, wide["dy"])
    ds = ds + wide["d_residual"]
    before = torch.zeros_like(ds, requires_grad=True)
    s = joined(leaf["x"], before, leaf["post_weight"], leaf.get("post_bias"), leaf["gate"])
    into = [leaf["x"], before, leaf["post_weight"], leaf["gate"]] + ([leaf["post_bias"]] if bias else [])
    dx, dr, d_post, d_gate, *d_post_bias = torch.autograd.grad(s, into, ds)
    return [dx, dr, d_post, d_pre, d_gate, *d_post_bias, *d_pre_bias]
