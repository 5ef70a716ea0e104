"""The rotary and paged-cache operators together, as a model serves and trains with them: prompts
through rotary positions and the prefill attention, the same tokens appended to a paged cache, and
single tokens that continue them; a training step through the rotary positions."""

import pytest
import torch

from oracle import reference as base
from oracle import serving_attention as ref
from oracle.recurrent import assert_within
from tileops.ops.attention import (
    MultiHeadAttentionFwdOp,
    PagedAttentionDecodeOp,
    PagedKVAppendOp,
    RotaryEmbeddingBwdOp,
    RotaryEmbeddingFwdOp,
    rotary_frequencies,
)
from tileops.ops.norm import FusedAddLayerNormFwdOp

pytestmark = pytest.mark.gpu


def _table(B, pages_each):
    order = torch.randperm(B * pages_each).view(B, pages_each)
    return order.to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """The prefill's output for its last token, and single-token attention's for the same token."""
    B, S, H, D, P = 2, 200, 4, 64, 16
    qkv = torch.randn(B, S, 3 * H * D, device="cuda").to(dtype)
    q, k, v = (t.unflatten(-1, (H, D)) for t in qkv.split(H * D, dim=-1))
    qr, kr = RotaryEmbeddingFwdOp(B, S, H, H, D, dtype=dtype)(q, k)
    o, lse = MultiHeadAttentionFwdOp(B, H, S, D, True, dtype)(qr, kr, v.contiguous())
    kc, vc = (torch.zeros(B * 13, P, H, D, device="cuda", dtype=dtype) for _ in range(2))
    table, lens = _table(B, 13), torch.full((B,), S, dtype=torch.int32, device="cuda")
    q_out = PagedKVAppendOp(H, D, P, H, D, dtype=dtype)(k, v, kc, vc, table, lens, q)
    assert torch.equal(q_out, qr)
    gathered = kc[table.long()].flatten(1, 2)[:, :S], vc[table.long()].flatten(1, 2)[:, :S]
    assert torch.equal(gathered[0], kr) and torch.equal(gathered[1], v)
    o1, lse1 = PagedAttentionDecodeOp(H, H, D, P, dtype=dtype)(qr[:, -1], kc, vc, table, lens)
    want = ref.attend(qr[:, -1], kc, vc, table, lens)
    assert_within(o1, want[0], want[2], "o")
    assert_within(lse1, want[1], want[3], "lse")
    torch.testing.assert_close(o[:, -1].cpu().double(), want[0], atol=1e-2, rtol=1e-2)
    torch.testing.assert_close(lse[:, :, -1].cpu().double(), want[1], atol=1e-5, rtol=1e-5)


def test_serving_loop_in_a_graph():
    """Ragged packed prompts, then captured steps (append and rotate, attention, the norm behind
    it) of a batch with an idle slot, replayed token after token across page bounds."""
    B, H, Hkv, D, P, steps, dt = 4, 8, 2, 64, 16, 20, torch.bfloat16
    prompt = [30, 0, 17, 64]
    table = _table(B, 6)
    kc, vc = (torch.zeros(B * 6, P, Hkv, D, device="cuda", dtype=dt) for _ in range(2))
    f = rotary_frequencies(D, factor=4.0, original_length=64)
    append = PagedKVAppendOp(Hkv, D, P, H, D, frequencies=f, amplitude=1.1)
    attend = PagedAttentionDecodeOp(H, Hkv, D, P, window=40)
    norm = FusedAddLayerNormFwdOp(dtype=dt)
    w, b = torch.ones(H * D, device="cuda"), torch.zeros(H * D, device="cuda")
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, *prompt]).cumsum(0).to(torch.int32).cuda()
    k, v = (torch.randn(sum(prompt), Hkv, D, device="cuda").to(dt) for _ in range(2))
    want_kc, want_vc = kc.clone().double().cpu(), vc.clone().double().cpu()

    def expect(k, v, q=None, cu=None):
        nonlocal want_kc, want_vc
        got = ref.append(k, v, want_kc, want_vc, table, lens, f, q, cu, 1.1)
        want_kc, want_vc = got[2], got[4]
        return got

    append(k, v, kc, vc, table, lens, None, cu)
    assert_within(kc, *expect(k, v, cu=cu)[2:4], "prompt")
    q, k, v = (torch.randn(B, n, D, device="cuda").to(dt) for n in (H, Hkv, Hkv))
    stream = torch.randn(B, H * D, device="cuda").to(dt)
    active = torch.tensor([1, 0, 1, 1], dtype=torch.int32, device="cuda")

    def step():
        lens.add_(active)
        qr = append(k, v, kc, vc, table, lens, q)
        o, lse = attend(qr, kc, vc, table, lens)
        y, s = norm(o.view(B, H * D), stream, w, b)
        return qr, o, lse, y, s

    keep = kc.clone(), vc.clone(), lens.clone()
    step()  # before the capture: device lookups
    for t, saved in zip((kc, vc, lens), keep):
        t.copy_(saved)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(steps):
        for t in (q, k, v):
            t.normal_()
        graph.replay()
        qr, o, lse, y, s = out
        got = expect(k, v, q)
        assert_within(qr, got[0], got[1], f"q, step {n}")
        assert_within(kc, got[2], got[3], f"k, step {n}")
        want_kc, want_vc = kc.cpu().double(), vc.cpu().double()  # as rounded
        want = ref.attend(qr, kc, vc, table, lens, window=40)
        assert_within(o, want[0], want[2], f"o, step {n}")
        live = lens > 0
        assert_within(lse[live], want[1][live.cpu()], want[3][live.cpu()], f"lse, step {n}")
        assert (o[1] == 0).all() and (qr[1] == 0).all()
        y_ref, s_ref = base.fused_add_layer_norm(o.view(B, H * D), stream, w, b)
        assert torch.equal(s.cpu(), s_ref)
        torch.testing.assert_close(y.cpu(), y_ref, atol=1.6e-2, rtol=1.6e-2)
    assert lens.tolist() == [n + steps if n else 0 for n in prompt]


def test_a_training_step():
    """q, k -> rotary positions -> scores -> softmax -> values in fp32; the gradients of the inputs
    through RotaryEmbeddingBwdOp against automatic differentiation of the formulas in 64 bits.

    The products and the softmax are torch's, in fp32 sums of up to 96 terms (96 u) three after
    another, the rotations 8 u each: 2000 u of each gradient's largest value holds them."""
    B, S, H, D, R = 2, 96, 3, 64, 48
    f = rotary_frequencies(R)
    at = torch.randint(0, 1 << 18, (B, S), device="cuda")
    q, k, v, d = (torch.randn(B, S, H, D, device="cuda") for _ in range(4))
    args = (B, S, H, H, D, R)
    fwd = RotaryEmbeddingFwdOp(*args, dtype=torch.float32)
    bwd = RotaryEmbeddingBwdOp(*args, dtype=torch.float32)
    qr, kr = (t.requires_grad_() for t in fwd(q, k, at))
    s = torch.einsum("bshd,bthd->bhst", qr, kr) / D**0.5
    o = torch.einsum("bhst,bthd->bshd", torch.softmax(s, -1), v)
    dq, dk = bwd(*torch.autograd.grad(o, (qr, kr), d), at)

    wide = [t.detach().cpu().double().requires_grad_() for t in (q, k)]
    turn = ref.angles(at, f)[..., None, :]

    def rotate(x):
        a, b, rest = x[..., :R // 2], x[..., R // 2:R], x[..., R:]
        c, s = torch.cos(turn), torch.sin(turn)
        return torch.cat([a * c - b * s, a * s + b * c, rest], -1)

    s = torch.einsum("bshd,bthd->bhst", *(rotate(t) for t in wide)) / D**0.5
    o = torch.einsum("bhst,bthd->bshd", torch.softmax(s, -1), v.cpu().double())
    want = torch.autograd.grad(o, wide, d.cpu().double())
    for g, w in zip((dq, dk), want):
        assert (g.cpu().double() - w).abs().max() <= 2000 * 2.0**-24 * w.abs().max()


def test_a_captured_backward_beside_an_eager_graph():
    """The backward op captured while an eager autograd graph of the same leaves lives."""
    B, S, H, D = 1, 12, 2, 64
    q, k = (torch.randn(B, S, H, D, device="cuda").requires_grad_() for _ in range(2))
    alive = (q * k).sum()
    bwd = RotaryEmbeddingBwdOp(B, S, H, H, D, dtype=torch.float32)
    want = bwd(q, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = bwd(q, k)
    graph.replay()
    assert torch.equal(got[0], want[0]) and not got[0].requires_grad
    alive.backward()
    assert torch.equal(q.grad, k.detach())
