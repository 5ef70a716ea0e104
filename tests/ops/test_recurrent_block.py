"""The recurrent-block operators together, as a model runs them: norm -> causal conv1d ->
gated linear recurrence -> gelu gate -> norm, forward over whole sequences and backwards through
the recurrence and the norm; and a prefill continued token by token."""

import pytest
import torch

from oracle import recurrent as ref
from oracle import reference as base
from tileops.ops.convolution import CausalDepthwiseConv1dFwdOp
from tileops.ops.elementwise import GeluAndMulFwdOp
from tileops.ops.linear_attention import (
    GatedLinearRecurrenceBwdOp,
    GatedLinearRecurrenceDecodeOp,
    GatedLinearRecurrenceFwdOp,
)
from tileops.ops.norm import FusedSandwichNormBwdOp, FusedSandwichNormFwdOp

pytestmark = pytest.mark.gpu


def test_block_forward():
    """Each step's output against the oracle's of the step's actual input."""
    B, T, D, dt = 2, 333, 256, torch.bfloat16
    x, stream = (torch.randn(B, T, D, device="cuda").to(dt) for _ in range(2))
    w = [1 + 0.1 * torch.randn(D, device="cuda") for _ in range(4)]
    gate = torch.randn(B, D, device="cuda")
    norm = FusedSandwichNormFwdOp(dtype=dt)
    y, stream = norm(x, stream, w[0], w[1], gate)
    # the block: projections in torch, then conv, recurrence and gate
    wide = y @ (torch.randn(D, 4 * D, device="cuda") / D**0.5).to(dt)
    branch, i, r, z = wide.split(D, dim=-1)
    cw, cb = (0.5 * torch.randn(D, 4, device="cuda")).to(dt), torch.zeros(D, device="cuda", dtype=dt)
    v = CausalDepthwiseConv1dFwdOp(activation="silu")(branch.transpose(1, 2).contiguous(), cw, cb)
    v = v.transpose(1, 2)
    lam = torch.randn(D, device="cuda") - 4
    h, final = GatedLinearRecurrenceFwdOp(B, T, D)(v, i, r, lam)
    h_ref, f_ref, h_tol, f_tol = ref.glr_fwd(v, i, r, lam)
    ref.assert_within(h, h_ref, h_tol, "h")
    ref.assert_within(final, f_ref, f_tol, "final")
    pair = torch.cat([z, h], dim=-1).reshape(B * T, 2 * D)
    out = GeluAndMulFwdOp(M=B * T, N=D, dtype=dt)(pair)
    torch.testing.assert_close(out.cpu(), base.gelu_and_mul(pair), atol=1.6e-2, rtol=1.6e-2)
    out = out.view(B, T, D)
    y2, s2 = norm(out, stream, w[2], w[3], gate)
    s_ref, s_tol = ref.sandwich_stream(out.reshape(-1, D), stream.reshape(-1, D), w[2], gate)
    ref.assert_within(s2.reshape(-1, D), s_ref, s_tol, "stream")
    y_ref, y_tol = ref.sandwich_next(s2.reshape(-1, D), w[3])
    ref.assert_within(y2.reshape(-1, D), y_ref, y_tol, "y")


def test_two_layers_train():
    """recurrence -> norm -> recurrence -> norm in fp32; every gradient against automatic
    differentiation in 64 bits of the same formulas.

    A gradient here passes two recurrences of decays below 0.99 (a sum of at most 100 tokens'
    weight each) and two norms, whose own bounds are about 100 u and 64 u relative to the largest
    values: 1e-4 of the largest value of each gradient (1700 u) holds them all."""
    B, T, D, layers = 2, 130, 96, 2
    torch.manual_seed(7)
    draw = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    leaves = {"x": draw(B, T, D), "res": draw(B, T, D)}
    for n in range(layers):
        leaves |= {f"i{n}": draw(B, T, D), f"r{n}": draw(B, T, D), f"lam{n}": draw(D) * 0.3 - 3,
                   f"h0{n}": draw(B, D), f"w1{n}": 1 + 0.1 * draw(D), f"w2{n}": 1 + 0.1 * draw(D),
                   f"g{n}": draw(B, D)}
    dy, ds = draw(B, T, D), draw(B, T, D)

    fwd = GatedLinearRecurrenceFwdOp(B, T, D, dtype=torch.float32, save_states=True)
    bwd = GatedLinearRecurrenceBwdOp(B, T, D, dtype=torch.float32)
    norm, norm_bwd = FusedSandwichNormFwdOp(), FusedSandwichNormBwdOp()
    y, s, kept = leaves["x"], leaves["res"], []
    for n in range(layers):
        p = [leaves[f"{k}{n}"] for k in ("i", "r", "lam", "h0", "w1", "w2", "g")]
        h, _, states = fwd(y, *p[:4])
        y_in, (y, s) = y, norm(h, s, *p[4:])
        kept.append((y_in, h, states, s))
    grads, d, d_s = {}, dy, ds
    for n in reversed(range(layers)):
        i, r, lam, h0, w1, w2, g = (leaves[f"{k}{n}"] for k in ("i", "r", "lam", "h0", "w1", "w2", "g"))
        y_in, h, states, s_out = kept[n]
        dh, d_s, grads[f"w1{n}"], grads[f"w2{n}"], grads[f"g{n}"], _, _ = norm_bwd(
            d, d_s, h, s_out, w1, w2, g)
        d, grads[f"i{n}"], grads[f"r{n}"], grads[f"lam{n}"], grads[f"h0{n}"] = bwd(
            dh, y_in, i, r, lam, states, h0)
    grads |= {"x": d, "res": d_s}

    wide = {k: v.detach().cpu().double().requires_grad_() for k, v in leaves.items()}

    def rms(v, w):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w

    y, s = wide["x"], wide["res"]
    for n in range(layers):
        la = -8 * torch.nn.functional.softplus(wide[f"lam{n}"]) * torch.sigmoid(wide[f"r{n}"])
        a, u = torch.exp(la), torch.sqrt(-torch.expm1(2 * la)) * torch.sigmoid(wide[f"i{n}"]) * y
        h, hs = wide[f"h0{n}"], []
        for t in range(T):
            h = a[:, t] * h + u[:, t]
            hs.append(h)
        s = s + wide[f"g{n}"][:, None] * rms(torch.stack(hs, 1), wide[f"w1{n}"])
        y = rms(s, wide[f"w2{n}"])
    want = torch.autograd.grad((y * dy.cpu()).sum() + (s * ds.cpu()).sum(), list(wide.values()))
    for k, w in zip(wide, want):
        off = (grads[k].cpu().double() - w).abs().max()
        assert off <= 1e-4 * w.abs().max(), (k, float(off), float(w.abs().max()))


def test_serving_loop_in_a_graph():
    """Prefill, then a captured decode step (recurrence in place, then the norm) replayed."""
    B, D, dt, steps = 3, 512, torch.bfloat16, 6
    lam = torch.randn(D, device="cuda") - 3
    x, i, r = (torch.randn(B, 40 + steps, D, device="cuda").to(dt) for _ in range(3))
    w = 1 + 0.1 * torch.randn(D, device="cuda")
    _, state = GatedLinearRecurrenceFwdOp(B, 40, D)(x[:, :40], i[:, :40], r[:, :40], lam)
    step = GatedLinearRecurrenceDecodeOp(B, D, inplace=True)
    norm = FusedSandwichNormFwdOp(dtype=dt)
    now = [t[:, 40].clone() for t in (x, i, r)]
    stream = torch.randn(B, D, device="cuda").to(dt)
    scratch = state.clone()
    h, _ = step(*now, lam, scratch)
    norm(h, stream, w, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, _ = step(*now, lam, state)
        y, s = norm(h, stream, w, w)
    y_ref, h_ref, y_tol, h_tol = ref.glr_fwd(x, i, r, lam)
    for t in range(40, 40 + steps):
        for a, b in zip(now, (x, i, r)):
            a.copy_(b[:, t])
        graph.replay()
        ref.assert_within(h, y_ref[:, t], y_tol[:, t], f"token {t}")
        n_ref, n_tol = ref.sandwich_next(s, w)
        ref.assert_within(y, n_ref, n_tol, f"norm {t}")
    ref.assert_within(state, h_ref, h_tol, "state")
