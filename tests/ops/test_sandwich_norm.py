"""GPU parity of the sandwich norm ops against the 64-bit oracle, within its error bounds plus
half a step of each type (``oracle.recurrent``); no tolerance is fitted."""

import pytest
import torch

from oracle import recurrent as ref
from tileops.ops.norm import FusedSandwichNormBwdOp, FusedSandwichNormFwdOp

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.bfloat16, torch.float32)]
NAMES = ("dx", "d_residual", "d_post_weight", "d_pre_weight", "d_gate", "d_post_bias",
         "d_pre_bias")


def _inputs(M, N, dtype, affine, G=1, bias=True, gate=True):
    x, dy, ds = (torch.randn(M, N, device="cuda").to(dtype) for _ in range(3))
    residual = (2 * torch.randn(M, N, device="cuda")).to(dtype)
    vec = lambda mean, s, *shape: (mean + s * torch.randn(*shape, device="cuda")).to(affine)  # noqa: E731
    w1, w2 = vec(1, 0.1, N), vec(1, 0.1, N)
    b1, b2 = (vec(0, 0.1, N), vec(0, 0.1, N)) if bias else (None, None)
    g = vec(0.5, 0.3, G, N) if gate else None
    return x, residual, dy, ds, (w1, w2, g, b1, b2)


def _check_fwd(x, residual, params, **kw):
    w1, w2, g, b1, b2 = params
    y, s = FusedSandwichNormFwdOp(**kw)(x, residual, *params)
    N = x.shape[-1]
    s_ref, s_tol = ref.sandwich_stream(x.reshape(-1, N), residual.reshape(-1, N), w1, g, b1, **kw)
    ref.assert_within(s.reshape(-1, N), s_ref, s_tol, "residual_out")
    y_ref, y_tol = ref.sandwich_next(s.reshape(-1, N), w2, b2, kw.get("norm", "rms"),
                                     kw.get("eps", 1e-6))
    ref.assert_within(y.reshape(-1, N), y_ref, y_tol, "y")
    assert y.shape == s.shape == x.shape and y.dtype == s.dtype == x.dtype


def _check_bwd(dy, ds, x, s, params, **kw):
    w1, w2, g, b1, b2 = params
    N = x.shape[-1]
    got = FusedSandwichNormBwdOp(**kw)(dy, ds, x, s, *params)
    flat = lambda t: None if t is None else t.reshape(-1, N)  # noqa: E731
    want, tol = ref.sandwich_bwd(flat(dy), flat(ds), flat(x), flat(s), w1, w2, g, b1, **kw)
    given = (x, x, w1, w2, g, b1, b2)
    for name, a, b, t, p in zip(NAMES, got, want, tol, given):
        if p is None:
            assert a is None, name
            continue
        assert a.dtype == p.dtype and a.shape == p.shape, name
        ref.assert_within(a.reshape(b.shape), b, t, name)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype, affine", TYPES)
@pytest.mark.parametrize("M, N", [
    (1, 1), (3, 2), (2, 7), (5, 64), (3, 100), (7, 1000), (4, 1024), (2, 1155), (3, 4096),
    (2, 4097), (2, 8192), (1, 16384), (2, 20000), (3, 4098), (2, 1001), (2, 20001),
])
def test_sizes(M, N, dtype, affine, norm):
    x, residual, dy, ds, params = _inputs(M, N, dtype, affine)
    kw = dict(norm=norm, eps=1e-5, residual_scale=0.75)
    _check_fwd(x, residual, params, **kw)
    _check_bwd(dy, ds, x, residual, params, **kw)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("bias, gate", [(False, False), (True, False), (False, True)])
def test_optional_parameters(bias, gate, norm):
    x, residual, dy, ds, params = _inputs(9, 264, torch.bfloat16, torch.float32, 3, bias, gate)
    _check_fwd(x, residual, params, norm=norm)
    _check_bwd(dy, ds, x, residual, params, norm=norm)
    _check_bwd(dy, None, x, residual, params, norm=norm)


@pytest.mark.parametrize("one", ["post", "pre"])
def test_one_bias(one):
    x, residual, dy, ds, (w1, w2, g, b1, b2) = _inputs(9, 264, torch.bfloat16, torch.float32, 3)
    params = (w1, w2, g, b1 if one == "post" else None, b2 if one == "pre" else None)
    _check_fwd(x, residual, params)
    _check_bwd(dy, ds, x, residual, params)


@pytest.mark.parametrize("M, N, dtype, affine", [
    (1500, 512, torch.bfloat16, torch.float32), (1300, 1024, torch.float16, torch.float16),
    (1201, 300, torch.float32, torch.float32), (700, 2048, torch.bfloat16, torch.bfloat16),
    (650, 4096, torch.bfloat16, torch.float32), (601, 1155, torch.bfloat16, torch.float32),
    (600, 8192, torch.bfloat16, torch.float32), (620, 2056, torch.float32, torch.float32),
])
@pytest.mark.parametrize("norm, bias", [("rms", False), ("layer", True)])
def test_many_rows(M, N, dtype, affine, norm, bias):
    """Enough rows for several a CTA."""
    x, residual, dy, ds, params = _inputs(M, N, dtype, affine, bias=bias)
    _check_fwd(x, residual, params, norm=norm, residual_scale=1.5)
    _check_bwd(dy, ds, x, residual, params, norm=norm, residual_scale=1.5)


@pytest.mark.parametrize("M, N, G", [(700, 10000, 7), (320, 20002, 1), (600, 8200, 600)])
def test_many_wide_rows(M, N, G):
    """Rows beyond a thread's registers, several a CTA, with the sums of several groups."""
    x, residual, dy, ds, params = _inputs(M, N, torch.bfloat16, torch.float32, G)
    _check_fwd(x, residual, params, norm="layer")
    _check_bwd(dy, ds, x, residual, params, norm="layer")


@pytest.mark.parametrize("M, G", [(6, 6), (6, 2), (12, 4), (400, 400), (900, 2), (1000, 8), (999, 9)])
def test_gate_groups(M, G):
    """A gate per group of rows, each with its own gradient; one per row at the end."""
    x, residual, dy, ds, params = _inputs(M, 136, torch.bfloat16, torch.float32, G)
    _check_fwd(x, residual, params)
    _check_bwd(dy, ds, x, residual, params)


def test_gate_vector_and_leading_dims():
    B, T, N = 3, 5, 72
    x, residual, dy, ds, (w1, w2, _, b1, b2) = _inputs(B * T, N, torch.float16, torch.float16)
    gate = torch.randn(N, device="cuda").half()
    x, residual, dy, ds = (t.view(B, T, N) for t in (x, residual, dy, ds))
    _check_fwd(x, residual, (w1, w2, gate, b1, b2))
    # (_check_bwd holds d_gate to the gate's own shape, (N,))
    _, _, _, _, dg, _, _ = FusedSandwichNormBwdOp()(dy, ds, x, residual, w1, w2, gate, b1, b2)
    want, tol = ref.sandwich_bwd(*(t.reshape(-1, N) for t in (dy, ds, x, residual)), w1, w2, gate,
                                 b1)
    assert dg.shape == (N,)
    ref.assert_within(dg, want[4][0], tol[4][0], "d_gate")


@pytest.mark.parametrize("N, shift", [(64, 1), (264, 4), (72, 0)])
def test_strides_and_alignment(N, shift):
    wide = torch.randn(10, 4, N + shift, device="cuda").bfloat16()
    x, residual, dy, ds = (wide[:, n, shift:] for n in range(4))
    flat = torch.randn(5 * N + 1, device="cuda")
    w1, w2, g, b1, b2 = (flat[1 + n * N:1 + (n + 1) * N] for n in range(5))
    params = (w1, w2, g.view(1, N), b1, b2)
    _check_fwd(x, residual, params)
    _check_bwd(dy, ds, x, residual, params)
    # contiguous rows that start off a 16-byte boundary
    store = torch.randn(4, 10 * N + 1, device="cuda").bfloat16()
    x, residual, dy, ds = (store[n, 1:].view(10, N) for n in range(4))
    _check_fwd(x, residual, params)
    _check_bwd(dy, ds, x, residual, params)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_rows_far_from_zero(norm):
    """A mean of 300 deviations: the centred variance is taken in two passes."""
    x, residual, dy, ds, params = _inputs(6, 500, torch.float32, torch.float32)
    x, residual = x + 300, residual + 600
    _check_fwd(x, residual, params, norm=norm)
    _check_bwd(dy, ds, x, residual, params, norm=norm)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_rows_of_one_value(norm):
    """Rows without deviation (or of zeros) are divided by sqrt(eps)."""
    x, residual, dy, ds, params = _inputs(4, 256, torch.float32, torch.float32)
    x = torch.zeros_like(x)
    residual[:2] = 0
    _check_fwd(x, residual, params, norm=norm, eps=1e-3)
    _check_bwd(dy, ds, x, residual, params, norm=norm, eps=1e-3)


def test_a_spoiled_row_stays_alone():
    x, residual, dy, ds, params = _inputs(700, 1024, torch.bfloat16, torch.float32)
    y, s = FusedSandwichNormFwdOp()(x, residual, *params)
    bwd = FusedSandwichNormBwdOp()
    dx, dr, *_ = bwd(dy, ds, x, s, *params)
    x2 = x.clone()
    x2[300] = float("nan")
    y2, s2 = FusedSandwichNormFwdOp()(x2, residual, *params)
    dx2, dr2, *grads = bwd(dy, ds, x2, s, *params)
    keep = torch.arange(700, device="cuda") != 300
    for a, b in ((y, y2), (s, s2), (dx, dx2), (dr, dr2)):
        assert torch.equal(a[keep], b[keep])
    assert y2[300].isnan().all() and dx2[300].isnan().all()
    assert grads[0].isnan().all()  # the weight's gradient has the row in its sum


def test_no_rows():
    x, residual, dy, ds, params = _inputs(0, 64, torch.bfloat16, torch.float32)
    y, s = FusedSandwichNormFwdOp()(x, residual, *params)
    assert y.shape == s.shape == (0, 64)
    dx, dr, *grads = FusedSandwichNormBwdOp()(dy, ds, x, residual, *params)
    assert dx.shape == dr.shape == (0, 64) and all((g == 0).all() for g in grads)


def test_deterministic_streams_and_graphs():
    x, residual, dy, ds, params = _inputs(1100, 1024, torch.bfloat16, torch.float32, 4)
    fwd, bwd = FusedSandwichNormFwdOp(norm="layer"), FusedSandwichNormBwdOp(norm="layer")

    def both():
        y, s = fwd(x, residual, *params)
        return y, s, *bwd(dy, ds, x, s, *params)

    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(both())
        graphs.append(g)
    for t in (x, residual, dy, ds):
        t.copy_(torch.randn_like(t))
    want = both()
    for g, out in zip(graphs, outs):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_one_op_in_two_threads():
    """An op object called by two threads, on two streams, with different sizes."""
    from threading import Barrier, Thread

    op, bwd = FusedSandwichNormFwdOp(norm="layer"), FusedSandwichNormBwdOp(norm="layer")
    cases = [_inputs(300, 1024, torch.bfloat16, torch.float32, 3),
             _inputs(7, 264, torch.bfloat16, torch.float32, 7)]

    def both(case):
        x, residual, dy, ds, params = case
        y, s = op(x, residual, *params)
        return y, s, *bwd(dy, ds, x, s, *params)

    want = [both(c) for c in cases]
    torch.cuda.synchronize()
    got, start = [None, None], Barrier(2)

    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for _ in range(50):
                got[n] = both(cases[n])
            torch.cuda.current_stream().synchronize()

    threads = [Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows as in a call of their own."""
    M, N = (1 << 19) + 3, 4104
    x = torch.randn(64, N, device="cuda").bfloat16().repeat(M // 64 + 1, 1)[:M]
    w = torch.ones(N, device="cuda", dtype=torch.bfloat16)
    op = FusedSandwichNormFwdOp()
    y, s = op(x, x, w, w)
    y1, s1 = op(x[-5:], x[-5:], w, w)
    assert torch.equal(y[-5:], y1) and torch.equal(s[-5:], s1)
    dx, dr, dw1, dw2, *_ = FusedSandwichNormBwdOp()(y, None, x, s, w, w)
    dx1, dr1, *_ = FusedSandwichNormBwdOp()(y1, None, x[-5:], s1, w, w)
    assert torch.equal(dx[-5:], dx1) and torch.equal(dr[-5:], dr1)
    assert dw1.isfinite().all() and dw2.isfinite().all()


def test_gradient_against_differences():
    """Central differences of the forward op's own fp32 values along random directions.

    L = <y, dy> + <s, ds> in 64 bits.  The forward's error is bounded by the oracle's bounds
    (E), so the quotient's by E / 2h per end; what the quotient itself is off by (h^2 f''' / 6)
    is measured on the 64-bit oracle and taken off."""
    M, N, h = 6, 200, 1e-2
    x, residual, dy, ds, params = _inputs(M, N, torch.float32, torch.float32, 2)
    kw = dict(norm="layer", eps=1e-5, residual_scale=0.75)
    fwd, bwd = FusedSandwichNormFwdOp(**kw), FusedSandwichNormBwdOp(**kw)
    at = [x, residual, *params]
    _, s = fwd(*at)
    grads = bwd(dy, ds, x, s, *params)
    order = (0, 1, 2, 3, 4, 5, 6)  # dx, d_residual, d_post, d_pre, d_gate, d_post_bias, d_pre_bias
    s64, _ = ref.sandwich_stream(x, residual, params[0], params[2], params[3], **kw)
    want, tol = ref.sandwich_bwd(dy, ds, x, s64, params[0], params[1], params[2], params[3], **kw)

    def loss(y, s):
        return ((y.cpu().double() * dy.cpu()).sum() + (s.cpu().double() * ds.cpu()).sum()).item()

    for n in order:
        way = torch.randn_like(at[n])
        ends, exact, err = [], [], 0.0
        for sign in (1, -1):
            v = list(at)
            v[n] = at[n] + sign * h * way
            ends.append(loss(*fwd(*v)))
            sv, es = ref.sandwich_stream(v[0], v[1], v[2], v[4], v[5], **kw)
            yv, ey = ref.sandwich_next(sv, v[3], v[6], "layer", 1e-5)
            exact.append(loss(yv, sv))
            es = es + ref.U * sv.abs()
            # an error of s moves y by at most rstd |w2| (1 + 1 + |hat| max|hat|) times it
            rstd = 1 / torch.sqrt(sv.var(-1, unbiased=False, keepdim=True) + 1e-5)
            hat = (sv - sv.mean(-1, keepdim=True)) * rstd
            through = rstd * v[3].cpu().abs() * (es + es.mean(-1, keepdim=True) + hat.abs() *
                                                 (hat.abs() * es).mean(-1, keepdim=True))
            err += ((ey + ref.U * yv.abs() + through) * dy.cpu().abs()).sum().item()
            err += (es * ds.cpu().abs()).sum().item()
        slope64 = (want[n].reshape(way.shape) * way.cpu().double()).sum().item()
        slope = (grads[n].cpu().double() * way.cpu().double()).sum().item()
        curve = (exact[0] - exact[1]) / (2 * h) - slope64
        # grads come from the rounded s; half a step of it against s64 through the oracle's bound
        s_moved, _ = ref.sandwich_bwd(dy, ds, x, s, params[0], params[1], params[2], params[3], **kw)
        moved = ((s_moved[n] - want[n]).reshape(way.shape).abs() * way.cpu().abs()).sum().item()
        grad_err = ((tol[n] + ref.U * want[n].abs()).reshape(way.shape)
                    * way.cpu().abs()).sum().item()
        assert abs((ends[0] - ends[1]) / (2 * h) - curve - slope) <= err / (2 * h) + grad_err + moved
