"""GPU parity of the rotary position ops against the 64-bit oracle; values are held to its error
bound plus half a step of their type."""

import pytest
import torch

from oracle import serving_attention as ref
from oracle.recurrent import assert_within
from tileops.ops.attention import RotaryEmbeddingBwdOp, RotaryEmbeddingFwdOp, rotary_frequencies

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _pair(B, S, H, Hkv, D, dtype):
    return (torch.randn(B, S, H, D, device="cuda").to(dtype),
            torch.randn(B, S, Hkv, D, device="cuda").to(dtype))


def _check(q, k, positions=None, rotary_dim=None, interleaved=False, frequencies=None,
           amplitude=1.0, inplace=False):
    B, S, H, D = q.shape
    r = D if rotary_dim is None else rotary_dim
    f = rotary_frequencies(r) if frequencies is None else frequencies
    at = torch.arange(S) if positions is None else positions
    if at.dim() == 1:
        at = at.expand(B, S)
    k = k if k.shape[2] else None
    for cls, back in ((RotaryEmbeddingFwdOp, False), (RotaryEmbeddingBwdOp, True)):
        op = cls(B, S, H, 0 if k is None else k.shape[2], D, rotary_dim, interleaved, frequencies, amplitude, q.dtype,
                 inplace)
        ins = [t.clone(memory_format=torch.preserve_format) if inplace and t is not None else t
               for t in (q, k)]
        got = op(*ins, positions)
        if inplace:
            assert got[0] is ins[0] and got[1] is ins[1]
        for name, g, t in zip("qk", got, (q, k)):
            if t is None:
                assert g is None
                continue
            assert g.dtype == t.dtype and (inplace or g.is_contiguous())
            assert_within(g, *ref.rotate(t, at, f, amplitude, interleaved, back), name)
            assert torch.equal(g[..., r:], t[..., r:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B, S, H, Hkv, D, R", [
    (1, 1, 1, 1, 2, 2), (1, 1, 32, 8, 128, 128), (2, 7, 4, 2, 64, 64), (1, 33, 3, 1, 80, 80),
    (2, 5, 2, 2, 72, 36), (1, 130, 5, 1, 96, 24), (3, 17, 2, 1, 33, 6), (1, 9, 1, 3, 35, 34),
    (1, 9, 3, 1, 128, 30), (2, 6, 2, 1, 40, 34), (1, 20, 5, 2, 60, 38), (1, 3, 30, 2, 256, 108),
    (1, 5, 40, 8, 128, 98), (2, 1, 1, 1, 8, 2), (1, 70, 1, 0, 16, 6),
    (2, 3, 40, 1, 256, 256), (1, 11, 2, 1, 576, 64), (5, 4, 1, 1, 40, 20), (1, 6, 2, 2, 64, 0),
])
def test_sizes(B, S, H, Hkv, D, R, interleaved, dtype):
    _check(*_pair(B, S, H, Hkv, D, dtype), rotary_dim=R, interleaved=interleaved)


@pytest.mark.parametrize("S, H, D, R", [(4096, 4, 128, 128), (1500, 33, 64, 64), (700, 128, 128, 128),
                                        (2500, 7, 64, 22), (900, 70, 40, 34), (3000, 1, 16, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_more_tokens_than_ctas(S, H, D, R, interleaved):
    _check(*_pair(1, S, H, 1, D, torch.bfloat16), rotary_dim=R, interleaved=interleaved)


def test_the_same_bits_whatever_the_words():
    """Dense rows, slices that allow words of 8, 4 and 2 bytes only, and a head with channels to
    spare (partners through shared memory) are rotated by the same operations."""
    B, S, H, D = 2, 50, 5, 64
    for R, interleaved in ((64, False), (64, True), (32, False), (12, False), (22, False), (22, True)):
        q = torch.randn(B, S, H, D, device="cuda").to(torch.bfloat16)
        op = RotaryEmbeddingFwdOp(B, S, H, 0, D, R, interleaved)
        want, _ = op(q, None)
        for at in (0, 4, 2, 1):
            wide = torch.empty(B, S, H, D + 8, device="cuda", dtype=torch.bfloat16)
            t = wide[..., at:at + D]
            t.copy_(q)
            assert torch.equal(op(t, None)[0], want), (R, interleaved, at)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("batched", [False, True])
def test_positions(batched, dtype):
    """Far, negative, repeated and unordered positions."""
    at = torch.tensor([0, 1, -1, 5, 5, 2**20 + 1, 2**31 - 1, -(2**31), 123456789, 7], dtype=dtype)
    if dtype is torch.int64:
        at[-1] = 2**33 + 5
    at = at.cuda()
    if batched:
        at = torch.stack([at, at.flip(0)])
    _check(*_pair(2, 10, 3, 2, 64, torch.float32), positions=at)


def test_positions_of_any_layout():
    at = torch.randint(0, 1 << 20, (20, 4), device="cuda")
    q, k = _pair(4, 20, 2, 1, 64, torch.float32)
    _check(q, k, positions=at.t())
    _check(q, k, positions=at[:, 1])
    _check(q, k, positions=at[:, :1].t().expand(4, 20))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scaled_frequencies_and_amplitude(dtype):
    f = rotary_frequencies(64, 500000.0, factor=8.0, original_length=8192, fast_turns=4.0)
    _check(*_pair(2, 40, 3, 1, 64, dtype), frequencies=f, amplitude=1.25)
    f = rotary_frequencies(64, factor=4.0)
    _check(*_pair(2, 40, 3, 1, 64, dtype), frequencies=f, amplitude=-0.5, interleaved=True)
    any_angles = [-3.0, 0.0, 1e-30, 100.0]  # backwards, none, more than a turn a token
    _check(*_pair(2, 40, 3, 1, 64, dtype), rotary_dim=8, frequencies=any_angles)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D, inner", [(64, 0), (64, 1), (64, 2), (64, 4), (60, 0), (50, 0)])
def test_column_slices_in_place_and_not(D, inner, interleaved, dtype):
    """Slices of one projection's output, at offsets that allow wider or narrower words."""
    B, S, H, Hkv = 2, 19, 3, 2
    wide = torch.randn(B, S, (H + 2 * Hkv) * D + inner, device="cuda").to(dtype)
    keep = wide.clone()
    q = wide[..., inner:inner + H * D].unflatten(-1, (H, D))
    k = wide[..., inner + H * D:inner + (H + Hkv) * D].unflatten(-1, (Hkv, D))
    r = D // 2 // 2 * 2
    _check(q, k, rotary_dim=r, interleaved=interleaved)
    f = rotary_frequencies(r)
    want = [ref.rotate(t, torch.arange(S).expand(B, S), f, interleaved=interleaved) for t in (q, k)]
    op = RotaryEmbeddingFwdOp(B, S, H, Hkv, D, r, interleaved, dtype=dtype, inplace=True)
    op(q, k)
    assert_within(q, *want[0], "q")
    assert_within(k, *want[1], "k")
    cols = torch.ones(wide.shape[-1], dtype=torch.bool)
    cols[inner:inner + (H + Hkv) * D] = False
    assert torch.equal(wide[..., cols.cuda()], keep[..., cols.cuda()])  # all else is as it was


def test_heads_before_tokens_and_spread_channels():
    q, k = (t.transpose(1, 2) for t in _pair(2, 3, 21, 21, 64, torch.bfloat16))  # (2, 21, 3, 64)
    _check(q, k)
    _check(q, k, inplace=True)
    q, k = (torch.randn(2, 64, 3, 21, device="cuda").permute(0, 3, 2, 1) for _ in range(2))
    _check(q, k)


def test_broadcast_inputs():
    q = torch.randn(1, 8, 1, 64, device="cuda").expand(3, 8, 5, 64)
    _check(q, q[:, :, :2])


@pytest.mark.parametrize("cls", [RotaryEmbeddingFwdOp, RotaryEmbeddingBwdOp])
def test_queries_or_keys_alone_and_none(cls):
    q, _ = _pair(2, 9, 3, 1, 64, torch.float32)
    want = ref.rotate(q, torch.arange(9).expand(2, 9), rotary_frequencies(64),
                      backward=cls is RotaryEmbeddingBwdOp)
    got, none = cls(2, 9, 3, 0, 64, dtype=torch.float32)(q, None)
    assert none is None
    assert_within(got, *want)
    none, got = cls(2, 9, 0, 3, 64, dtype=torch.float32)(None, q)
    assert none is None
    assert_within(got, *want)
    empty = torch.empty(2, 0, 3, 64, device="cuda")
    a, b = cls(2, 0, 3, 3, 64, dtype=torch.float32)(empty, empty)
    assert a.shape == b.shape == (2, 0, 3, 64)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_pair(bad):
    q, k = _pair(1, 12, 4, 1, 64, torch.bfloat16)
    op = RotaryEmbeddingFwdOp(1, 12, 4, 1, 64)
    clean = op(q, k)[0]
    q[0, 5, 2, 7] = bad
    got = op(q, k)[0]
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[0, 5, 2, [7, 39]] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()


def test_gradient_is_the_transposed_map():
    """<R q, d> = <q, R^T d>, and the gradient of a sum against differences of the op itself: the
    map is linear, so a difference of any step is exact up to rounding."""
    q, k = _pair(1, 6, 2, 1, 32, torch.float32)
    d, _ = _pair(1, 6, 2, 1, 32, torch.float32)
    at = torch.randint(0, 1 << 20, (6,), device="cuda")
    args = dict(rotary_dim=20, amplitude=1.5, dtype=torch.float32)
    fwd, bwd = RotaryEmbeddingFwdOp(1, 6, 2, 1, 32, **args), RotaryEmbeddingBwdOp(1, 6, 2, 1, 32, **args)
    grad = bwd(d, k, at)[0].double()
    for n in range(0, q.numel(), 5):
        up, down = q.clone(), q.clone()
        up.view(-1)[n] += 1.0
        down.view(-1)[n] -= 1.0
        step = (up.view(-1)[n] - down.view(-1)[n]).double()
        diff = ((fwd(up, k, at)[0].double() - fwd(down, k, at)[0].double()) * d.double()).sum() / step
        # Two channels differ, each of at most 1.5 * 2 * 6 off by 9 u, times d below 6: 1e-4.
        assert abs(diff - grad.view(-1)[n]) < 1e-4


def test_captured_and_replayed():
    q, k = _pair(2, 30, 4, 2, 64, torch.bfloat16)
    at = torch.zeros(2, 30, dtype=torch.int32, device="cuda")
    op = RotaryEmbeddingFwdOp(2, 30, 4, 2, 64)
    op(q, k, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, k, at)
    for start in (5, 1 << 19):
        at.copy_(torch.arange(30, device="cuda") + start)
        q.normal_()
        graph.replay()
        assert_within(got[0], *ref.rotate(q, at, rotary_frequencies(64)))


def test_another_stream():
    q, k = _pair(2, 500, 8, 2, 64, torch.bfloat16)
    op = RotaryEmbeddingFwdOp(2, 500, 8, 2, 64)
    want = op(q, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = op(q, k)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits():
    """Rows more than 2^32 elements apart."""
    far = torch.empty(2**32 + 4096, dtype=torch.float16, device="cuda")
    q = far.as_strided((2, 3, 2, 64), (2**32, 256, 64, 1))
    q.normal_()
    _check(q, q[:, :, :1])
    op = RotaryEmbeddingFwdOp(2, 3, 2, 0, 64, dtype=torch.float16, inplace=True)
    want = ref.rotate(q, torch.arange(3).expand(2, 3), rotary_frequencies(64))
    op(q, None)
    assert_within(q, *want)
