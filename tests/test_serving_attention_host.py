"""Host side of the rotary and paged-cache ops: the 64-bit oracle against differences and against
itself by another route, refusals before any launch, roofline formulas, the C entry points'
argument checks.  CPU only."""

import ctypes
import math
from fractions import Fraction

import pytest
import torch

from oracle import serving_attention as ref
from tileops import _native
from tileops.benchmark.msprof import _extract_op_init_args
from tileops.kernels.attention import (
    PagedAttentionDecodeKernel,
    PagedKVAppendKernel,
    RotaryEmbeddingBwdKernel,
    RotaryEmbeddingFwdKernel,
)
from tileops.kernels.attention._layouts import Layouts, layout_of, overlaps
from tileops.kernels.attention.rotary_embedding import turns_array
from tileops.kernels.kernel_base import Kernel
from tileops.manifest import load_workloads
from tileops.ops.attention import (
    PagedAttentionDecodeOp,
    PagedKVAppendOp,
    RotaryEmbeddingBwdOp,
    RotaryEmbeddingFwdOp,
    rotary_frequencies,
)

NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(1 << 20)  # never read: every call here fails its checks before a launch


# ------------------------------------------------------------ the oracle
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_gradient_against_differences(interleaved):
    f = rotary_frequencies(6)
    x, d = (torch.randn(3, 2, 8, dtype=torch.float64) for _ in range(2))
    at = torch.tensor([0, 5, -3])
    grad, _ = ref.rotate(d, at, f, 1.5, interleaved, backward=True)

    def loss():
        return (ref.rotate(x, at, f, 1.5, interleaved)[0] * d).sum().item()

    for n in range(x.numel()):
        flat, keep = x.view(-1), x.view(-1)[n].item()
        flat[n] = keep + 0.5
        up = loss()
        flat[n] = keep - 0.5
        # A linear map: the difference is exact but for rounding, 2^-53 of sums below 100.
        assert abs((up - loss()) - grad.view(-1)[n].item()) < 1e-12
        flat[n] = keep


def test_rotation_keeps_lengths_and_relative_positions():
    f = rotary_frequencies(32)
    q, k = (torch.randn(1, 32, dtype=torch.float64) for _ in range(2))

    def score(p, r):
        a, _ = ref.rotate(q[None], torch.tensor([p]), f)
        b, _ = ref.rotate(k[None], torch.tensor([r]), f)
        return (a * b).sum().item()

    assert abs(score(7, 3) - score(1000007, 1000003)) < 1e-9
    a, _ = ref.rotate(q[None], torch.tensor([12345]), f)
    assert abs(a.norm() - q.norm()) < 1e-12


def test_angles_of_far_positions_lose_nothing():
    """Against 64-bit products where those are exact enough, and by whole turns where not."""
    f = rotary_frequencies(16)
    near = torch.arange(-500, 500)
    want = near[:, None].double() * torch.tensor(f, dtype=torch.float64)
    off = (torch.sin(ref.angles(near, f)) - torch.sin(want)).abs().max()
    assert off < 1e-12
    turn = [math.tau]  # math.tau is 2 pi less 2.45e-16: a million turns are 2.45e-10 off
    assert (torch.sin(ref.angles(torch.tensor([10**6]), turn)) + 2.4492935982947064e-10).abs() < 1e-15


def test_attention_oracle_against_torch():
    B, H, Hkv, D, P = 2, 4, 2, 16, 4
    k, v = (torch.randn(2, 12, Hkv, D, dtype=torch.float64) for _ in range(2))
    q = torch.randn(B, H, D, dtype=torch.float64)
    table = torch.tensor([[2, 0, 5], [1, 3, 4]])
    kc, vc = (torch.full((6, P, Hkv, D), math.nan, dtype=torch.float64) for _ in range(2))
    lens = torch.tensor([11, 5])
    for b in range(B):
        for t in range(int(lens[b])):
            kc[table[b, t // P], t % P], vc[table[b, t // P], t % P] = k[b, t], v[b, t]
    o, lse, _, _ = ref.attend(q, kc, vc, table, lens, window=6)
    for b in range(B):
        n, first = int(lens[b]), max(0, int(lens[b]) - 6)
        for h in range(H):
            s = k[b, first:n, h // 2] @ q[b, h] / D**0.5
            torch.testing.assert_close(o[b, h], torch.softmax(s, 0) @ v[b, first:n, h // 2])
            torch.testing.assert_close(lse[b, h], torch.logsumexp(s, 0) / math.log(2))


def test_append_oracle_positions_and_padding():
    kc, vc = torch.zeros(3, 4, 1, 2), torch.zeros(3, 4, 1, 2)
    k = torch.arange(1.0, 7.0).repeat_interleave(2).view(6, 1, 2)
    table = torch.tensor([[2, -1], [0, 1]])
    cu = torch.tensor([0, 3, 5])
    _, _, got, bound, values = ref.append(k, -k, kc, vc, table, torch.tensor([2, 6]), cu_seqlens=cu)
    want = torch.zeros(3, 4)
    want[2, 0], want[2, 1] = 2, 3  # row 0 has position -1: padding; row 5 lies behind the last
    want[1, 0], want[1, 1] = 4, 5
    assert torch.equal(got[..., 0, 0], want.double()) and torch.equal(values, -got)
    assert not bound.any()


# ------------------------------------------------------------ frequencies
def test_frequencies():
    f = rotary_frequencies(8)
    assert f == pytest.approx((1.0, 0.1, 0.01, 0.001), rel=1e-15)
    assert rotary_frequencies(8, factor=4.0) == pytest.approx([x / 4 for x in f], rel=1e-15)
    g = rotary_frequencies(8, factor=4.0, original_length=1000, slow_turns=1.0, fast_turns=32.0)
    turns = [1000 * x / math.tau for x in f]  # 159, 15.9, 1.59, 0.159
    kept = [1.0, (turns[1] - 1) / 31, (turns[2] - 1) / 31, 0.0]
    assert g == pytest.approx([x * (r + (1 - r) / 4) for x, r in zip(f, kept)], rel=1e-15)
    assert rotary_frequencies(0) == ()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, base=math.inf), dict(rotary_dim=8, factor=0.0),
                dict(rotary_dim=8, factor=math.nan), dict(rotary_dim=8, original_length=0),
                dict(rotary_dim=8, original_length=9, slow_turns=2.0, fast_turns=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_turns_are_rounded_once():
    f = rotary_frequencies(64, 500000.0) + (0.0, -1.0, 1e-30, 100.0, 1e15)
    exact = [round(Fraction(x) * ref._TURNS_PER_RADIAN * 2**64) % 2**64 for x in f]
    assert list(turns_array(f)) == exact


# ------------------------------------------------------------ layouts
def test_overlaps():
    t = torch.empty(4, 6, 8)
    for fine in (t, t.transpose(0, 2), t[:, ::2, 1:], t[:1].expand(1, 6, 8), t.permute(2, 0, 1)):
        assert not overlaps(fine.shape, fine.stride())
    for bad in (t[:1].expand(3, 6, 8), t.as_strided((4, 4), (1, 1)), t.as_strided((3, 5), (4, 1))):
        assert overlaps(bad.shape, bad.stride())


def test_layouts_are_values():
    """Another tensor of the same layout has the same one; whatever differs shows."""
    a, b = torch.empty(2, 3, 4), torch.empty(2, 3, 4)
    assert layout_of(a, None) == layout_of(b, None)
    for other in (a.half(), a.transpose(0, 1), a.expand(2, 3, 4)[:1], torch.empty(2, 4, 3)):
        assert layout_of(a) != layout_of(other)
    assert layout_of("no tensor") is None and layout_of(a, 3) is None
    kept = Layouts()
    for n in range(1000):
        kept.keep((n,), n)
    assert len(kept) <= 256 and kept.get((999,)) == 999
    kept.keep(None, 5)
    assert kept.get(None) is None


# ------------------------------------------------------------ refusals
class _AcceptCpu:
    name = "cuda"

    def is_device_tensor(self, t):
        return isinstance(t, torch.Tensor)

    def is_available(self):
        return False


@pytest.fixture
def accept_cpu(monkeypatch):
    """Admit CPU tensors so the later checks run here; every case raises before a launch."""
    import tileops.ops.attention._arguments as arguments
    import tileops.ops.attention.paged_attention as paged
    import tileops.ops.attention.rotary_embedding as rotary

    fake = _AcceptCpu()
    for mod in (arguments, paged, rotary):
        monkeypatch.setattr(mod, "get_device_backend", lambda: fake)


def _rotary_args(B=2, S=5, H=4, Hkv=2, D=8, dtype=torch.float32):
    return torch.randn(B, S, H, D).to(dtype), torch.randn(B, S, Hkv, D).to(dtype)


@pytest.mark.parametrize("cls, names", [(RotaryEmbeddingFwdOp, "q"), (RotaryEmbeddingBwdOp, "dq")])
def test_rotary_refusals(cls, names, accept_cpu):
    op = cls(2, 5, 4, 2, 8, dtype=torch.float32)
    q, k = _rotary_args()
    with pytest.raises(ValueError, match="must be on a cuda device"):  # all checks passed
        op(q, k)
    with pytest.raises(ValueError, match=rf"Expected {names}.shape \(2, 5, 4, 8\)"):
        op(q[:, :4], k)
    with pytest.raises(ValueError, match=rf"Expected {names}.dtype"):
        op(q.half(), k)
    with pytest.raises(ValueError, match="shape"):
        op(q, q)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        op(q, None)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        op(q.tolist(), k)
    for at, match in ((torch.zeros(4, dtype=torch.int32), "positions.shape"),
                      (torch.zeros(5, 2, dtype=torch.int32), "positions.shape"),
                      (torch.zeros(5), "int32 or int64"), ([0] * 5, "must be a cuda tensor")):
        with pytest.raises(ValueError, match=match):
            op(q, k, at)


def test_rotary_in_place_refusals(accept_cpu):
    op = RotaryEmbeddingFwdOp(2, 5, 4, 4, 8, dtype=torch.float32, inplace=True)
    q, k = _rotary_args(Hkv=4)
    with pytest.raises(ValueError, match="share memory"):
        op(q[:1].expand(2, 5, 4, 8), k)
    with pytest.raises(ValueError, match="contiguous channels"):
        op(torch.randn(2, 5, 8, 4).transpose(2, 3), k)
    with pytest.raises(ValueError, match="q and k share memory"):
        op(q, q)
    with pytest.raises(ValueError, match="must be on a cuda device"):
        op(q, k)


@pytest.mark.parametrize("cls", [RotaryEmbeddingFwdOp, RotaryEmbeddingBwdOp])
def test_rotary_rejects_sizes_and_types_at_construction(cls):
    with pytest.raises(ValueError, match="only supports dtypes"):
        cls(1, 4, 2, 2, 8, dtype=torch.float64)
    with pytest.raises(ValueError, match="rotary_dim"):
        cls(1, 4, 2, 2, 8, rotary_dim=7)
    with pytest.raises(ValueError, match="rotary_dim"):
        cls(1, 4, 2, 2, 8, rotary_dim=10)
    with pytest.raises(ValueError, match="rotary_dim"):
        cls(1, 4, 2, 2, 512)
    with pytest.raises(ValueError, match="frequencies must have"):
        cls(1, 4, 2, 2, 8, frequencies=[1.0] * 3)
    for f in (math.nan, math.inf, 1e20):
        with pytest.raises(ValueError, match="frequencies must be finite"):
            cls(1, 4, 2, 2, 8, frequencies=[1.0, 1.0, 1.0, f])
    for amplitude in (math.nan, math.inf, 1e39):
        with pytest.raises(ValueError, match="amplitude"):
            cls(1, 4, 2, 2, 8, amplitude=amplitude)
    for size in ((-1, 4, 2, 2, 8), (1, -1, 2, 2, 8), (1, 4, -1, 2, 8), (1, 4, 2, 5000, 8),
                 (1, 4, 2, 2, 0), (1, 4, 2, 2, 5000), (2**31, 1, 1, 1, 8), (2**16, 2**15, 1, 1, 8)):
        with pytest.raises(ValueError, match="supports"):
            cls(*size, rotary_dim=0)


def test_rejects_cpu_tensors():
    q, k = _rotary_args()
    with pytest.raises(ValueError, match="q must be a cuda tensor"):
        RotaryEmbeddingFwdOp(2, 5, 4, 2, 8, dtype=torch.float32)(q, k)
    with pytest.raises(ValueError, match="dq must be a cuda tensor"):
        RotaryEmbeddingBwdOp(2, 5, 4, 2, 8, dtype=torch.float32)(q, k)
    c = torch.zeros(3, 4, 2, 8)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="k must be a cuda tensor"):
        PagedKVAppendOp(2, 8, 4, dtype=torch.float32)(k[:, 0], k[:, 0], c, c, table, lens)
    with pytest.raises(ValueError, match="q must be a cuda tensor"):
        PagedAttentionDecodeOp(4, 2, 8, 4, dtype=torch.float16)(q[:, 0].half(), c, c, table, lens)


def _paged(dtype, B=2, H=4, Hkv=2, D=8, P=4, pages=3):
    c = torch.zeros(2, pages, P, Hkv, D, dtype=dtype)
    return dict(k=torch.zeros(B, Hkv, D, dtype=dtype), v=torch.zeros(B, Hkv, D, dtype=dtype),
                q=torch.zeros(B, H, D, dtype=dtype), k_cache=c[0], v_cache=c[1],
                page_table=torch.zeros(B, 3, dtype=torch.int32),
                seq_lens=torch.ones(B, dtype=torch.int32))


COMMON = [
    (dict(k_cache=torch.zeros(3, 4, 2, 8)[..., :4]), "k_cache.shape"),
    (dict(k_cache=torch.zeros(3, 4, 16)), "k_cache must have 4 dimensions"),
    (dict(v_cache=torch.zeros(2, 4, 2, 8)), "v_cache.shape"),
    (dict(v_cache=torch.zeros(3, 4, 2, 8, dtype=torch.float64)), "v_cache.dtype"),
    (dict(k_cache=torch.zeros(0, 4, 2, 8), v_cache=torch.zeros(0, 4, 2, 8)), "between 1 and"),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), "page_table.shape"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), "page_table.dtype"),
    (dict(page_table=torch.zeros(6, dtype=torch.int32)), "page_table must have 2 dimensions"),
    (dict(page_table=None), "page_table must be a cuda tensor"),
    (dict(seq_lens=torch.ones(3, dtype=torch.int32)), "seq_lens.shape"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int64)), "seq_lens.dtype"),
    (dict(seq_lens=[1, 1]), "seq_lens must be a cuda tensor"),
]


def _cast(change, dtype):
    return {k: v.to(dtype) if isinstance(v, torch.Tensor) and v.dtype is torch.float32 else v
            for k, v in change.items()}


@pytest.mark.parametrize("change, match", COMMON + [
    (dict(k=torch.zeros(2, 3, 8)), "k.shape"), (dict(v=torch.zeros(3, 2, 8)), "v.shape"),
    (dict(v=torch.zeros(2, 2, 8, dtype=torch.float64)), "v.dtype"), (dict(k=torch.zeros(2, 16)), "k must be"),
    (dict(q=torch.zeros(2, 3, 8)), "q.shape"), (dict(q=torch.zeros(3, 4, 8)), "q.shape"),
    (dict(cu_seqlens=torch.tensor([0, 2])), "cu_seqlens.dtype"),
    (dict(cu_seqlens=torch.tensor([[0, 1, 2]], dtype=torch.int32)), "cu_seqlens.shape"),
    (dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), "at least one offset"),
    (dict(cu_seqlens=torch.tensor([0, 2], dtype=torch.int32)), "page_table.shape"),
    (dict(cu_seqlens=[0, 1, 2]), "cu_seqlens must be a cuda tensor"),
    (dict(k=torch.zeros(2, 1, 2, 8), v=torch.zeros(2, 1, 2, 8), q=None,
          cu_seqlens=torch.tensor([0, 1, 2], dtype=torch.int32)), "must be packed"),
    (dict(k_cache=torch.zeros(1, 4, 2, 8).expand(3, 4, 2, 8)), "share memory"),
    ((lambda c: dict(k_cache=c, v_cache=c))(torch.zeros(3, 4, 2, 8)), "k_cache and v_cache share memory"),
    (dict(v_cache=torch.zeros(3, 4, 8, 2).transpose(2, 3)), "contiguous channels"),
])
def test_append_refusals(change, match, accept_cpu):
    op = PagedKVAppendOp(2, 8, 4, 4, 8, dtype=torch.float32)
    args = _paged(torch.float32)
    with pytest.raises(ValueError, match="must be on a cuda device"):
        op(**args)
    with pytest.raises(ValueError, match=match):
        op(**{**args, **change})


@pytest.mark.parametrize("change, match", COMMON + [
    (dict(q=torch.zeros(2, 3, 8)), "q.shape"), (dict(q=torch.zeros(2, 4, 1, 8)), "q.shape"),
    (dict(q=torch.zeros(2, 4, 8, dtype=torch.float64)), "q.dtype"), (dict(q=None), "q must be a cuda tensor"),
    (dict(page_table=torch.zeros(2, 1, dtype=torch.int32).expand(2, 2**29)), "at most 2\\^31 - 129"),
    (dict(k_cache=torch.zeros(3, 4, 2, 12, dtype=torch.float16)[..., :8]), "multiples of 8"),
    (dict(v_cache=torch.zeros(3, 4, 8, 2).transpose(2, 3)), "contiguous channels"),
])
def test_decode_refusals(change, match, accept_cpu):
    op = PagedAttentionDecodeOp(4, 2, 8, 4, dtype=torch.float16)
    args = _paged(torch.float16)
    del args["k"], args["v"]
    with pytest.raises(ValueError, match="must be on a cuda device"):
        op(**args)
    with pytest.raises(ValueError, match=match):
        op(**{**args, **_cast(change, torch.float16)})


def test_paged_ops_reject_sizes_and_types_at_construction():
    for bad in (dict(heads_kv=0), dict(dim=0), dict(page_size=0), dict(heads=-1), dict(dim=5000),
                dict(rotary_dim=10), dict(rotary_dim=3), dict(frequencies=[1.0]),
                dict(dtype=torch.int32), dict(amplitude=math.nan)):
        with pytest.raises(ValueError):
            PagedKVAppendOp(**{**dict(heads_kv=2, dim=8, page_size=4), **bad})
    for bad in (dict(heads=3), dict(heads_kv=0), dict(dim=12), dict(dim=264), dict(dim=0),
                dict(page_size=0), dict(page_size=2**31), dict(scale=math.inf), dict(scale=math.nan),
                dict(window=0), dict(window=-1), dict(window=2**31), dict(dtype=torch.float32),
                dict(heads=8192, heads_kv=1)):
        with pytest.raises(ValueError):
            PagedAttentionDecodeOp(**{**dict(heads=4, heads_kv=2, dim=8, page_size=4), **bad})


def test_kernel_maps():
    for op, key, cls in (
            (RotaryEmbeddingFwdOp(1, 1, 1, 1, 8), "rotary_fwd", RotaryEmbeddingFwdKernel),
            (RotaryEmbeddingBwdOp(1, 1, 1, 1, 8), "rotary_bwd", RotaryEmbeddingBwdKernel),
            (PagedKVAppendOp(1, 8, 4), "paged_kv_append", PagedKVAppendKernel),
            (PagedAttentionDecodeOp(1, 1, 8, 4), "paged_attention_decode", PagedAttentionDecodeKernel)):
        assert op.default_kernel_map == {key: cls} and type(op.kernel) is cls


def test_kernel_overrides_need_a_forward_only(accept_cpu):
    """What a kernel_map puts in a kernel's place gets the op's arguments, after its checks."""
    seen = []

    class Other(Kernel):
        def __init__(self, *args):
            super().__init__()

        def forward(self, *args):
            seen.append(args)
            return "done"

    q, k = _rotary_args()
    op = RotaryEmbeddingFwdOp(2, 5, 4, 2, 8, dtype=torch.float32, kernel_map={"rotary_fwd": Other})
    for _ in range(2):
        assert op(q, k) == "done" and seen.pop() == (q, k, None, False)
    with pytest.raises(ValueError, match="q.shape"):
        op(q[:1], k)
    args = _paged(torch.float16)
    op = PagedKVAppendOp(2, 8, 4, 4, dtype=torch.float16, kernel_map={"paged_kv_append": Other})
    assert op(**args) == "done" and seen.pop()[6] is args["q"]
    del args["k"], args["v"]
    op = PagedAttentionDecodeOp(4, 2, 8, 4, dtype=torch.float16,
                                kernel_map={"paged_attention_decode": Other})
    assert op(**args) == "done" and len(seen.pop()) == 5


# ------------------------------------------------------------ C entry points
def _ints(*values):
    return (ctypes.c_int64 * len(values))(*values)


def test_rotary_entry_point_checks():
    fn = _native.lib().tileops_rotary
    turns = (ctypes.c_uint64 * 128)()
    s = _ints(*[0] * 12)

    def call(q=SOME, k=SOME, at=NULL, out=SOME, t=turns, B=1, S=4, H=2, Hkv=1, D=8, R=8, st=s, at_type=7,
             dtype=2):
        return fn(q, k, at, out, out, t, B, S, H, Hkv, D, R, st, 0, at_type, 0, 0, 1.0, dtype, NULL)

    for bad in (dict(B=-1), dict(S=-1), dict(H=-1), dict(H=5000), dict(D=0), dict(D=5000), dict(R=7),
                dict(R=10), dict(R=-2), dict(D=512, R=258), dict(B=2**16, S=2**15)):
        assert call(**bad) == _native.EBADSHAPE, bad
    assert call(dtype=7) == _native.EBADDTYPE and call(at=SOME, at_type=0) == _native.EBADDTYPE
    for bad in (dict(q=NULL), dict(k=NULL), dict(out=NULL), dict(st=None), dict(t=None)):
        assert call(**bad) == _native.EINVAL, bad
    assert call(q=NULL, k=NULL, B=0) == _native.OK and call(q=NULL, k=NULL, H=0, Hkv=0) == _native.OK


def test_append_entry_point_checks():
    fn = _native.lib().tileops_paged_kv_append
    turns = (ctypes.c_uint64 * 128)()
    s = _ints(*[0] * 18)

    def call(q=SOME, k=SOME, v=SOME, c=SOME, vc=ctypes.c_void_p(1 << 21), table=SOME, lens=SOME, cu=NULL,
             t=turns, N=2, T=4, H=2, Hkv=1, D=8, R=8, pages=3, P=4, width=2, st=s, dtype=2):
        return fn(q, k, v, q, c, vc, table, lens, cu, t, N, T, H, Hkv, D, R, pages, P, width, width, st,
                  0, 1.0, dtype, NULL)

    for bad in (dict(N=-1), dict(T=-1), dict(T=5), dict(N=0), dict(H=-1), dict(Hkv=0), dict(D=0),
                dict(R=9), dict(pages=-1), dict(pages=2**31), dict(P=0), dict(P=2**31), dict(width=-1)):
        assert call(**bad) == _native.EBADSHAPE, bad
    assert call(dtype=3) == _native.EBADDTYPE
    for bad in (dict(q=NULL), dict(k=NULL), dict(v=NULL), dict(c=NULL), dict(vc=NULL), dict(vc=SOME),
                dict(table=NULL), dict(lens=NULL), dict(t=None), dict(st=None)):
        assert call(**bad) == _native.EINVAL, bad
    assert call(q=NULL, k=NULL, N=0, T=0) == _native.OK


def test_decode_entry_point_checks():
    lib = _native.lib()
    fn = lib.tileops_paged_decode_fwd

    def call(q=SOME, c=SOME, table=SOME, lens=SOME, out=SOME, ws=SOME, B=2, H=4, Hkv=2, D=8, pages=3, P=4,
             width=2, st=_ints(*[8] * 8), window=0, dtype=2):
        return fn(q, c, c, table, lens, out, out, ws, B, H, Hkv, D, pages, P, width, width, st, window,
                  0, 1.0, dtype, NULL)

    for bad in (dict(B=-1), dict(H=3), dict(H=0), dict(Hkv=0), dict(D=12), dict(D=264), dict(D=0),
                dict(pages=-1), dict(P=0), dict(P=2**30, width=2), dict(width=-1), dict(window=-1)):
        assert call(**bad) == _native.EBADSHAPE, bad
    # 2^31 and more units of 32 tokens
    assert call(B=2**20, H=32, Hkv=32, P=64, width=2**10) == _native.EBADSHAPE
    assert call(dtype=0) == _native.EBADDTYPE and call(dtype=7) == _native.EBADDTYPE
    for bad in (dict(q=NULL), dict(c=NULL), dict(table=NULL), dict(lens=NULL), dict(out=NULL),
                dict(ws=NULL), dict(st=None)):
        assert call(**bad) == _native.EINVAL, bad
    off = ctypes.c_void_p((1 << 20) + 8)
    for bad in (dict(q=off), dict(c=off), dict(ws=off), dict(st=_ints(*[8] * 7, 4))):
        assert call(**bad) == _native.EALIGN, bad
    assert call(q=NULL, c=NULL, B=0) == _native.OK
    assert lib.tileops_paged_decode_workspace_bytes(4, 3, 8) == -1
    assert lib.tileops_paged_decode_workspace_bytes(4, 2, 12) == -1
    # counters, then (exponent, sum) and sums of 2 x 2 rows for each of 592 CTAs
    assert lib.tileops_paged_decode_workspace_bytes(4, 2, 64) == 592 * 4 + 592 * 2 * 2 * (2 + 64) * 4
    assert lib.tileops_paged_decode_workspace_bytes(32, 1, 72) == 592 * 4 + 592 * 2 * 32 * (2 + 80) * 4


# ------------------------------------------------------------ formulas, manifest
def test_rooflines():
    assert RotaryEmbeddingFwdOp(2, 10, 4, 2, 64, 32).eval_roofline() == (
        3 * 20 * 6 * 32, 2 * 20 * 6 * 64 * 2)
    assert RotaryEmbeddingBwdOp(2, 10, 4, 2, 64, dtype=torch.float32).eval_roofline() == (
        3 * 20 * 6 * 64, 2 * 20 * 6 * 64 * 4)
    op = PagedKVAppendOp(2, 64, 16, 4, 64)
    assert op.eval_roofline() == (0, 0)
    op._last = (7, 2, 64), True
    assert op.eval_roofline() == (3 * 7 * 6 * 64, 2 * 7 * 8 * 64 * 2)
    op._last = (3, 7, 2, 64), False
    assert op.eval_roofline() == (3 * 21 * 2 * 64, 2 * 21 * 4 * 64 * 2)
    op = PagedAttentionDecodeOp(8, 2, 64, 16)
    op._last = (3, 5)
    assert op.eval_roofline() == (4 * 3 * 8 * 64 * 80, (2 * 3 * 80 * 2 * 64 + 2 * 3 * 8 * 64) * 2 + 4 * 24)
    op = PagedAttentionDecodeOp(8, 2, 64, 16, window=10)
    op._last = (3, 5)
    assert op.eval_roofline()[0] == 4 * 3 * 8 * 64 * 10


def test_manifest_has_the_serving_ops():
    for row in load_workloads("RotaryEmbeddingFwdOp") + load_workloads("RotaryEmbeddingBwdOp"):
        RotaryEmbeddingFwdOp(row["batch"], row["seq_len"], row["heads"], row["heads_kv"], row["dim"],
                             row.get("rotary_dim"))
    for row in load_workloads("PagedKVAppendOp"):
        PagedKVAppendOp(row["heads_kv"], row["dim"], row["page_size"], row["heads"], row["rotary_dim"])
    for row in load_workloads("PagedAttentionDecodeOp"):
        PagedAttentionDecodeOp(row["heads"], row["heads_kv"], row["dim"], row["page_size"],
                               window=row.get("window"))


def test_ops_are_rebuilt_from_their_attributes():
    f = rotary_frequencies(32, factor=2.0)
    for op in (RotaryEmbeddingFwdOp(2, 10, 4, 2, 64, 32, True, f, 1.5, torch.float16, True),
               PagedKVAppendOp(2, 64, 16, 4, 32, True, f, 1.5, torch.float16),
               PagedAttentionDecodeOp(8, 2, 64, 16, 0.3, 100, torch.float16)):
        again = type(op)(**_extract_op_init_args(op))
        assert _extract_op_init_args(again) == _extract_op_init_args(op)
        assert len(_extract_op_init_args(op)) >= 7


# ------------------------------------------------------------ kept workspaces
def test_a_workspace_is_shared_only_by_calls_one_after_another(monkeypatch):
    """torch's own streams keep one each; others (their number is their handle) may be destroyed and
    their handle given again, and one handle, 2, is another stream in each host thread."""
    from concurrent.futures import ThreadPoolExecutor

    from tileops.kernels.attention import paged_attention as kernels

    now = dict(number=0, handle=0, capturing=False)
    monkeypatch.setattr(kernels, "_workspaces", {})
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: now["capturing"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: now["handle"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentStream", lambda i: (now["number"], i, 1), raising=False)
    for name in ("empty", "zeros"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda n, dtype, device, real=real: real(n, dtype=dtype))

    def ask(room=64, device=0, **stream):
        now.update(dict(number=0, handle=0, capturing=False), **stream)
        return kernels._workspace(torch.device("cuda", device), room)

    default, pool = ask(), ask(number=3, handle=0x7000)
    assert default[1] and pool[1] and default[0] is not pool[0]
    assert ask()[0] is default[0] and ask(number=3, handle=0x7000)[0] is pool[0]
    assert ask(device=1)[0] is not default[0]
    larger = ask(room=128)
    assert larger[0].numel() == 128 and larger[1] and ask()[0] is larger[0]
    assert not ask(capturing=True)[1] and ask(capturing=True)[0] is not larger[0]
    kept = len(kernels._workspaces)
    other = [ask(number=0x8000, handle=0x8000) for _ in range(2)]
    assert other[0][0] is not other[1][0] and not other[0][1] and not other[1][1]
    assert len(kernels._workspaces) == kept
    here = ask(number=2, handle=2)
    with ThreadPoolExecutor(1) as pool:
        there = pool.submit(ask, number=2, handle=2).result()
    assert here[0] is not there[0] and here[0] is not other[0][0]
    if here[1]:
        assert ask(number=2, handle=2)[0] is here[0]


def test_decode_entry_point_checks_its_output_alignment():
    """Rows of o are written four channels, 8 bytes, at a time."""
    fn = _native.lib().tileops_paged_decode_fwd
    for off, status in ((2, _native.EALIGN), (4, _native.EALIGN)):
        o = ctypes.c_void_p((1 << 20) + off)
        assert fn(SOME, SOME, SOME, SOME, SOME, o, SOME, SOME, 2, 4, 2, 8, 3, 4, 2, 2, _ints(*[8] * 8), 0, 0,
                  1.0, 2, NULL) == status


def test_kernel_overrides_of_a_shipped_kernel(accept_cpu):
    """A subclass that has a forward of its own gets the op's arguments and no more; one that calls the
    shipped forward, or has its own plan as well, keeps what belongs together."""
    seen = []

    class Rotary(RotaryEmbeddingFwdKernel):
        def forward(self, q, k, positions=None, inplace=False):
            seen.append("rotary")
            return q, k

    class RotaryBack(RotaryEmbeddingBwdKernel):
        def forward(self, q, k, positions=None, inplace=False):
            seen.append("back")
            return super().forward(q, k, positions, inplace)

    class Append(PagedKVAppendKernel):
        def forward(self, k, v, k_cache, v_cache, page_table, seq_lens, q=None, cu_seqlens=None):
            seen.append("append")

    class Decode(PagedAttentionDecodeKernel):
        def forward(self, q, k_cache, v_cache, page_table, seq_lens):
            seen.append("decode")
            return q, None

    class Planned(PagedAttentionDecodeKernel):
        def plan(self, *args):
            return "planned"

        def forward(self, q, k_cache, v_cache, page_table, seq_lens, plan=None):
            seen.append(plan)

    class Inherits(PagedAttentionDecodeKernel):
        pass

    q, k = _rotary_args()
    sizes = (2, 5, 4, 2, 8)
    op = RotaryEmbeddingFwdOp(*sizes, dtype=torch.float32, kernel_map={"rotary_fwd": Rotary})
    for _ in range(2):
        op(q, k)
    op = RotaryEmbeddingBwdOp(*sizes, dtype=torch.float32, kernel_map={"rotary_bwd": RotaryBack})
    with pytest.raises(ValueError, match="must be on a cuda device"):  # the shipped forward's
        op(q, k)
    args = _paged(torch.float16)
    op = PagedKVAppendOp(2, 8, 4, 4, dtype=torch.float16, kernel_map={"paged_kv_append": Append})
    for _ in range(2):
        op(**args)
    del args["k"], args["v"]
    for cls in (Decode, Planned):
        op = PagedAttentionDecodeOp(4, 2, 8, 4, dtype=torch.float16, kernel_map={"paged_attention_decode": cls})
        for _ in range(2):
            op(**args)
    op = PagedAttentionDecodeOp(4, 2, 8, 4, dtype=torch.float16, kernel_map={"paged_attention_decode": Inherits})
    with pytest.raises(ValueError, match="must be on a cuda device"):
        op(**args)
    assert seen == ["rotary", "rotary", "back", "append", "append", "decode", "decode", "planned", "planned"]


# ------------------------------------------------------------ tensors that share memory in part
def test_in_place_refuses_rows_that_share_memory_in_part(accept_cpu):
    """Slices of one projection lie apart; where they share a channel, or a whole head, both would be
    rotated by two threads."""
    B, S, D = 2, 5, 8
    wide = torch.randn(B, S, 8 * D)

    def heads(first, count):
        return wide[..., first:first + count * D].unflatten(-1, (count, D))

    op = RotaryEmbeddingFwdOp(B, S, 4, 2, D, dtype=torch.float32, inplace=True)
    for _ in range(2):
        for q, k in ((0, 4 * D), (2 * D, 0), (0, 6 * D), (16, 4 * D + 16)):
            with pytest.raises(ValueError, match="must be on a cuda device"):  # all checks passed
                op(heads(q, 4), heads(k, 2))
        for q, k in ((0, 0), (0, 2 * D), (0, 4 * D - 1), (4, 0), (D, 4 * D), (2 * D, D + 1)):
            with pytest.raises(ValueError, match="q and k share memory"):
                op(heads(q, 4), heads(k, 2))
    both = torch.randn(B, S, 2, 4, D)  # another stride between tokens than between slices
    op = RotaryEmbeddingFwdOp(B, S, 4, 4, D, dtype=torch.float32, inplace=True)
    with pytest.raises(ValueError, match="must be on a cuda device"):
        op(both[:, :, 0], both[:, :, 1])
    rows = torch.randn(3, S, 4, D)
    with pytest.raises(ValueError, match="q and k share memory"):
        op(rows[:2], rows[1:])  # the second row of one is the first of the other


def test_append_refuses_caches_that_share_memory_in_part(accept_cpu):
    P, Hkv, D = 4, 2, 8
    op = PagedKVAppendOp(Hkv, D, P, 4, dtype=torch.float32)
    args = _paged(torch.float32)
    pool = torch.zeros(4, P, Hkv, D)
    both = torch.zeros(3, P, 2, Hkv, D)
    mixed = torch.zeros(3, P, Hkv, 2 * D)
    halves = torch.zeros(3, 2, Hkv, P, D)
    for k, v in ((both[:, :, 0], both[:, :, 1]), (both[:, :, 1], both[:, :, 0]),
                 (mixed[..., :D], mixed[..., D:]),
                 (halves[:, 0].transpose(1, 2), halves[:, 1].transpose(1, 2))):
        for _ in range(2):
            with pytest.raises(ValueError, match="must be on a cuda device"):  # all checks passed
                op(**{**args, "k_cache": k, "v_cache": v})
    for k, v in ((pool[:3], pool[1:]), (pool[1:], pool[:3]), (mixed[..., :D], mixed[..., D - 1:-1]),
                 (both[:, :, 0], both[:, :, 0])):
        for _ in range(2):
            with pytest.raises(ValueError, match="k_cache and v_cache share memory"):
                op(**{**args, "k_cache": k, "v_cache": v})


def test_apart_against_every_address():
    from random import Random

    from tileops.kernels.attention._layouts import Apart

    rng = Random(0)
    buf = torch.zeros(4000)

    def view():
        shape = [rng.randint(1, 4) for _ in range(3)] + [rng.randint(1, 5)]
        strides = [rng.choice([1, 2, 3, 5, 8, 10, 16, 20, 40, 41, 60]) for _ in range(3)] + [1]
        return torch.as_strided(buf, shape, strides, rng.randint(0, 120))

    counts = [0, 0]
    for _ in range(3000):
        a, b = view(), view()
        if rng.random() < 0.5:
            b = torch.as_strided(buf, a.shape, a.stride(), b.storage_offset())
        places = [{t.storage_offset() + sum(i * s for i, s in zip(at, t.stride()))
                   for at in torch.cartesian_prod(*[torch.arange(n) for n in t.shape]).view(-1, 4).tolist()}
                  for t in (a, b)]
        apart = not (places[0] & places[1])
        counts[apart] += 1
        assert Apart(a, b)(a.data_ptr(), b.data_ptr()) == apart, (a.shape, a.stride(), b.shape, b.stride())
    assert min(counts) > 500
    a = torch.zeros(3, 4)
    assert not Apart(a, a)(a.data_ptr(), a.data_ptr() + 2)  # across elements
    assert Apart(a, a)(a.data_ptr(), a.data_ptr() + 48)
    none = torch.zeros(0, 4)
    assert Apart(none, a)(a.data_ptr(), a.data_ptr()) and Apart(none, none)(0, 0)


def test_decode_roofline_counts_the_tokens_of_the_last_call(accept_cpu):
    """A table is as wide as the longest sequence allowed: what a short batch reads goes by its lengths."""

    class Other(Kernel):
        def __init__(self, *args):
            super().__init__()

        def forward(self, *args):
            return args[0], None

    B, H, Hkv, D, P = 4, 4, 2, 8, 4
    args = dict(q=torch.zeros(B, H, D, dtype=torch.float16), page_table=torch.zeros(B, 50, dtype=torch.int32))
    args["k_cache"], args["v_cache"] = torch.zeros(2, 3, P, Hkv, D, dtype=torch.float16)
    for window, lens, seen in ((None, [5, 0, 12, 3], 20), (None, [-2, 1, 2**31 - 1, 0], 201),
                               (4, [5, 0, 12, 3], 11)):
        op = PagedAttentionDecodeOp(H, Hkv, D, P, window=window, dtype=torch.float16,
                                    kernel_map={"paged_attention_decode": Other})
        op(**args, seq_lens=torch.tensor(lens, dtype=torch.int32))
        assert op.eval_roofline() == (4 * seen * H * D,
                                      (2 * seen * Hkv * D + 2 * B * H * D) * 2 + 4 * B * H)
