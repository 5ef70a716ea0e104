"""Host side of the recurrent-block ops (gated linear recurrence, sandwich norm): the 64-bit
oracle's gradients against differences, refusals before any launch, roofline formulas, the C
entry points' argument checks.  CPU only."""

import ctypes

import pytest
import torch

from oracle import recurrent as ref
from tileops import _native
from tileops.benchmark.msprof import _extract_op_init_args
from tileops.kernels.linear_attention import (
    GatedLinearRecurrenceBwdKernel,
    GatedLinearRecurrenceFwdKernel,
)
from tileops.kernels.norm import FusedSandwichNormFwdKernel
from tileops.manifest import load_workloads
from tileops.ops.linear_attention import (
    GatedLinearRecurrenceBwdOp,
    GatedLinearRecurrenceDecodeOp,
    GatedLinearRecurrenceFwdOp,
)
from tileops.ops.norm import FusedSandwichNormBwdOp, FusedSandwichNormFwdOp

NULL = ctypes.c_void_p(0)


# ------------------------------------------------- the oracle against differences
def _differences(f, tensors, step=1e-6):
    """Central differences of the scalar f at every element of every tensor."""
    grads = []
    for t in tensors:
        g, flat = torch.empty_like(t), t.view(-1)
        for n in range(flat.numel()):
            keep = flat[n].item()
            flat[n] = keep + step
            up = f()
            flat[n] = keep - step
            g.view(-1)[n] = (up - f()) / (2 * step)
            flat[n] = keep
        grads.append(g)
    return grads


@pytest.mark.parametrize("packed", [False, True])
def test_recurrence_oracle_gradients_against_differences(packed):
    B, T, D = (1, 7, 3) if packed else (2, 5, 3)
    cu = torch.tensor([0, 3, 3, 7]) if packed else None
    nseq = 3 if packed else B
    x, i, r = (torch.randn(B, T, D, dtype=torch.float64) for _ in range(3))
    lam, h0 = torch.randn(D, dtype=torch.float64) - 2, torch.randn(nseq, D, dtype=torch.float64)
    dy, dT = torch.randn(B, T, D, dtype=torch.float64), torch.randn(nseq, D, dtype=torch.float64)

    def loss():
        y, final, _, _ = ref.glr_fwd(x, i, r, lam, h0, cu)
        return ((y * dy).sum() + (final * dT).sum()).item()

    (dx, di, dr, dlam, d0), _ = ref.glr_bwd(dy, x, i, r, lam, h0, dT, cu)
    # Central differences: h^2 f''' / 6 + 2^-53 |f| / h with h = 1e-6, |f| < 100: below 1e-7.
    for got, want in zip((dx, di, dr, dlam, d0), _differences(loss, (x, i, r, lam, h0))):
        torch.testing.assert_close(got, want, rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_sandwich_oracle_gradients_against_differences(norm):
    M, N, G = 4, 5, 2
    x, r, dy, ds = (torch.randn(M, N, dtype=torch.float64) for _ in range(4))
    w1, w2, b1, b2 = (1 + 0.1 * torch.randn(N, dtype=torch.float64) for _ in range(4))
    gate = torch.randn(G, N, dtype=torch.float64)

    def loss():
        s, _ = ref.sandwich_stream(x, r, w1, gate, b1, norm, 1e-6, 0.75)
        y, _ = ref.sandwich_next(s, w2, b2, norm, 1e-6)
        return ((y * dy).sum() + (s * ds).sum()).item()

    s, _ = ref.sandwich_stream(x, r, w1, gate, b1, norm, 1e-6, 0.75)
    got, _ = ref.sandwich_bwd(dy, ds, x, s, w1, w2, gate, b1, norm, 1e-6, 0.75)
    for a, b in zip(got, _differences(loss, (x, r, w1, w2, gate, b1, b2))):
        torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-7)


def test_oracle_states_and_identity_gates():
    x, i, r = (torch.randn(1, 130, 2) for _ in range(3))
    lam, h0 = torch.zeros(2), torch.randn(1, 2)
    states, bound = ref.glr_states(x, i, r, lam, h0)
    y, final, _, _ = ref.glr_fwd(x, i, r, lam, h0)
    assert states.shape == (1, 5, 2) and torch.equal(states[0, 0], h0[0].double())
    assert torch.equal(states[0, 4], y[0, 127]) and torch.equal(final[0], y[0, -1])
    assert (bound[:, 1:] > 0).all()
    shut = torch.full_like(r, -float("inf"))
    y, final, _, _ = ref.glr_fwd(x, i, shut, lam, h0)
    assert torch.equal(y, h0.double()[:, None].expand_as(y))


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
    import tileops.ops.linear_attention.gated_linear_recurrence as rec
    import tileops.ops.norm.sandwich_norm as norm

    fake = _AcceptCpu()
    for mod in (rec, norm):
        monkeypatch.setattr(mod, "get_device_backend", lambda: fake)


def _rec(B=2, T=5, D=8, dtype=torch.float32):
    return [torch.randn(B, T, D, dtype=dtype) for _ in range(3)] + [torch.randn(D)]


def test_recurrence_rejects_cpu_tensors():
    with pytest.raises(ValueError, match="x must be a cuda tensor"):
        GatedLinearRecurrenceFwdOp(2, 5, 8, dtype=torch.float32)(*_rec())
    with pytest.raises(ValueError, match="x must be a cuda tensor"):
        GatedLinearRecurrenceBwdOp(2, 5, 8, dtype=torch.float32)(
            torch.randn(2, 5, 8), *_rec(), torch.randn(2, 1, 8))
    with pytest.raises(ValueError, match="x must be a cuda tensor"):
        GatedLinearRecurrenceDecodeOp(2, 8, dtype=torch.float32)(
            *(torch.randn(2, 8) for _ in range(3)), torch.randn(8), torch.randn(2, 8))


@pytest.mark.parametrize("cls", [GatedLinearRecurrenceFwdOp, GatedLinearRecurrenceBwdOp])
def test_recurrence_rejects_sizes_and_types_at_construction(cls):
    with pytest.raises(ValueError, match="only supports dtypes"):
        cls(1, 4, 8, dtype=torch.float64)
    for c in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="decay_scale"):
            cls(1, 4, 8, c)
    for size in ((-1, 4, 8), (1, -1, 8), (1, 4, 0), (65536, 4, 8), (1, 2**31, 8)):
        with pytest.raises(ValueError, match="supports batch"):
            cls(*size)


@pytest.mark.parametrize("at, other, match", [
    (0, torch.randn(2, 5, 7), r"x.shape"),
    (1, torch.randn(2, 4, 8), r"input_gate.shape"),
    (2, torch.randn(10, 8), r"decay_gate.shape"),
    (3, torch.randn(1, 8), r"decay_param.shape"),
    (0, torch.randn(2, 5, 8).half(), r"x.dtype"),
    (1, torch.randn(2, 5, 8).half(), r"input_gate.dtype"),
    (3, torch.randn(8).half(), r"decay_param.dtype"),
    (2, torch.empty(2, 5, 8, device="meta"), r"decay_gate on cpu"),
])
def test_recurrence_rejects_wrong_inputs(accept_cpu, at, other, match):
    args = _rec()
    args[at] = other
    with pytest.raises(ValueError, match=match):
        GatedLinearRecurrenceFwdOp(2, 5, 8, dtype=torch.float32)(*args)
    with pytest.raises(ValueError, match=match):
        GatedLinearRecurrenceBwdOp(2, 5, 8, dtype=torch.float32)(
            torch.randn(2, 5, 8), *args, torch.randn(2, 1, 8))


def test_recurrence_rejects_wrong_states_and_offsets(accept_cpu):
    op = GatedLinearRecurrenceFwdOp(2, 5, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="initial_state.shape"):
        op(*_rec(), torch.randn(1, 8))
    with pytest.raises(ValueError, match="initial_state.dtype"):
        op(*_rec(), torch.randn(2, 8).half())
    with pytest.raises(ValueError, match="batch size is expected to be 1"):
        op(*_rec(), None, torch.tensor([0, 5]))
    op = GatedLinearRecurrenceFwdOp(1, 5, 8, dtype=torch.float32)
    args = _rec(B=1)
    with pytest.raises(ValueError, match="int32 or int64"):
        op(*args, None, torch.tensor([0.0, 5.0]))
    for cu in (torch.tensor([0]), torch.tensor([[0, 5]])):
        with pytest.raises(ValueError, match="1-D tensor of N"):
            op(*args, None, cu)
    with pytest.raises(ValueError, match="initial_state.shape"):
        op(*args, torch.randn(1, 8), torch.tensor([0, 2, 5]))
    bwd = GatedLinearRecurrenceBwdOp(1, 65, 8, dtype=torch.float32)
    args = _rec(B=1, T=65)
    dy = torch.randn(1, 65, 8)
    with pytest.raises(ValueError, match="states.shape"):
        bwd(dy, *args, torch.randn(1, 1, 8))
    with pytest.raises(ValueError, match="d_final_state.shape"):
        bwd(dy, *args, torch.randn(1, 3, 8), None, torch.randn(2, 8))
    with pytest.raises(ValueError, match="dy.shape"):
        bwd(dy[:, :64], *args, torch.randn(1, 3, 8))


def test_decode_rejects_wrong_inputs(accept_cpu):
    op = GatedLinearRecurrenceDecodeOp(2, 8, dtype=torch.float32, inplace=True)
    x = [torch.randn(2, 8) for _ in range(3)]
    lam = torch.randn(8)
    with pytest.raises(ValueError, match="state.shape"):
        op(*x, lam, torch.randn(1, 8))
    with pytest.raises(ValueError, match="state.dtype"):
        op(*x, lam, torch.randn(2, 8).half())
    with pytest.raises(ValueError, match="contiguous when it is updated in place"):
        op(*x, lam, torch.randn(2, 16)[:, ::2])


def test_sandwich_rejects_cpu_tensors_and_bad_construction():
    x, w = torch.randn(4, 8), torch.randn(8)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        FusedSandwichNormFwdOp()(x, x, w, w)
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        FusedSandwichNormBwdOp()(x, x, x, x, w, w)
    with pytest.raises(ValueError, match="norm must be"):
        FusedSandwichNormFwdOp(norm="batch")
    with pytest.raises(ValueError, match="only supports dtypes"):
        FusedSandwichNormFwdKernel(4, 8, "rms", 1e-6, 1.0, torch.int32)
    with pytest.raises(ValueError, match="supports norm in"):
        FusedSandwichNormFwdKernel(4, 8, "batch", 1e-6, 1.0, torch.float32)


def test_sandwich_rejects_wrong_inputs(accept_cpu):
    x, w = torch.randn(6, 8).half(), torch.randn(8).half()
    op = FusedSandwichNormFwdOp(dtype=torch.float16)
    for args, match in (
        ((x.float(), x, w, w), "x.dtype"), ((x, x.float(), w, w), "residual.dtype"),
        ((x, x[:, :4], w, w), "residual shape"), ((x, x, w[:4], w), "post_weight shape"),
        ((x, x, w, w.float()), "pre_weight.dtype"), ((x, x, w.double(), w), "post_weight.dtype"),
        ((x, x, w, w, w.float()), "gate.dtype"), ((x, x, w, w, torch.ones(4, 8).half()), "gate shape"),
        ((x, x, w, w, torch.ones(2, 4).half()), "gate shape"),
        ((x, x, w, w, torch.ones(0, 8).half()), "gate shape"),
        ((x, x, w, w, torch.ones(1, 2, 8).half()), "gate shape"),
        ((x, x, w, w, None, w[:2]), "post_bias shape"),
        ((x, x, w, w, None, None, w.float()), "pre_bias.dtype"),
        ((x, x.to("meta"), w, w), "residual on cpu"),
        ((x, x, w.to("meta"), w), "post_weight on cpu"),
        ((x[:, :0], x[:, :0], w[:0], w[:0]), "N >= 1"),
    ):
        with pytest.raises(ValueError, match=match):
            op(*args)
    with pytest.raises(ValueError, match="Expected M=3"):
        FusedSandwichNormFwdOp(M=3)(x, x, w, w)
    with pytest.raises(ValueError, match="hidden dim 4"):
        FusedSandwichNormFwdOp(N=4)(x, x, w, w)
    bwd = FusedSandwichNormBwdOp(dtype=torch.float16)
    with pytest.raises(ValueError, match="dy shape"):
        bwd(x[:3], None, x, x, w, w)
    with pytest.raises(ValueError, match="d_residual_out.dtype"):
        bwd(x, x.float(), x, x, w, w)


# ------------------------------------------------------------ formulas, manifest
def test_rooflines_and_init_args():
    op = GatedLinearRecurrenceFwdOp(2, 100, 64, 4.0, torch.float16, save_states=True)
    assert op.eval_roofline() == (20 * 12800, 4 * 12800 * 2 + 8 * 128 + 4 * 64)
    assert _extract_op_init_args(op) == dict(batch=2, seq_len=100, dim=64, decay_scale=4.0,
                                             dtype=torch.float16, save_states=True)
    op = GatedLinearRecurrenceBwdOp(2, 100, 64, dtype=torch.float32)
    assert op.eval_roofline() == (40 * 12800,
                                  7 * 12800 * 4 + 4 * 2 * 4 * 64 + 8 * 128 + 8 * 64)
    op = GatedLinearRecurrenceDecodeOp(3, 64, dtype=torch.float32)
    assert op.eval_roofline() == (20 * 192, 4 * 192 * 4 + 8 * 192 + 4 * 64)
    with pytest.raises(RuntimeError, match="requires a prior"):
        FusedSandwichNormFwdOp().eval_roofline()
    with pytest.raises(RuntimeError, match="requires a prior"):
        FusedSandwichNormBwdOp().eval_roofline()


def test_manifest_has_the_recurrent_block():
    for name in ("GatedLinearRecurrenceFwdOp", "GatedLinearRecurrenceBwdOp",
                 "GatedLinearRecurrenceDecodeOp", "FusedSandwichNormFwdOp",
                 "FusedSandwichNormBwdOp"):
        assert load_workloads(name)


# ------------------------------------------------------------ the C entry points
def test_glr_entry_points_check_their_arguments():
    lib = _native.lib()
    fwd = lambda b, t, d, cu=NULL, n=0, dt=2: lib.tileops_glr_fwd(  # noqa: E731
        *[NULL] * 5, cu, n, NULL, NULL, NULL, b, t, d, *[0] * 6, 8.0, dt, NULL)
    bwd = lambda b, t, d, cu=NULL, n=0, dt=2: lib.tileops_glr_bwd(  # noqa: E731
        *[NULL] * 8, cu, n, *[NULL] * 6, b, t, d, *[0] * 8, 8.0, dt, NULL)
    some = ctypes.c_void_p(16)
    for f in (fwd, bwd):
        assert f(-1, 4, 8) == f(1, -4, 8) == f(1, 4, -8) == _native.EBADSHAPE
        assert f(65536, 4, 8) == f(1, 1 << 31, 8) == f(1, 4, 1 << 31) == _native.EBADSHAPE
        assert f(1, 0, 8) == _native.EBADSHAPE
        assert f(2, 4, 8, some, 2) == f(1, 4, 8, some, 0) == _native.EBADSHAPE
        assert f(1, 4, 8, dt=7) == _native.EBADDTYPE
        assert f(0, 4, 8) == f(1, 4, 0) == _native.OK
        assert f(1, 4, 8) == _native.EINVAL
    assert lib.tileops_glr_bwd_workspace_bytes(-1, 4, 8) == -1
    assert lib.tileops_glr_bwd_workspace_bytes(2, 100, 64) >= 4 * 64
    step = lambda b, d, dt=2: lib.tileops_glr_decode_fwd(  # noqa: E731
        *[NULL] * 7, b, d, 0, 0, 0, 8.0, dt, NULL)
    assert step(-1, 8) == step(65536, 8) == _native.EBADSHAPE
    assert step(1, 8, 3) == _native.EBADDTYPE
    assert step(0, 8) == step(4, 0) == _native.OK
    assert step(4, 8) == _native.EINVAL


def test_sandwich_entry_points_check_their_arguments():
    lib = _native.lib()
    fwd = lambda m, n, g=1, norm=0, dt=2, aff=2: lib.tileops_sandwich_norm_fwd(  # noqa: E731
        *[NULL] * 9, m, n, g, norm, 1e-6, 1.0, dt, aff, NULL)
    bwd = lambda m, n, g=1, norm=0, dt=2, aff=2: lib.tileops_sandwich_norm_bwd(  # noqa: E731
        *[NULL] * 16, m, n, g, norm, 1e-6, 1.0, dt, aff, NULL)
    for f in (fwd, bwd):
        assert f(-1, 8) == f(4, 0) == f(4, 8, 3) == f(4, 8, 0) == _native.EBADSHAPE
        assert f(4, 8, norm=2) == _native.EINVAL
        assert f(4, 8) == _native.EINVAL  # NULL tensors
    assert fwd(0, 8) == _native.OK and bwd(0, 8) == _native.EBADSHAPE
    size = lib.tileops_sandwich_norm_bwd_workspace_bytes
    assert size(4, 8, 3, 0) == -1 and size(4, 0, 1, 0) == -1 and size(4, 8, 2, 1) > 0


def test_supported_types_of_the_kernels():
    for dtype in GatedLinearRecurrenceFwdKernel.SUPPORTED_DTYPES:
        assert GatedLinearRecurrenceFwdKernel(1, 1, 1, 1.0, dtype).dtype_str


# ------------------------------------------------------------ layouts, with the launch stubbed
def _overlapping(B, D, dtype=torch.float32):
    """Rows that overlap: a window slid along one signal, strides (1, 1)."""
    return torch.randn(B + 2 * D, dtype=dtype).unfold(0, D, 1)[:B]


@pytest.mark.parametrize("layout", ["overlapping", "expanded", "strided", "dense"])
def test_decode_output_rows_are_dense(accept_cpu, monkeypatch, layout):
    """The entry point writes y as dense rows, whatever strides x has."""
    B, D = 8, 32
    x = {"overlapping": lambda: _overlapping(B, D), "expanded": lambda: torch.randn(D).expand(B, D),
         "strided": lambda: torch.randn(2 * B, 2 * D)[::2, 3:3 + D],
         "dense": lambda: torch.randn(B, D)}[layout]()
    written = torch.arange(B * D, dtype=torch.float32)

    def launch(name, device, *args):
        assert name == "tileops_glr_decode_fwd" and args[0] == x.data_ptr() and args[9] == x.stride(0)
        ctypes.memmove(args[5], written.data_ptr(), 4 * B * D)

    monkeypatch.setattr(_native, "launch", launch)
    y, _ = GatedLinearRecurrenceDecodeOp(B, D, dtype=torch.float32)(
        x, torch.randn(B, D), torch.randn(B, D), torch.randn(D), torch.randn(B, D))
    assert torch.equal(y, written.view(B, D))


# ------------------------------------------------------------ required arguments left out
@pytest.mark.parametrize("at, name", [(0, "x"), (1, "residual"), (2, "post_weight"),
                                      (3, "pre_weight")])
def test_sandwich_names_a_required_argument_that_is_none(accept_cpu, at, name):
    x, w = torch.randn(4, 8), torch.randn(8)
    args = [x, x, w, w]
    args[at] = None
    with pytest.raises(ValueError, match=f"{name} must be a cuda tensor"):
        FusedSandwichNormFwdOp()(*args)


@pytest.mark.parametrize("at, name", [(0, "dy"), (2, "x"), (3, "residual_out"),
                                      (4, "post_weight"), (5, "pre_weight")])
def test_sandwich_backward_names_a_required_argument_that_is_none(accept_cpu, at, name):
    x, w = torch.randn(4, 8), torch.randn(8)
    for ds in (None, x):
        args = [x, ds, x, x, w, w]
        args[at] = None
        with pytest.raises(ValueError, match=f"{name} must be a cuda tensor"):
            FusedSandwichNormBwdOp()(*args)


@pytest.mark.parametrize("at", [2, 4, 5, 6])
def test_sandwich_refuses_what_is_no_tensor(accept_cpu, at):
    x, w = torch.randn(4, 8), torch.randn(8)
    args = [x, x, w, w, w, w, w]
    args[at] = w.tolist()
    with pytest.raises(ValueError, match="must be a cuda tensor"):
        FusedSandwichNormFwdOp()(*args)


# ------------------------------------------------------------ offsets beyond int32
@pytest.mark.parametrize("offsets", [[0, 2**32 + 50, 100], [0, 50, 2**32 + 100], [-2**32, 50, 100],
                                     [0, -2**32 + 50, 100], [0, -2**40, 2**33]])
def test_offsets_keep_their_sign_and_order_in_32_bits(offsets):
    """64-bit offsets that int32 cannot hold saturate: what breaks the rule still breaks it."""
    kernel = GatedLinearRecurrenceFwdKernel(1, 100, 8, 8.0, torch.float32)
    wide = torch.tensor(offsets)
    cu, nseq = kernel._sequences(wide, torch.device("cpu"))
    assert cu.dtype == torch.int32 and nseq == 2
    whole = lambda c: c[0] == 0 and c[-1] == 100 and (c.diff() >= 0).all()  # noqa: E731
    assert not whole(wide) and not whole(cu)
    good = torch.tensor([0, 50, 100])
    for t in (good, good.int(), good.int().repeat_interleave(2)[::2]):
        cu, _ = kernel._sequences(t, torch.device("cpu"))
        assert cu.tolist() == [0, 50, 100] and cu.is_contiguous() and cu.dtype == torch.int32


@pytest.mark.parametrize("c", [1e39, 1e-39, 5e-324])
def test_recurrence_rejects_a_decay_scale_that_float32_cannot_hold(c):
    """1e39 would be inf in the kernels, and inf * sigmoid(-inf) NaN; 1e-39 a subnormal."""
    for cls in (GatedLinearRecurrenceFwdOp, GatedLinearRecurrenceBwdOp):
        with pytest.raises(ValueError, match="decay_scale"):
            cls(1, 4, 8, c)
    with pytest.raises(ValueError, match="decay_scale"):
        GatedLinearRecurrenceDecodeOp(1, 8, c)
    GatedLinearRecurrenceDecodeOp(1, 8, 1e38)
    GatedLinearRecurrenceDecodeOp(1, 8, 1.2e-38)


# ------------------------------------------------------------ no token: states pass through
def test_states_that_pass_through_carry_no_graph():
    """These ops build no autograd graph, without a token either."""
    x, lam = torch.randn(2, 0, 8), torch.randn(8)
    h0 = torch.randn(2, 8, requires_grad=True)
    _, final, states = GatedLinearRecurrenceFwdKernel(2, 0, 8, 8.0, torch.float32)(
        x, x, x, lam, h0, None, True)
    assert not final.requires_grad and torch.equal(final, h0) and final.data_ptr() != h0.data_ptr()
    *_, d0 = GatedLinearRecurrenceBwdKernel(2, 0, 8, 8.0, torch.float32)(
        x, x, x, x, lam, states, None, h0)
    assert not d0.requires_grad and torch.equal(d0, h0) and d0.data_ptr() != h0.data_ptr()


# ------------------------------------------------------------ roofline of packed calls
def test_rooflines_count_a_state_for_each_packed_sequence(accept_cpu, monkeypatch):
    monkeypatch.setattr(_native, "launch", lambda *args: None)
    args, cu = _rec(B=1, T=100), torch.tensor([0, 10, 10, 70, 100])
    op = GatedLinearRecurrenceFwdOp(1, 100, 8, dtype=torch.float32, save_states=True)
    states = op(*args, None, cu)[2]
    assert op.eval_roofline() == (20 * 800, 4 * 800 * 4 + 8 * 4 * 8 + 4 * 8)
    op(*args)
    assert op.eval_roofline() == (20 * 800, 4 * 800 * 4 + 8 * 8 + 4 * 8)
    bwd = GatedLinearRecurrenceBwdOp(1, 100, 8, dtype=torch.float32)
    bwd(torch.randn(1, 100, 8), *args, states, None, None, cu)
    assert bwd.eval_roofline() == (40 * 800, 7 * 800 * 4 + 4 * 4 * 8 + 8 * 4 * 8 + 8 * 8)


# ------------------------------------------------------------ workspaces of the C entry points
def test_entry_points_refuse_a_misaligned_workspace():
    """16-byte words go to the workspace: one off that boundary is refused before any launch."""
    lib = _native.lib()
    some = ctypes.c_void_p(1 << 20)
    for off in (1, 2, 4, 8):
        ws = ctypes.c_void_p((1 << 20) + off)
        assert lib.tileops_glr_bwd(*[some] * 6, NULL, NULL, NULL, 0, *[some] * 5, ws, 1, 4, 8,
                                   *[8] * 8, 8.0, 2, NULL) == _native.EALIGN
        for bias in (NULL, some):
            assert lib.tileops_sandwich_norm_bwd(
                some, NULL, some, some, some, some, NULL, bias, some, some, some, some, NULL, bias,
                NULL, ws, 4, 8, 1, 0, 1e-6, 1.0, 2, 2, NULL) == _native.EALIGN
