"""GPU parity of the gated linear recurrence ops against the 64-bit oracle.

Every value is held to the oracle's running error bound plus half a step of its type
(``oracle.recurrent``); no tolerance is fitted.
"""

import pytest
import torch

from oracle import recurrent as ref
from tileops import _native as nat
from tileops.ops.linear_attention import (
    GatedLinearRecurrenceBwdOp,
    GatedLinearRecurrenceDecodeOp,
    GatedLinearRecurrenceFwdOp,
)

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ("dx", "d_input_gate", "d_decay_gate", "d_decay_param", "d_initial_state")


def _inputs(B, T, D, dtype, nseq=None, slow=True):
    """x, gates, lambda, initial state, dy, d_final.  slow: decays of 0.9 to 0.999 a token."""
    x, i, r, dy = (torch.randn(B, T, D, device="cuda").to(dtype) for _ in range(4))
    if slow:
        a = 0.9 + 0.099 * torch.rand(D, device="cuda")
        lam = torch.log(torch.expm1(-torch.log(a) / 8.0))
    else:
        lam = 2 * torch.randn(D, device="cuda")  # decays from almost none to almost all
    h0, dT = (torch.randn(nseq or B, D, device="cuda") for _ in range(2))
    return (x, i, r, lam), h0, dy, dT


def _check_all(gates, h0, dy, dT, cu=None, scale=8.0):
    x = gates[0]
    B, T, D = x.shape
    y, final, states = GatedLinearRecurrenceFwdOp(B, T, D, scale, x.dtype, save_states=True)(
        *gates, h0, cu)
    y_ref, final_ref, y_tol, final_tol = ref.glr_fwd(*gates, h0, cu, scale)
    ref.assert_within(y, y_ref, y_tol, "y")
    ref.assert_within(final, final_ref, final_tol, "final_state")
    if cu is None:
        ref.assert_within(states, *ref.glr_states(*gates, h0, scale), "states")
    got = GatedLinearRecurrenceBwdOp(B, T, D, scale, x.dtype)(dy, *gates, states, h0, dT, cu)
    want, tol = ref.glr_bwd(dy, *gates, h0, dT, cu, scale)
    for name, g, w, t in zip(NAMES, got, want, tol):
        ref.assert_within(g, w, t, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, T, D", [
    (1, 1, 1), (2, 1, 64), (3, 2, 65), (1, 7, 130), (2, 16, 64), (2, 17, 96), (1, 63, 200),
    (1, 64, 64), (1, 65, 33), (2, 127, 72), (1, 128, 128), (1, 129, 66), (2, 300, 190),
    (1, 515, 256), (1, 1025, 70), (1, 2500, 34), (5, 260, 100),
])
def test_sizes(B, T, D, dtype):
    _check_all(*_inputs(B, T, D, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_decay(dtype):
    _check_all(*_inputs(2, 333, 140, dtype, slow=False))


@pytest.mark.parametrize("scale", [0.01, 1.0, 40.0])
def test_decay_scale(scale):
    _check_all(*_inputs(1, 150, 66, torch.bfloat16, slow=False), scale=scale)


def test_wide_logits():
    """Gates from shut to open to the last bit."""
    gates, h0, dy, dT = _inputs(1, 200, 96, torch.float32, slow=False)
    x, i, r, lam = gates
    _check_all((x, i * 30, r * 30, lam), h0, dy, dT)


def test_many_batches():
    _check_all(*_inputs(70, 20, 66, torch.bfloat16))


@pytest.mark.parametrize("B, T, D", [(1, 4096, 8), (33, 130, 512), (1, 700, 2050)])
def test_long_and_wide(B, T, D):
    _check_all(*_inputs(B, T, D, torch.bfloat16))


@pytest.mark.parametrize("B, T, D", [
    (3, 1100, 1024),   # CTAs of 32 channels that have an SM each, several steps
    (1, 2100, 1600),   # of 16 channels
    (1, 1500, 1000),   # clusters of two
    (1, 5000, 272),    # clusters of eight
    (40, 700, 200),    # more CTAs than SMs
])
@pytest.mark.parametrize("packed, dtype", [(False, torch.bfloat16), (True, torch.bfloat16),
                                           (True, torch.float32)])
def test_every_split_of_the_tokens(B, T, D, packed, dtype):
    """Long enough for each choice of warps and clusters to take several steps."""
    if packed:
        B = 1
        cuts = torch.randint(0, T + 1, (20,)).sort().values.tolist()
        lengths = [b - a for a, b in zip([0, *cuts], [*cuts, T])]
        _check_all(*_inputs(1, T, D, dtype, nseq=21), cu=_cu(lengths))
    else:
        _check_all(*_inputs(B, T, D, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_whole_sm_a_cta(dtype):
    """One sequence whose channels fill more than half the SMs, over several steps."""
    _check_all(*_inputs(1, 1000, 2600, dtype))


def test_many_partial_sums():
    _check_all(*_inputs(300, 5, 40, torch.float32))


def test_without_states():
    gates, _, dy, _ = _inputs(2, 100, 66, torch.float32)
    y, final = GatedLinearRecurrenceFwdOp(2, 100, 66, dtype=torch.float32)(*gates)
    y_ref, final_ref, y_tol, f_tol = ref.glr_fwd(*gates)
    ref.assert_within(y, y_ref, y_tol)
    ref.assert_within(final, final_ref, f_tol)
    states = GatedLinearRecurrenceFwdOp(2, 100, 66, dtype=torch.float32, save_states=True)(*gates)[2]
    got = GatedLinearRecurrenceBwdOp(2, 100, 66, dtype=torch.float32)(dy, *gates, states)
    want, tol = ref.glr_bwd(dy, *gates)
    for name, g, w, t in zip(NAMES, got, want, tol):
        ref.assert_within(g, w, t, name)


# ------------------------------------------------------------ packed sequences
def _cu(lengths, dtype=torch.int32):
    return torch.tensor([0, *lengths], device="cuda").cumsum(0).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [
    [40], [1] * 33, [0, 5, 0, 0, 90, 1, 0], [64, 64, 64], [63, 1, 65, 130], [0, 0, 20, 300, 0],
    [700, 3, 1, 1, 900, 2], [17] * 40,
])
def test_packed(lengths, dtype):
    cu = _cu(lengths)
    _check_all(*_inputs(1, int(cu[-1]), 70, dtype, nseq=len(lengths)), cu=cu)


def test_packed_many_short():
    lengths = [int(n) for n in torch.randint(0, 4, (900,))]
    cu = _cu(lengths, torch.int64)
    _check_all(*_inputs(1, int(cu[-1]), 36, torch.bfloat16, nseq=len(lengths)), cu=cu)


def test_packed_without_states():
    lengths = [30, 0, 100]
    gates, _, dy, _ = _inputs(1, 130, 66, torch.float32)
    cu = _cu(lengths)
    y, final, states = GatedLinearRecurrenceFwdOp(1, 130, 66, dtype=torch.float32,
                                                  save_states=True)(*gates, None, cu)
    y_ref, final_ref, y_tol, f_tol = ref.glr_fwd(*gates, None, cu)
    ref.assert_within(y, y_ref, y_tol)
    ref.assert_within(final, final_ref, f_tol)
    got = GatedLinearRecurrenceBwdOp(1, 130, 66, dtype=torch.float32)(dy, *gates, states, None,
                                                                     None, cu)
    want, tol = ref.glr_bwd(dy, *gates, None, None, cu)
    for name, g, w, t in zip(NAMES, got, want, tol):
        ref.assert_within(g, w, t, name)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nothing_crosses_a_sequence(bad):
    """Infinities and NaN in x, the gates, dy and the states of one sequence stay in it."""
    lengths = [30, 50, 45]
    cu = _cu(lengths)
    gates, h0, dy, dT = _inputs(1, 125, 66, torch.float32, nseq=3)
    fwd = GatedLinearRecurrenceFwdOp(1, 125, 66, dtype=torch.float32, save_states=True)
    bwd = GatedLinearRecurrenceBwdOp(1, 125, 66, dtype=torch.float32)

    def both(gates, h0, dy, dT):
        y, final, states = fwd(*gates, h0, cu)
        dx, di, dr, _, d0 = bwd(dy, *gates, states, h0, dT, cu)
        return y, dx, di, dr, final, d0

    clean = both(gates, h0, dy, dT)
    spoiled = [t.clone() for t in (*gates[:3], dy)]
    for t in spoiled:
        t[0, 30:80] = bad
    h1, d1 = h0.clone(), dT.clone()
    h1[1], d1[1] = bad, bad
    got = both((*spoiled[:3], gates[3]), h1, spoiled[3], d1)
    for a, b in zip(clean[:4], got[:4]):
        assert torch.equal(a[0, :30], b[0, :30]) and torch.equal(a[0, 80:], b[0, 80:])
    for a, b in zip(clean[4:], got[4:]):
        assert torch.equal(a[[0, 2]], b[[0, 2]])


def test_nan_stays_in_its_channel_and_is_kept():
    gates, h0, _, _ = _inputs(1, 200, 66, torch.bfloat16)
    x, i, r, lam = gates
    op = GatedLinearRecurrenceFwdOp(1, 200, 66)
    clean, _ = op(*gates, h0)
    for at in range(3):
        t = [v.clone() for v in (x, i, r)]
        t[at][0, 100, 5] = float("nan")
        y, final = op(*t, lam, h0)
        keep = torch.arange(66, device="cuda") != 5
        assert torch.equal(y[..., keep], clean[..., keep])
        assert torch.equal(y[0, :100, 5], clean[0, :100, 5])
        assert y[0, 100:, 5].isnan().all() and final[0, 5].isnan()
    lam = lam.clone()
    lam[7] = float("nan")
    y, _ = op(x, i, r, lam, h0)
    assert y[..., 7].isnan().all() and not y[..., 8].isnan().any()


# ------------------------------------------------------------ gates at their ends
@pytest.mark.parametrize("dtype", DTYPES)
def test_shut_decay_gate_keeps_the_state(dtype):
    """decay_gate = -inf (a padded token): the state stays, and the token has no gradient.

    The state before each run of tokens is joined from the maps of the runs before it, so two
    runs see the same state with different roundings, each within the oracle's bound; a token
    by itself (the decode op) keeps it to the bit."""
    (x, i, r, lam), h0, dy, dT = _inputs(2, 90, 66, dtype)
    r[:, 40:70] = -float("inf")
    fwd = GatedLinearRecurrenceFwdOp(2, 90, 66, dtype=dtype, save_states=True)
    y, final, states = fwd(x, i, r, lam, h0)
    y_ref, _, y_tol, _ = ref.glr_fwd(x, i, r, lam, h0)
    assert torch.equal(y_ref[:, 40:70], y_ref[:, 39:40].expand(-1, 30, -1))
    ref.assert_within(y, y_ref, y_tol, "y")
    _, kept = GatedLinearRecurrenceDecodeOp(2, 66, dtype=dtype)(x[:, 50], i[:, 50], r[:, 50], lam, h0)
    assert torch.equal(kept, h0)
    whole = torch.cat([torch.arange(40), torch.arange(70, 90)]).cuda()
    _, final_cut = GatedLinearRecurrenceFwdOp(2, 60, 66, dtype=dtype)(
        *(t[:, whole].contiguous() for t in (x, i, r)), lam, h0)
    _, _, _, tol = ref.glr_fwd(x[:, whole], i[:, whole], r[:, whole], lam, h0)
    assert ((final - final_cut).abs().cpu() <= 2 * tol).all()
    dx, di, dr, dlam, d0 = GatedLinearRecurrenceBwdOp(2, 90, 66, dtype=dtype)(
        dy, x, i, r, lam, states, h0, dT)
    assert (dx[:, 40:70] == 0).all() and (di[:, 40:70] == 0).all() and (dr[:, 40:70] == 0).all()
    assert all(t.isfinite().all() for t in (dx, di, dr, dlam, d0))


def test_lowest_values_in_the_gates():
    (x, i, r, lam), h0, dy, dT = _inputs(1, 50, 66, torch.bfloat16)
    low = torch.finfo(torch.bfloat16).min
    i[:, 10:20], r[:, 20:30], i[:, 30:35], r[:, 30:35] = low, low, -low, -low
    _check_all((x, i, r, lam), h0, dy, dT)


def test_channels_that_never_decay():
    """lambda far below zero: a = 1 and m = 0 to the last bit; gradients stay finite."""
    (x, i, r, lam), h0, dy, dT = _inputs(1, 80, 66, torch.float32)
    lam = torch.full_like(lam, -200.0)
    y, _, states = GatedLinearRecurrenceFwdOp(1, 80, 66, dtype=torch.float32, save_states=True)(
        x, i, r, lam, h0)
    assert torch.equal(y, h0[:, None].expand_as(y))
    got = GatedLinearRecurrenceBwdOp(1, 80, 66, dtype=torch.float32)(dy, x, i, r, lam, states, h0,
                                                                     dT)
    assert all(t.isfinite().all() for t in got)
    assert (got[3] == 0).all()


# ------------------------------------------------------------ strides, streams, graphs
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D, shift", [(64, 0), (66, 1), (65, 0), (96, 2)])
def test_column_slices_are_read_in_place(D, shift, dtype):
    B, T = 2, 140
    wide = torch.randn(B, T, 4 * D + shift, device="cuda").to(dtype)
    x, i, r, dy = wide[..., shift:].split(D, dim=-1)
    (_, _, _, lam), h0, _, dT = _inputs(B, T, D, dtype)
    _check_all((x, i, r, lam), h0, dy, dT)


def test_other_layouts():
    B, T, D = 2, 70, 64
    (x, i, r, lam), h0, dy, dT = _inputs(B, T, D, torch.bfloat16)
    x = x.transpose(0, 1).contiguous().transpose(0, 1)  # time first
    i = i.transpose(1, 2).contiguous().transpose(1, 2)  # channels not contiguous: copied
    r = r[:1].expand(B, T, D)                           # one row for the whole batch
    dy = dy[:, :1].expand(B, T, D)
    lam = torch.stack([lam, lam], dim=1)[:, 0]
    h0 = h0.t().contiguous().t()
    _check_all((x, i, r, lam), h0, dy, dT)


def test_deterministic_and_equal_on_another_stream():
    (x, i, r, lam), h0, dy, dT = _inputs(2, 1500, 320, torch.bfloat16)
    fwd = GatedLinearRecurrenceFwdOp(2, 1500, 320, save_states=True)
    bwd = GatedLinearRecurrenceBwdOp(2, 1500, 320)

    def both():
        y, final, states = fwd(x, i, r, lam, h0)
        return y, final, states, *bwd(dy, x, i, r, lam, states, h0, dT)

    first = both()
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("packed", [False, True])
def test_captured_and_replayed(packed):
    """Two graphs from one pool: forward + backward, replayed on new inputs."""
    B, T, D = (1, 1200, 130) if packed else (2, 600, 130)
    lengths = [500, 0, 300, 400]
    cu = _cu(lengths) if packed else None
    (x, i, r, lam), h0, dy, dT = _inputs(B, T, D, torch.bfloat16, nseq=4 if packed else None)
    fwd = GatedLinearRecurrenceFwdOp(B, T, D, save_states=True)
    bwd = GatedLinearRecurrenceBwdOp(B, T, D)

    def both():
        y, final, states = fwd(x, i, r, lam, h0, cu)
        return y, final, *bwd(dy, x, i, r, lam, states, h0, dT, cu)

    both()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(both())
        graphs.append(g)
    for t in (x, i, r, dy):
        t.copy_(torch.randn_like(t))
    want = both()
    for g, out in zip(graphs, outs):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


# ------------------------------------------------------------ empty, large, malformed
def test_nothing_to_do():
    for B, T in ((0, 5), (2, 0), (0, 0)):
        gates, h0, dy, dT = _inputs(B, T, 8, torch.bfloat16)
        y, final, states = GatedLinearRecurrenceFwdOp(B, T, 8, save_states=True)(*gates, h0)
        assert y.shape == (B, T, 8) and torch.equal(final, h0)
        got = GatedLinearRecurrenceBwdOp(B, T, 8)(dy, *gates, states, h0, dT)
        assert torch.equal(got[4], dT) and (got[3] == 0).all() and got[0].shape == (B, T, 8)
        assert (GatedLinearRecurrenceFwdOp(B, T, 8)(*gates)[1] == 0).all()
    gates, h0, dy, dT = _inputs(1, 0, 8, torch.bfloat16, nseq=3)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    y, final = GatedLinearRecurrenceFwdOp(1, 0, 8)(*gates, h0, cu)
    assert y.shape == (1, 0, 8) and torch.equal(final, h0)


def test_offsets_beyond_32_bits():
    """More than 2^32 output elements from one repeated row: every channel settles at
    u / (1 - a)."""
    T, D = (1 << 20) + 77, 4104
    row = torch.randn(3, 1, 1, D, device="cuda").bfloat16()
    x, i, r = (t.expand(1, T, D) for t in row)
    lam = torch.zeros(D, device="cuda")
    y, final = GatedLinearRecurrenceFwdOp(1, T, D)(x, i, r, lam)
    _, last, _, tol = ref.glr_fwd(*(t.expand(1, 3000, D) for t in row.cpu()), lam)
    ref.assert_within(final, last, tol, "final_state")
    ref.assert_within(y[:, -1], last, tol, "last row")
    ref.assert_within(y[:, T // 2], last, tol, "middle row")


@pytest.mark.parametrize("offsets", [[0, 50, 90], [1, 50, 100], [0, 60, 40, 100],
                                     [0, 50, 1 << 30], [-5, 50, 100], [0, 101, 100]])
def test_malformed_offsets_set_the_error_flag(offsets):
    (x, i, r, lam), _, dy, _ = _inputs(1, 100, 66, torch.bfloat16)
    cu = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    flag = lambda: nat.lib().tileops_device_error_flag(nat.stream_handle(x.device), 1)  # noqa: E731
    flag()
    _, _, states = GatedLinearRecurrenceFwdOp(1, 100, 66, save_states=True)(x, i, r, lam, None, cu)
    assert flag() == 2
    GatedLinearRecurrenceBwdOp(1, 100, 66)(dy, x, i, r, lam, states, None, None, cu)
    assert flag() == 2
    cu = torch.tensor([0, 50, 50, 100], dtype=torch.int32, device="cuda")
    GatedLinearRecurrenceFwdOp(1, 100, 66)(x, i, r, lam, None, cu)
    assert flag() == 0


# ------------------------------------------------------------ differences
def test_gradient_against_differences():
    """The forward op's own values along random directions: (L(+h) - L(-h)) / 2h in fp32.

    L = <y, dy> + <final, dT> is summed in 64 bits; the forward's error of each value is bounded
    by the oracle, so L's is at most <bounds, |dy|> =: E and the quotient's E / h; the quotient's
    own h^2 f''' / 6 is measured on the 64-bit oracle at the same points and taken off."""
    B, T, D, h = 1, 60, 66, 1e-2
    gates, h0, dy, dT = _inputs(B, T, D, torch.float32)
    fwd = GatedLinearRecurrenceFwdOp(B, T, D, dtype=torch.float32, save_states=True)
    _, _, states = fwd(*gates, h0)
    grads = GatedLinearRecurrenceBwdOp(B, T, D, dtype=torch.float32)(dy, *gates, states, h0, dT)
    at = [*gates, h0]

    def loss(y, final):
        return ((y.cpu().double() * dy.cpu()).sum() + (final.cpu().double() * dT.cpu()).sum()).item()

    for n, t in enumerate(at):
        way = torch.randn_like(t)
        ends, exact, err = [], [], 0.0
        for sign in (1, -1):
            moved = list(at)
            moved[n] = t + sign * h * way
            y, final, _ = fwd(*moved)
            y64, f64, ey, ef = ref.glr_fwd(*moved)
            ends.append(loss(y, final))
            exact.append(loss(y64, f64))
            err += ((ey + ref.U * y64.abs()) * dy.cpu().abs()).sum().item()
            err += (ef * dT.cpu().abs()).sum().item()
        want, tol = ref.glr_bwd(dy, *gates, h0, dT)
        slope64 = (want[n] * way.cpu().double()).sum().item()
        slope = (grads[n].cpu().double() * way.cpu().double()).sum().item()
        curve = (exact[0] - exact[1]) / (2 * h) - slope64  # the quotient's own error
        grad_err = (tol[n] * way.cpu().abs()).sum().item() + ref.U * abs(slope) * 8
        assert abs((ends[0] - ends[1]) / (2 * h) - curve - slope) <= err / (2 * h) + grad_err


# ------------------------------------------------------------ decode
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, D", [(1, 1), (1, 2560), (3, 65), (130, 72), (2, 4097)])
def test_decode(B, D, dtype):
    (x, i, r, lam), h0, _, _ = _inputs(B, 1, D, dtype)
    args = (x[:, 0], i[:, 0], r[:, 0], lam)
    y_ref, h_ref, y_tol, h_tol = ref.glr_fwd(x, i, r, lam, h0)
    keep = h0.clone()
    y, h = GatedLinearRecurrenceDecodeOp(B, D, dtype=dtype)(*args, h0)
    ref.assert_within(y, y_ref[:, 0], y_tol[:, 0], "y")
    ref.assert_within(h, h_ref, h_tol, "state")
    assert torch.equal(h0, keep)
    y2, h2 = GatedLinearRecurrenceDecodeOp(B, D, dtype=dtype, inplace=True)(*args, h0)
    assert h2 is h0 and torch.equal(h2, h) and torch.equal(y2, y)


@pytest.mark.parametrize("D, shift", [(64, 0), (66, 1), (33, 0)])
def test_decode_slices_and_empty(D, shift):
    wide = torch.randn(5, 3 * D + shift, device="cuda").bfloat16()
    x, i, r = wide[:, shift:].split(D, dim=-1)
    lam, h0 = torch.randn(D, device="cuda"), torch.randn(5, D, device="cuda")
    y, h = GatedLinearRecurrenceDecodeOp(5, D)(x, i, r, lam, h0)
    y_ref, h_ref, y_tol, h_tol = ref.glr_fwd(x[:, None], i[:, None], r[:, None], lam, h0)
    ref.assert_within(y, y_ref[:, 0], y_tol[:, 0], "y")
    ref.assert_within(h, h_ref, h_tol, "state")
    y, h = GatedLinearRecurrenceDecodeOp(0, D)(x[:0], i[:0], r[:0], lam, h0[:0])
    assert y.shape == (0, D) and h.shape == (0, D)


def test_decode_follows_a_prefill():
    """Prefill, then token by token in place, against one scan over all of it."""
    B, T, D, cut = 2, 90, 130, 77
    (x, i, r, lam), h0, _, _ = _inputs(B, T, D, torch.bfloat16)
    y_ref, h_ref, y_tol, h_tol = ref.glr_fwd(x, i, r, lam, h0)
    _, state = GatedLinearRecurrenceFwdOp(B, cut, D)(x[:, :cut], i[:, :cut], r[:, :cut], lam, h0)
    step = GatedLinearRecurrenceDecodeOp(B, D, inplace=True)
    for t in range(cut, T):
        y, _ = step(x[:, t], i[:, t], r[:, t], lam, state)
        ref.assert_within(y, y_ref[:, t], y_tol[:, t], f"token {t}")
    ref.assert_within(state, h_ref, h_tol, "state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["overlapping", "step 2", "expanded", "strided"])
@pytest.mark.parametrize("B, D", [(8, 32), (3, 65), (40, 48)])
def test_decode_layouts(B, D, layout, dtype):
    """Rows of x and the gates at any distance, none and one element among them."""
    def rows():
        signal = torch.randn(2 * (B + D), device="cuda").to(dtype)
        wide = torch.randn(2 * B, 3 * D, device="cuda").to(dtype)
        return {"overlapping": signal.unfold(0, D, 1)[:B], "step 2": signal.unfold(0, D, 2)[:B],
                "expanded": signal[:D].expand(B, D), "strided": wide[::2, 1:1 + D]}[layout]

    x, i, r = rows(), rows(), rows()
    assert x.shape == (B, D)
    lam, h0 = torch.randn(D, device="cuda") - 2, torch.randn(B, D, device="cuda")
    y_ref, h_ref, y_tol, h_tol = ref.glr_fwd(x[:, None], i[:, None], r[:, None], lam, h0)
    y, h = GatedLinearRecurrenceDecodeOp(B, D, dtype=dtype)(x, i, r, lam, h0)
    ref.assert_within(y, y_ref[:, 0], y_tol[:, 0], "y")
    ref.assert_within(h, h_ref, h_tol, "state")
    y2, h2 = GatedLinearRecurrenceDecodeOp(B, D, dtype=dtype, inplace=True)(x, i, r, lam, h0)
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_overlapping_rows_in_whole_sequences(dtype):
    """Tokens that overlap, of x, the gates and dy."""
    B, T, D = 2, 70, 40
    x, i, r, dy = (torch.randn(B, T + D, device="cuda").to(dtype).unfold(1, D, 1)[:, :T]
                   for _ in range(4))
    (_, _, _, lam), h0, _, dT = _inputs(B, T, D, dtype)
    _check_all((x, i, r, lam), h0, dy, dT)


@pytest.mark.parametrize("offsets", [[0, 2**32 + 50, 100], [0, 50, 2**32 + 100], [-2**32, 50, 100]])
def test_offsets_that_int32_cannot_hold_set_the_error_flag(offsets):
    (x, i, r, lam), _, dy, _ = _inputs(1, 100, 66, torch.bfloat16)
    cu = torch.tensor(offsets, device="cuda")
    flag = lambda: nat.lib().tileops_device_error_flag(nat.stream_handle(x.device), 1)  # noqa: E731
    flag()
    _, _, states = GatedLinearRecurrenceFwdOp(1, 100, 66, save_states=True)(x, i, r, lam, None, cu)
    assert flag() == 2
    GatedLinearRecurrenceBwdOp(1, 100, 66)(dy, x, i, r, lam, states, None, None, cu)
    assert flag() == 2
    cu = torch.tensor([0, 50, 100], device="cuda")
    GatedLinearRecurrenceFwdOp(1, 100, 66)(x, i, r, lam, None, cu)
    assert flag() == 0


# ------------------------------------------------------------ padded tokens
def _padded(T, D, dtype, B=2):
    """Inputs whose decay gate is shut over some tokens, and those tokens."""
    (x, i, r, lam), h0, dy, dT = _inputs(B, T, D, dtype)
    shut = torch.zeros(T, dtype=torch.bool, device="cuda")
    for a, b in ((0, 5), (16, 32), (40, 70), (T - 9, T)):
        shut[a:b] = True
    r[:, shut] = -float("inf")
    return x, i, r, lam, h0, dy, dT, shut


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, D", [(90, 66), (700, 64), (2100, 272)])
def test_padded_tokens_have_no_say(T, D, dtype):
    """Whatever finite x and input gate a padded token holds, its type's ends too, every output is
    the same to the bit, and its own gradients are zeros."""
    x, i, r, lam, h0, dy, dT, shut = _padded(T, D, dtype)
    B, most = x.shape[0], torch.finfo(dtype).max
    lam[::2] = -torch.rand(lam[::2].shape, device="cuda")  # every second channel decays fast
    fwd = GatedLinearRecurrenceFwdOp(B, T, D, dtype=dtype, save_states=True)
    bwd = GatedLinearRecurrenceBwdOp(B, T, D, dtype=dtype)
    first = None
    for xs, gs in ((0.0, 0.0), (most, most), (-most, 1.0), (most, -most), (1.0, -most)):
        x[:, shut], i[:, shut] = xs, gs
        out = fwd(x, i, r, lam, h0)
        out += bwd(dy, x, i, r, lam, out[2], h0, dT)
        for name, t in zip(NAMES[:3], out[3:6]):
            assert (t[:, shut] == 0).all(), (name, xs, gs)
        assert all(t.isfinite().all() for t in out), (xs, gs)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out)), (xs, gs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_tokens_repeat_the_state(dtype):
    """A run of 16 tokens is walked from one state: a padded token in it has its neighbour's y to
    the bit."""
    x, i, r, lam, h0, _, _, shut = _padded(90, 66, dtype)
    y, final = GatedLinearRecurrenceFwdOp(2, 90, 66, dtype=dtype)(x, i, r, lam, h0)
    for t in range(1, 90):
        if shut[t] and t % 16:
            assert torch.equal(y[:, t], y[:, t - 1]), t
    if dtype == torch.float32:
        assert torch.equal(final, y[:, -1])


# ------------------------------------------------------------ infinities stay what they are
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lam", [2.0, 30.0])  # decays of e^-8 and of e^-120 a token
@pytest.mark.parametrize("B, T, D", [(2, 150, 66), (1, 700, 272), (3, 600, 1024), (40, 300, 200)])
@pytest.mark.parametrize("packed", [False, True])
def test_infinities_outlive_any_decay(B, T, D, lam, packed, dtype):
    """a > 0 however strong: an infinite state stays infinite to its sequence's end, and an
    infinite gradient to its beginning, wherever the tokens are split; as token by token."""
    if packed:
        B, cu = 1, _cu([T // 3, 0, T - T // 3])
    else:
        cu = None
    (x, i, r, _), h0, dy, dT = _inputs(B, T, D, dtype, nseq=3 if packed else None)
    i, r, x = i.clamp(-3, 3), r.clamp(-3, 3), torch.where(x < 0, x - 0.1, x + 0.1)
    lam = torch.full((D,), lam, device="cuda")
    fwd = GatedLinearRecurrenceFwdOp(B, T, D, dtype=dtype, save_states=True)
    bwd = GatedLinearRecurrenceBwdOp(B, T, D, dtype=dtype)
    clean = fwd(x, i, r, lam, h0, cu)
    clean += bwd(dy, x, i, r, lam, clean[2], h0, dT, cu)
    inf = float("inf")
    h1, x1, dy1, dT1 = h0.clone(), x.clone(), dy.clone(), dT.clone()
    h1[0, 3], h1[-1, 8] = inf, -inf
    x1[0, T // 2, 5] = -inf
    dT1[-1, 17], dT1[0, 22], dy1[0, T // 2 + 3, 30] = -inf, inf, inf
    y, final, states = fwd(x1, i, r, lam, h1, cu)
    y_ref, f_ref, _, _ = ref.glr_fwd(x1, i, r, lam, h1, cu)
    dx, di, _, _, d0 = bwd(dy1, x1, i, r, lam, states, h1, dT1, cu)
    want, _ = ref.glr_bwd(dy1, x1, i, r, lam, h1, dT1, cu)
    assert y_ref.isinf().any() and want[0].isinf().any() and want[4].isinf().any()
    same = torch.ones(D, dtype=torch.bool, device="cuda")
    same[[3, 5, 8, 17, 22, 30]] = False
    for name, got, exact, before in (("y", y, y_ref, clean[0]), ("final", final, f_ref, clean[1]),
                                     ("dx", dx, want[0], clean[3]), ("d0", d0, want[4], clean[7]),
                                     ("di", di, want[1], clean[4])):
        assert torch.equal(got[..., same], before[..., same]), name
        if name == "di":  # x = -inf times 0 at one token, by the formula too
            got, exact = got[..., [17, 22, 30]], exact[..., [17, 22, 30]]
        got = got.cpu().double()
        assert not got.isnan().any(), name
        assert torch.equal(got.isinf() * got.sign(), exact.isinf() * exact.sign()), name


def test_infinities_token_by_token():
    D, inf = 66, float("inf")
    for lam in (2.0, 30.0):
        (x, i, r, _), h0, _, _ = _inputs(2, 30, D, torch.float32)
        h0[0, 3], h0[1, 4] = inf, -inf
        lam = torch.full((D,), lam, device="cuda")
        y_ref, _, _, _ = ref.glr_fwd(x, i, r, lam, h0)
        step = GatedLinearRecurrenceDecodeOp(2, D, dtype=torch.float32, inplace=True)
        for t in range(30):
            y, _ = step(x[:, t], i[:, t], r[:, t], lam, h0)
            assert not y.isnan().any()
            assert torch.equal(y.cpu().isinf(), y_ref[:, t].isinf())
