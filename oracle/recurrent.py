"""The recurrent-block operators in 64 bits, with error bounds (test infrastructure only).

Plain CPU implementations of the gated linear recurrence and the sandwich norm
(forward and backward) that take tensors of any type and compute in float64,
token by token and row by row.  They have no counterpart in the reference.

Next to a value each function can give a bound on how far an implementation in
fp32 may be from it, by a running error analysis with u = 2^-24 (half a step of
fp32, relative).  With la = log a and the gates' logits z:

* ex2.approx and rcp.approx are off by at most 4u and 2u, and -z log2(e) is
  rounded before the exponential, so sigmoid(z) is off by (|z| + 8) u;
* a = exp(la) is off by (|la| (|r| + 9) + 6) u: la's own error times |la|, then
  the exponential's (for |la| < 1/4 the error of a sum that starts with 1);
* m = sqrt(1 - a^2) is off by half of la's and q's errors, and by a's twice
  where 1 - a^2 is formed by a difference (la < -1/4, so 1 - a^2 > 0.39):
  at most (|r| + 16 + 4 |la| (|r| + 9) exp(2 la)) u;
* u_t = m sigma_i x_t adds sigma_i's error and two products;
* a scan may join the factors a in any order: one more rounding per token;
* what is subnormal in fp32 may be flushed to zero, a by ex2.approx.ftz itself: up to
  FLUSH = 2^-126 is lost where a is formed and where it enters a product, and later
  factors (k up to hundreds) multiply that loss;
* rcp.approx.ftz(1 + exp(-z)) is zero where sigmoid(z) < 2^-126: a decay gate that far down
  is shut exactly, so m ~ sqrt(2 k sigma_r) (at most 2^-62 sqrt(k)) is lost as a whole, and
  with it what m or sigma_r is a factor of.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

U = 2.0**-24
FLUSH = 2.0**-126


def _wide(t):
    return None if t is None else t.detach().cpu().double()


def _ranges(batch, seq_len, cu_seqlens):
    """(batch index, first token, end, sequence) of every sequence."""
    if cu_seqlens is None:
        return [(b, 0, seq_len, b) for b in range(batch)]
    cu = cu_seqlens.tolist()
    return [(0, cu[n], cu[n + 1], n) for n in range(len(cu) - 1)]


def _gates(x, i, r, lam, c):
    la = -c * F.softplus(lam, threshold=80) * torch.sigmoid(r)
    a = torch.exp(la)
    m = torch.sqrt(-torch.expm1(2 * la))
    return la, a, m, torch.sigmoid(i), torch.sigmoid(r)


def _shut(sr):
    return sr < 4 * FLUSH


def _gate_errors(x, i, r, la, a, m, si, sr):
    i, r = i.abs().clamp(max=200), r.abs().clamp(max=200)
    fall = torch.where(la < 0, -la, torch.zeros_like(la)).clamp(max=200)
    ea = a * (fall * (r + 9) + 6) * U + FLUSH
    em = (r + 16 + 4 * fall * (r + 9) * a * a) * U  # relative
    em = torch.where(_shut(sr), torch.ones_like(em), em)
    eu = (m * si * x).abs() * (em + (i + 12) * U) + FLUSH * (m * x).abs()
    return ea, em, eu


def glr_fwd(x, input_gate, decay_gate, decay_param, initial_state=None, cu_seqlens=None,
            decay_scale: float = 8.0):
    """``(y, final_state, y_bound, final_bound)``."""
    x, i, r, lam, h0 = map(_wide, (x, input_gate, decay_gate, decay_param, initial_state))
    B, T, D = x.shape
    la, a, m, si, sr = _gates(x, i, r, lam, decay_scale)
    u = m * si * x
    ea, _, eu = _gate_errors(x, i, r, la, a, m, si, sr)
    ranges = _ranges(B, T, cu_seqlens)
    y, ey = torch.zeros_like(x), torch.zeros_like(x)
    final = torch.zeros(len(ranges), D, dtype=torch.float64)
    efinal = torch.zeros_like(final)
    for b, t0, t1, n in ranges:
        h = h0[n].clone() if h0 is not None else torch.zeros(D, dtype=torch.float64)
        size, err = h.abs(), torch.zeros_like(h)
        for t in range(t0, t1):
            err = a[b, t] * err + (ea[b, t] + 2 * U * a[b, t]) * size + eu[b, t]
            size = a[b, t] * size + u[b, t].abs()
            h = a[b, t] * h + u[b, t]
            err = err + 2 * U * size
            y[b, t], ey[b, t] = h, err
        final[n], efinal[n] = h, err
    return y, final, ey, efinal


def glr_bwd(dy, x, input_gate, decay_gate, decay_param, initial_state=None, d_final_state=None,
            cu_seqlens=None, decay_scale: float = 8.0):
    """``(gradients, bounds)``, both (dx, d_input_gate, d_decay_gate, d_decay_param,
    d_initial_state)."""
    dy, x, i, r, lam, h0, dT = map(_wide, (dy, x, input_gate, decay_gate, decay_param,
                                           initial_state, d_final_state))
    B, T, D = x.shape
    la, a, m, si, sr = _gates(x, i, r, lam, decay_scale)
    ea, em, eu = _gate_errors(x, i, r, la, a, m, si, sr)
    y, _, ey, _ = glr_fwd(x, i, r, lam, h0, cu_seqlens, decay_scale)
    ranges = _ranges(B, T, cu_seqlens)
    hp, ehp, G, eG, sG = (torch.zeros_like(x) for _ in range(5))
    d0 = torch.zeros(len(ranges), D, dtype=torch.float64)
    e0 = torch.zeros_like(d0)
    for b, t0, t1, n in ranges:
        back = dT[n].clone() if dT is not None else torch.zeros(D, dtype=torch.float64)
        err, size = torch.zeros_like(back), back.abs()
        for t in reversed(range(t0, t1)):
            if t > t0:
                hp[b, t], ehp[b, t] = y[b, t - 1], ey[b, t - 1]
            elif h0 is not None:
                hp[b, t] = h0[n]
            G[b, t] = dy[b, t] + back
            sG[b, t] = dy[b, t].abs() + size
            eG[b, t] = err + 2 * U * sG[b, t]
            back = a[b, t] * G[b, t]
            size = a[b, t] * sG[b, t]
            err = a[b, t] * eG[b, t] + (ea[b, t] + 2 * U * a[b, t]) * sG[b, t]
        d0[n], e0[n] = back, err
    over_m = torch.where(m > 0, 1 / m.clamp(min=1e-300), torch.zeros_like(m))
    k = decay_scale * F.softplus(lam, threshold=80)
    dx = G * m * si
    di = dx * x * (1 - si)
    first, second = a * G * hp, G * si * x * a * a * over_m
    dla = first - second
    dr = -k * sr * (1 - sr) * dla
    terms = -sr * dla
    dlam = decay_scale * torch.sigmoid(lam) * terms.sum(dim=(0, 1))
    # |z| u of a logit's sigmoid, the factors' errors, and those of G and h.
    ai, ar = i.abs().clamp(max=200), r.abs().clamp(max=200)
    edx = m * si * eG + dx.abs() * (em + (ai + 12) * U) + FLUSH * (G * m).abs()
    edi = x.abs() * (1 - si) * edx + di.abs() * (ai + 16) * U + dx.abs() * x.abs() * 4 * U
    edla = (a * (eG * hp.abs() + G.abs() * ehp) + G.abs() * hp.abs() * (ea + 4 * a * U)
            + eG * (si * x * a * a * over_m).abs()
            + second.abs() * (em + (ai + 20) * U) + 2 * (G * si * x * a * over_m).abs() * ea
            + 4 * FLUSH)
    gone = _shut(sr).double()  # sigma_r as a factor
    edr = gone * dr.abs() + k * sr * (1 - sr) * edla + dr.abs() * (ar + 24) * U + k * sr * dla.abs() * 4 * U
    # Sums of up to 512 terms in a row, then partial sums of those.
    eterms = (sr * edla + gone * terms.abs() + terms.abs() * (ar + 12) * U).sum(dim=(0, 1))
    edlam = (decay_scale * torch.sigmoid(lam)
             * (eterms + 600 * U * terms.abs().sum(dim=(0, 1))) + dlam.abs() * 16 * U)
    return (dx, di, dr, dlam, d0), (edx, edi, edr, edlam, e0)


def glr_states(x, input_gate, decay_gate, decay_param, initial_state=None, decay_scale=8.0,
               segment: int = 32):
    """The state before every ``segment`` tokens, and its bound (no packed sequences)."""
    h0 = _wide(initial_state)
    y, _, ey, _ = glr_fwd(x, input_gate, decay_gate, decay_param, initial_state,
                          decay_scale=decay_scale)
    first = h0 if h0 is not None else torch.zeros_like(y[:, 0])
    states = torch.cat([first[:, None], y[:, segment - 1::segment]], dim=1)
    bound = torch.cat([torch.zeros_like(first)[:, None], ey[:, segment - 1::segment]], dim=1)
    n = -(-x.shape[1] // segment)
    return states[:, :n], bound[:, :n]


# ------------------------------------------------------------ sandwich norm
# One fp32 sum over a row: at most 48 terms in a row per thread, then a tree.
ROW = 64 * U


def _norm(v, layer, eps):
    """Normalised rows, 1 / deviation, and a bound on the normalised rows' error."""
    mean = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[..., :1])
    centre = v - mean
    rstd = 1 / torch.sqrt(centre.square().mean(-1, keepdim=True) + eps)
    hat = centre * rstd
    size = v.abs().mean(-1, keepdim=True) if layer else 0.0
    e_centre = ROW * size + 2 * U * (v.abs() + size)
    return hat, rstd, rstd * e_centre + hat.abs() * (ROW + rstd * rstd * 2
                                                    * (centre.abs() * e_centre).mean(-1, keepdim=True))


def _rows(gate, shape):
    """The gate of every row."""
    M, N = shape
    if gate is None:
        return torch.ones(1, N, dtype=torch.float64).expand(M, N)
    gate = gate.view(-1, N)
    return gate.repeat_interleave(M // gate.shape[0], dim=0)


def sandwich_stream(x, residual, post_weight, gate=None, post_bias=None, norm="rms", eps=1e-6,
                    residual_scale=1.0):
    """``(s, bound)`` before rounding, of (M, N) rows."""
    x, residual, w, gate, b = map(_wide, (x, residual, post_weight, gate, post_bias))
    hat, _, ehat = _norm(x, norm == "layer", eps)
    g = _rows(gate, x.shape)
    b = torch.zeros_like(w) if b is None else b
    s = residual_scale * residual + g * (hat * w + b)
    size = (residual_scale * residual).abs() + (g * hat * w).abs() + (g * b).abs()
    return s, (g * w).abs() * ehat + 6 * U * size


def sandwich_next(residual_out, pre_weight, pre_bias=None, norm="rms", eps=1e-6):
    """``(y, bound)`` from the rounded stream."""
    s, w, b = map(_wide, (residual_out, pre_weight, pre_bias))
    hat, _, ehat = _norm(s, norm == "layer", eps)
    b = torch.zeros_like(w) if b is None else b
    return hat * w + b, w.abs() * ehat + 4 * U * ((hat * w).abs() + b.abs())


def sandwich_bwd(dy, d_residual_out, x, residual_out, post_weight, pre_weight, gate=None,
                 post_bias=None, norm="rms", eps=1e-6, residual_scale=1.0):
    """``(gradients, bounds)``: (dx, d_residual, d_post_weight, d_pre_weight, d_gate,
    d_post_bias, d_pre_bias), d_gate (G, N)."""
    dy, ds, x, s, w1, w2, gate, b1 = map(_wide, (dy, d_residual_out, x, residual_out, post_weight,
                                                 pre_weight, gate, post_bias))
    M, N = x.shape
    layer = norm == "layer"
    ds = torch.zeros_like(dy) if ds is None else ds
    b1 = torch.zeros_like(w1) if b1 is None else b1
    groups = 1 if gate is None else gate.view(-1, N).shape[0]
    g = _rows(gate, x.shape)
    xh, xr, exh = _norm(x, layer, eps)
    sh, sr, esh = _norm(s, layer, eps)

    def back(v, ev, hat, ehat, rstd):
        """rstd (v - [mean v] - hat mean(v hat)) and its bound, v known to ev."""
        mean = v.mean(-1, keepdim=True) if layer else 0.0
        dot = (v * hat).mean(-1, keepdim=True)
        out = rstd * (v - mean - hat * dot)
        size = v.abs() + (v.abs().mean(-1, keepdim=True) if layer else 0.0)
        e_dot = (v.abs() * ehat + ev * hat.abs() + ROW * (v * hat).abs()).mean(-1, keepdim=True)
        e_mean = (ev.mean(-1, keepdim=True) + ROW * v.abs().mean(-1, keepdim=True)) if layer else 0.0
        bound = rstd * (ev + e_mean + ehat * dot.abs() + hat.abs() * e_dot
                        + 8 * U * (size + (hat * dot).abs())) + ROW * out.abs()
        # the deviation's own error, through the mean's where a mean is taken
        bound = bound + out.abs() * (ehat * hat.abs()).mean(-1, keepdim=True) * 2
        return out, bound

    f = dy * w2
    t, et = back(f, 2 * U * f.abs(), sh, esh, sr)
    t, et = ds + t, et + 2 * U * (ds.abs() + t.abs())
    e = t * g * w1
    dx, edx = back(e, et * (g * w1).abs() + 3 * U * e.abs(), xh, exh, xr)

    def columns(v, ev, grouped=False):
        """Column sums, at most 1024 rows in a row, then partial sums."""
        v, ev = (q.view(groups, M // groups, N).sum(1) for q in (v, ev + 1100 * U * v.abs()))
        return (v, ev) if grouped else (v.sum(0), ev.sum(0))

    P, eP = columns(t * xh, t.abs() * exh + et * xh.abs() + 2 * U * (t * xh).abs(), True)
    Q, eQ = columns(t, et, True)
    gg = torch.ones(1, N, dtype=torch.float64) if gate is None else gate.view(-1, N)
    d_gate = w1 * P + b1 * Q
    e_gate = w1.abs() * eP + b1.abs() * eQ + 4 * U * ((w1 * P).abs() + (b1 * Q).abs())

    def over_groups(v, ev):
        n = (4 + groups) * U
        return (gg * v).sum(0), (gg.abs() * ev + n * (gg * v).abs()).sum(0)

    d_post, e_post = over_groups(P, eP)
    d_post_bias, e_post_bias = over_groups(Q, eQ)
    d_pre, e_pre = columns(dy * sh, dy.abs() * esh + 2 * U * (dy * sh).abs())
    d_pre_bias, e_pre_bias = columns(dy, torch.zeros_like(dy))
    return ((dx, residual_scale * t, d_post, d_pre, d_gate, d_post_bias, d_pre_bias),
            (edx, abs(residual_scale) * (et + U * t.abs()), e_post, e_pre, e_gate, e_post_bias,
             e_pre_bias))


# ------------------------------------------------------------ comparison
def assert_within(got, want, bound, what=""):
    """``got`` is the rounding of a value within ``bound`` of ``want``: half a step of its type
    more (eps / 2 relative, half the smallest subnormal near zero)."""
    info = torch.finfo(got.dtype)
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    half = info.eps / 2 if got.numel() else 0.0
    limit = bound + half * (want.abs() + bound) + info.smallest_normal * info.eps / 2
    limit = limit + 2 * FLUSH  # the last product and the output
    off = (got - want).abs()
    bad = ~(off <= limit)
    if bad.any():
        at = tuple(int(v) for v in bad.nonzero()[0])
        worst = float((off / limit).nan_to_num(nan=float("inf")).max())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values beyond the bound "
                             f"(worst {worst:.3g} times it), first at {at}: got {float(got[at])!r}, "
                             f"want {float(want[at])!r} +- {float(limit[at])!r}")
