"""Rotary positions, the paged cache and single-token attention in 64 bits, with error bounds
(test infrastructure only; the reference has no such operators).

Plain CPU implementations that take tensors of any type and compute in float64, position after
position and sequence after sequence.  The bounds say how far an implementation in fp32 may be,
with u = 2^-24 (half a step of fp32, relative):

* an angle reaches sin and cos as a fraction of half a turn, cut to 2^-31 and rounded to fp32: off by
  2^-25 + 2^-31 half turns and the position's 2^-64 a token, below 1.7 u in sin or cos; the functions
  add 2 ulp (2 u below 1), the amplitude one rounding: 5 u.  A rotated channel adds two products and a
  sum: 8 u times amplitude (|x_a| + |x_b|) in all;
* a score is a sum of D products that are exact in fp32.  The matrix instructions may cut, not round,
  each sum: 2 u a term, (D + 16) 2 u sum |q k| (nothing where q and k are whole numbers so small that
  every sum is exact);
* a weight exp2(t - base): t and the difference round (4 u of the largest |t|), ex2.approx is off by 4 u;
* up to 8 query heads a key head the weights enter the second product as two numbers of the inputs'
  type, half a step of half a step off; those of more heads are rounded once, half a step off.  Sums of n
  terms may cut each term.
"""

from __future__ import annotations

import math
from fractions import Fraction

import torch

U = 2.0**-24
_TURNS_PER_RADIAN = Fraction("0.159154943091895335768883763372514362034459645740456448747667")


def _wide(t):
    return None if t is None else t.detach().cpu().double()


# ------------------------------------------------------------ rotary positions
def angles(positions, frequencies):
    """Position times frequency modulo a turn, in radians: whole-number arithmetic, so far
    positions lose nothing."""
    turns = [Fraction(f) * _TURNS_PER_RADIAN for f in frequencies]
    whole = [round(t * 2**160) for t in turns]
    flat = positions.detach().cpu().reshape(-1).tolist()
    rows = [[((p * w) % 2**160) / 2**160 * math.tau for w in whole] for p in flat]
    out = torch.tensor(rows, dtype=torch.float64).reshape(len(flat), len(whole))
    return out.reshape(*positions.shape, len(whole))


def rotate(x, positions, frequencies, amplitude=1.0, interleaved=False, backward=False):
    """``(value, bound)`` of x (..., heads, dim) at positions (...)."""
    x = _wide(x)
    r = 2 * len(frequencies)
    a = angles(positions, frequencies)[..., None, :]
    c, s = amplitude * torch.cos(a), amplitude * torch.sin(a)
    if backward:
        s = -s
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    out, bound = x.clone(), torch.zeros_like(x)
    xa, xb = x[..., first], x[..., second]
    out[..., first], out[..., second] = c * xa - s * xb, s * xa + c * xb
    off = 8 * U * abs(amplitude) * (xa.abs() + xb.abs())
    bound[..., first], bound[..., second] = off, off
    return out, bound


# ------------------------------------------------------------ paged cache
def new_rows(batch, tokens, seq_lens, cu_seqlens=None):
    """``(row, sequence, position)`` of every new token that is no padding; a row is the index
    among all tokens."""
    lens, out = seq_lens.tolist(), []
    for b in range(batch):
        begin, end = (b * tokens, (b + 1) * tokens) if cu_seqlens is None else (
            int(cu_seqlens[b]), int(cu_seqlens[b + 1]))
        for row in range(begin, end):
            position = lens[b] - (end - row)
            if position >= 0:
                out.append((row, b, position))
    return out


def append(k, v, k_cache, v_cache, page_table, seq_lens, frequencies=(), q=None, cu_seqlens=None,
           amplitude=1.0, interleaved=False):
    """``(q_out, q_bound, k_cache, k_bound, v_cache)`` in float64; q_out is None without q."""
    P = k_cache.shape[1]
    if cu_seqlens is None:
        batch, tokens = k.shape[0], k.shape[1] if k.dim() == 4 else 1
    else:
        batch, tokens = cu_seqlens.numel() - 1, None
    shape = None if q is None else q.shape
    k, v = (_wide(t).reshape(-1, *t.shape[-2:]) for t in (k, v))
    q = None if q is None else _wide(q).reshape(-1, *q.shape[-2:])
    kc, vc = _wide(k_cache).clone(), _wide(v_cache).clone()
    bound = torch.zeros_like(kc)
    table = page_table.tolist()
    q_out = None if q is None else torch.zeros_like(q)
    q_bound = None if q is None else torch.zeros_like(q)
    for row, b, p in new_rows(batch, tokens, seq_lens, cu_seqlens):
        at = torch.tensor(p)
        page, slot = table[b][p // P], p % P
        kc[page, slot], bound[page, slot] = rotate(k[row], at, frequencies, amplitude, interleaved)
        vc[page, slot] = v[row]
        if q is not None:
            q_out[row], q_bound[row] = rotate(q[row], at, frequencies, amplitude, interleaved)
    if q is not None:
        q_out, q_bound = q_out.reshape(shape), q_bound.reshape(shape)
    return q_out, q_bound, kc, bound, vc


# ------------------------------------------------------------ single-token attention
def attend(q, k_cache, v_cache, page_table, seq_lens, scale=None, window=None,
           exact_scores=False):
    """``(o, lse, o_bound, lse_bound)``; the bounds count what weights in q's type are off by."""
    half = torch.finfo(q.dtype).eps / 2
    B, H, D = q.shape
    P, Hkv = k_cache.shape[1], k_cache.shape[2]
    if H // Hkv <= 8:
        half *= half
    scale = D**-0.5 if scale is None else scale
    q = _wide(q)
    kc, vc = k_cache.detach().cpu(), v_cache.detach().cpu()
    table = page_table.cpu().long()
    o, o_bound = torch.zeros(2, B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros(B, H, dtype=torch.float64)
    for b, n in enumerate(seq_lens.tolist()):
        first = max(0, n - window) if window else 0
        if n <= 0:
            continue
        at = torch.arange(first, n)
        k, v = (c[table[b, at // P], at % P].double() for c in (kc, vc))  # (n, Hkv, D)
        for h in range(H):
            kh, vh = k[:, h // (H // Hkv)], v[:, h // (H // Hkv)]
            t = (kh @ q[b, h]) * (scale / math.log(2.0))
            top = t.max()
            w = torch.exp2(t - top)
            total = w.sum()
            o[b, h] = (w @ vh) / total
            lse[b, h] = top + math.log2(total)
            e_t = 0.0 if exact_scores else (
                2 * U * (D + 16) * (kh.abs() @ q[b, h].abs()).max() * abs(scale) / math.log(2.0))
            largest = t.abs().max() + 15  # fp16 weights are taken relative to 2^-15 of the largest
            e_w = math.log(2.0) * (e_t + 4 * U * largest) + 8 * U
            terms = 2 * U * (len(at) + 64)
            size = (w @ vh.abs()) / total
            o_bound[b, h] = size * (e_w + half + terms) + o[b, h].abs() * (e_w + terms)
            # weights below the type's smallest normal number (times 2^15 in fp16)
            o_bound[b, h] += len(at) * 2.0**-39 * vh.abs().amax(0) / total
            lse_bound[b, h] = (e_w + terms) / math.log(2.0) + 4 * U * (lse[b, h].abs() + largest)
    return o, lse, o_bound, lse_bound
