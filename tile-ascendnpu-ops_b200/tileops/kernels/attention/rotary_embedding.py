"""Rotary position kernels: queries and keys rotated, forward and backward.

Shims over ``tileops_rotary`` (formulas in ``csrc/rotary.cu``).  Rows whose
channels are contiguous are read in place whatever their other strides are
(column slices of one projection's output).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from tileops import _native
from tileops.kernels.attention._layouts import channels_last, row_of
from tileops.kernels.kernel_base import Kernel, check_dtype

__all__ = ["RotaryEmbeddingBwdKernel", "RotaryEmbeddingFwdKernel"]

MAX_ROTARY_DIM = 256
_TURNS_PER_RADIAN = 0x28be60db9391054a7f09d5f47d4d377036d8a5664f10e4107f9458  # 2^216 / 2 pi


def turns_array(frequencies: Sequence[float]) -> ctypes.Array:
    """Angles a token, in radians, as whole numbers of 2^-64 turns modulo one turn."""
    turns = []
    for f in frequencies:
        n, d = float(f).as_integer_ratio()  # d a power of two
        turns.append(((n * _TURNS_PER_RADIAN // d >> 151) + 1 >> 1) % 2**64)  # rounded
    return (ctypes.c_uint64 * max(1, len(turns)))(*turns)


def check_rotation(name: str, dim: int, rotary_dim: int, frequencies: Sequence[float],
                   amplitude: float) -> None:
    if not 0 <= rotary_dim <= min(dim, MAX_ROTARY_DIM) or rotary_dim % 2:
        raise ValueError(f"{name} supports an even rotary_dim up to dim and {MAX_ROTARY_DIM}, got "
                         f"{rotary_dim} of dim {dim}")
    if len(frequencies) != rotary_dim // 2:
        raise ValueError(f"frequencies must have rotary_dim / 2 = {rotary_dim // 2} values, got "
                         f"{len(frequencies)}")
    if not all(abs(f) < 2.0**64 for f in frequencies):
        raise ValueError("frequencies must be finite and below 2^64")
    if not abs(amplitude) <= torch.finfo(torch.float32).max:
        raise ValueError(f"amplitude must be a finite float32, got {amplitude}")


class _RotaryEmbeddingKernel(Kernel):
    SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
    BACKWARD = 0

    def __init__(self, batch: int, seq_len: int, heads: int, heads_kv: int, dim: int,
                 rotary_dim: int, interleaved: bool, frequencies: Sequence[float],
                 amplitude: float = 1.0, dtype: torch.dtype = torch.bfloat16,
                 config: Optional[dict] = None):
        super().__init__()
        check_dtype(self, dtype, self.SUPPORTED_DTYPES)
        if (min(batch, seq_len, heads, heads_kv) < 0 or max(batch, seq_len, batch * seq_len) >= 2**31
                or max(heads, heads_kv) > 4096 or not 1 <= dim <= 4096):
            raise ValueError(f"{type(self).__name__} supports fewer than 2^31 tokens, up to 4096 heads "
                             f"and dim 1..4096, got ({batch}, {seq_len}, {heads}, {heads_kv}, {dim})")
        check_rotation(type(self).__name__, dim, rotary_dim, frequencies, amplitude)
        self.batch, self.seq_len, self.heads, self.heads_kv = batch, seq_len, heads, heads_kv
        self.dim, self.rotary_dim, self.interleaved = dim, rotary_dim, bool(interleaved)
        self.amplitude = float(amplitude)
        self.dtype = dtype
        self._code = _native.dtype_code(dtype)
        self._turns = turns_array(frequencies)
        self.init_config(config)

    def plan(self, q, k, positions=None, inplace: bool = False):
        """What a call of this layout needs, for ``forward``: device, whether q, k and positions have
        to be copied, the stride array, the positions' stride and type, and the outputs' shapes."""
        copy = tuple(t is not None and not channels_last(t) and not inplace for t in (q, k))
        like = tuple(None if t is None or inplace else row_of(t) for t in (q, k))
        values = []
        for t, dense in (*zip((q, k), copy), (q, not inplace), (k, not inplace)):
            if t is None:
                values += (0, 0, 0)
            elif dense:
                values += (t.shape[1] * t.shape[2] * t.shape[3], t.shape[2] * t.shape[3], t.shape[3])
            else:
                values += t.stride()[:3]
        stride, code, copy_at = 0, 7, False
        if positions is not None:
            copy_at = positions.stride(-1) != 1
            if positions.dim() == 2:
                stride = positions.shape[1] if copy_at else positions.stride(0)
            code = 7 if positions.dtype is torch.int32 else 8
        return ((k if q is None else q).device, any(copy) or copy_at, (*copy, copy_at),
                (ctypes.c_int64 * 12)(*values), stride, code, like)

    def forward(self, q, k, positions=None, inplace: bool = False, plan=None):
        """Return ``(q_out, k_out)``; ``inplace`` writes over ``q`` and ``k``.  ``plan``: what
        ``plan()`` gave for arguments of the same layout."""
        if plan is None:
            plan = self.plan(q, k, positions, inplace)
        device, copies, copy, strides, stride, code, (q_like, k_like) = plan
        if copies:
            q, k, positions = (t.contiguous() if c else t for t, c in zip((q, k, positions), copy))
        q_out = q if q_like is None else torch.empty_like(q_like)
        k_out = k if k_like is None else torch.empty_like(k_like)
        _native.launch(
            "tileops_rotary", device, 0 if q is None else q.data_ptr(),
            0 if k is None else k.data_ptr(), 0 if positions is None else positions.data_ptr(),
            0 if q is None else q_out.data_ptr(), 0 if k is None else k_out.data_ptr(),
            self._turns, self.batch, self.seq_len, self.heads, self.heads_kv, self.dim,
            self.rotary_dim, strides, stride, code, self.interleaved, self.BACKWARD,
            self.amplitude, self._code)
        return q_out, k_out


class RotaryEmbeddingFwdKernel(_RotaryEmbeddingKernel):
    """Queries and keys rotated by their positions.

    Args:
        batch, seq_len, heads, heads_kv, dim: problem shape.
        rotary_dim: channels of a head that rotate, the first ones.
        interleaved: pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
        frequencies: the pairs' angles a token.
        amplitude: factor on the rotated channels.
        dtype: float32, float16 or bfloat16.
        config: Optional config dict (no tunables).
    """


class RotaryEmbeddingBwdKernel(_RotaryEmbeddingKernel):
    """Gradients of the forward: the transposed rotation; the same arguments."""

    BACKWARD = 1
