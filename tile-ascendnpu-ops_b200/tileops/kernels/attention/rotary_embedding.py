"""Rotary position kernels: queries and keys rotated, forward and backward.

Shims over ``tileops_rotary`` (formulas in ``csrc/rotary.cu``).  Rows whose
channels are contiguous are read in place whatever their other strides are
(column slices of one projection's output).
"""

from __future__ import annotations

import ctypes
import math
from fractions import Fraction
from typing import Optional, Sequence

import torch

from tileops import _native
from tileops.kernels.kernel_base import Kernel, check_dtype

__all__ = ["RotaryEmbeddingBwdKernel", "RotaryEmbeddingFwdKernel"]

MAX_ROTARY_DIM = 256
_TURNS_PER_RADIAN = Fraction("0.15915494309189533576888376337251436203445964574046")  # 1 / 2 pi
_KEPT = 64  # layouts an op keeps the stride arrays of


def turns_array(frequencies: Sequence[float]) -> ctypes.Array:
    """Angles a token, in radians, as whole numbers of 2^-64 turns modulo one turn."""
    turns = [round(Fraction(f) * _TURNS_PER_RADIAN * 2**64) % 2**64 for f in frequencies]
    return (ctypes.c_uint64 * max(1, len(turns)))(*turns)


def check_rotation(name: str, dim: int, rotary_dim: int, frequencies: Sequence[float],
                   amplitude: float) -> None:
    if not 0 <= rotary_dim <= min(dim, MAX_ROTARY_DIM) or rotary_dim % 2:
        raise ValueError(f"{name} supports an even rotary_dim up to dim and {MAX_ROTARY_DIM}, got "
                         f"{rotary_dim} of dim {dim}")
    if len(frequencies) != rotary_dim // 2:
        raise ValueError(f"frequencies must have rotary_dim / 2 = {rotary_dim // 2} values, got "
                         f"{len(frequencies)}")
    if not all(math.isfinite(f) for f in frequencies):
        raise ValueError("frequencies must be finite")
    if not abs(amplitude) <= torch.finfo(torch.float32).max:
        raise ValueError(f"amplitude must be a finite float32, got {amplitude}")


def overlaps(shape: Sequence[int], strides: Sequence[int]) -> bool:
    """Whether two indices of a tensor can share an element (never wrongly no)."""
    reach = 0
    for stride, size in sorted((st, n) for st, n in zip(strides, shape) if n > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


def dense_like(t: torch.Tensor) -> torch.Tensor:
    """A dense output of ``t``'s shape and type (``empty_like`` costs the host half of what
    ``empty`` does, but takes over the order of ``t``'s strides)."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def channels_last(t: torch.Tensor) -> torch.Tensor:
    """``t``, copied only when its channels are not contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _RotaryEmbeddingKernel(Kernel):
    SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
    BACKWARD = 0

    def __init__(self, batch: int, seq_len: int, heads: int, heads_kv: int, dim: int,
                 rotary_dim: int, interleaved: bool, frequencies: Sequence[float],
                 amplitude: float = 1.0, dtype: torch.dtype = torch.bfloat16,
                 config: Optional[dict] = None):
        super().__init__()
        check_dtype(self, dtype, self.SUPPORTED_DTYPES)
        if (min(batch, seq_len, heads, heads_kv) < 0 or max(batch, seq_len) > 2**31 - 1
                or max(heads, heads_kv) > 4096 or not 1 <= dim <= 4096):
            raise ValueError(f"{type(self).__name__} supports batch and seq_len below 2^31, up to "
                             f"4096 heads and dim 1..4096, got ({batch}, {seq_len}, {heads}, "
                             f"{heads_kv}, {dim})")
        check_rotation(type(self).__name__, dim, rotary_dim, frequencies, amplitude)
        self.batch, self.seq_len, self.heads, self.heads_kv = batch, seq_len, heads, heads_kv
        self.dim, self.rotary_dim, self.interleaved = dim, rotary_dim, bool(interleaved)
        self.amplitude = float(amplitude)
        self.dtype = dtype
        self._code = _native.dtype_code(dtype)
        self._turns = turns_array(frequencies)
        self._strides: dict = {}
        self.init_config(config)

    def _stride_array(self, q, k, q_out, k_out):
        key = tuple(None if t is None else t.stride() for t in (q, k, q_out, k_out))
        found = self._strides.get(key)
        if found is None:
            if len(self._strides) >= _KEPT:
                self._strides.clear()
            found = (ctypes.c_int64 * 12)(*(v for s in key for v in (s[:3] if s else (0, 0, 0))))
            self._strides[key] = found
        return found

    def forward(self, q, k, positions=None, inplace: bool = False):
        """Return ``(q_out, k_out)``; ``inplace`` writes over ``q`` and ``k``."""
        if inplace:
            q_out, k_out = q, k
        else:
            q = None if q is None else channels_last(q)
            k = None if k is None else channels_last(k)
            q_out = None if q is None else dense_like(q)
            k_out = None if k is None else dense_like(k)
        stride, code = 0, 7
        if positions is not None:
            if positions.stride(-1) != 1:
                positions = positions.contiguous()
            stride = positions.stride(0) if positions.dim() == 2 else 0
            code = 7 if positions.dtype is torch.int32 else 8
        _native.launch(
            "tileops_rotary", (k if q is None else q).device, _native.data_ptr(q),
            _native.data_ptr(k), _native.data_ptr(positions), _native.data_ptr(q_out),
            _native.data_ptr(k_out), self._turns, self.batch, self.seq_len, self.heads,
            self.heads_kv, self.dim, self.rotary_dim, self._stride_array(q, k, q_out, k_out),
            stride, code, self.interleaved, self.BACKWARD, self.amplitude, self._code)
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
