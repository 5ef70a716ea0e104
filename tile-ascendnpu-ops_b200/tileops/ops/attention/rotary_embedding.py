"""Rotary position ops: queries and keys rotated by their positions, and the gradients.

For pair i of a head at position p, with ``c, s = amplitude * cos, sin(p * frequencies[i])``::

    x'[a] = c x[a] - s x[b]        (a, b) = (i, i + rotary_dim / 2), or with
    x'[b] = s x[a] + c x[b]        interleaved (2 i, 2 i + 1)

in fp32, rounded once; channels from ``rotary_dim`` on pass unchanged.  Angles are exact whatever
the position (whole multiples of 2^-64 turns), so no table bounds the length.

    RotaryEmbeddingFwdOp(batch, seq_len, heads, heads_kv, dim, rotary_dim=None, interleaved=False,
                         frequencies=None, amplitude=1.0, dtype=torch.bfloat16, inplace=False,
                         kernel_map=None)
    forward(q, k, positions=None) -> (q_out, k_out)

    RotaryEmbeddingBwdOp(...the same...)
    forward(dq, dk, positions=None) -> (dq_in, dk_in)

q (batch, seq_len, heads, dim) and k (batch, seq_len, heads_kv, dim) of ``dtype``, the layout of
MultiHeadAttentionFwdOp; column slices of a wider tensor are read in place.  positions: integers
(seq_len,) or (batch, seq_len), any sign; None is 0, 1, ....  With heads_kv 0, k is None.
``inplace`` writes over q and k (contiguous channels, no element twice, in one or in both) and
returns them.  Like every op here, these build no autograd graph: a training loop calls the two
ops itself.

``rotary_frequencies`` makes the angles, also those scaled for long contexts.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Sequence

import torch

from tileops.device import get_device_backend
from tileops.kernels.attention import RotaryEmbeddingBwdKernel, RotaryEmbeddingFwdKernel
from tileops.kernels.attention._layouts import (
    NO_PLAN,
    Apart,
    Layouts,
    channels_last,
    layout_of,
    overlaps,
    plan_of,
)
from tileops.kernels.kernel_base import Kernel
from tileops.ops.attention._arguments import check_tensor
from tileops.ops.op_base import Op

__all__ = ["RotaryEmbeddingBwdOp", "RotaryEmbeddingFwdOp", "rotary_frequencies"]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, factor: float = 1.0,
                       original_length: Optional[int] = None, slow_turns: float = 1.0,
                       fast_turns: float = 32.0) -> tuple:
    """Angles a token of the rotary_dim / 2 pairs, ``base ** (-2 i / rotary_dim)``, in 64 bits.

    ``factor`` stretches them to a context that many times as long: all alike without
    ``original_length`` (positions interpolated); with it by parts: a pair that turns less than
    ``slow_turns`` times over ``original_length`` tokens is slowed down by ``factor``, one of more
    than ``fast_turns`` stays, a linear ramp in its turns between them.  (For a stretched base,
    pass ``base * factor ** (rotary_dim / (rotary_dim - 2))``; the ops' ``amplitude`` takes the
    1 + 0.1 ln(factor) that goes with stretching by parts.)
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    if not 0 < base < math.inf or not 0 < factor < math.inf:
        raise ValueError(f"base and factor must be positive and finite, got {base} and {factor}")
    if original_length is not None and (original_length < 1 or not slow_turns < fast_turns):
        raise ValueError("stretching by parts takes an original_length of at least 1 and slow_turns "
                         f"below fast_turns, got {original_length}, {slow_turns} and {fast_turns}")
    out = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        kept = 0.0
        if original_length is not None:
            turns = original_length * f / (2.0 * math.pi)
            kept = min(1.0, max(0.0, (turns - slow_turns) / (fast_turns - slow_turns)))
        out.append(f * (kept + (1.0 - kept) / factor))
    return tuple(out)


class _RotaryEmbeddingOp(Op):
    _names = ("q", "k")

    def __init__(self, batch: int, seq_len: int, heads: int, heads_kv: int, dim: int,
                 rotary_dim: Optional[int] = None, interleaved: bool = False,
                 frequencies: Optional[Sequence[float]] = None, amplitude: float = 1.0,
                 dtype: torch.dtype = torch.bfloat16, inplace: bool = False,
                 kernel_map: Optional[Dict[str, Kernel]] = None) -> None:
        self.batch, self.seq_len = batch, seq_len
        self.heads, self.heads_kv, self.dim = heads, heads_kv, dim
        self.rotary_dim = dim if rotary_dim is None else rotary_dim
        self.interleaved = interleaved
        self.frequencies = (rotary_frequencies(self.rotary_dim) if frequencies is None
                            else tuple(float(f) for f in frequencies))
        self.amplitude = amplitude
        self.dtype = dtype
        self.inplace = inplace
        self.dispatch_kernel(kernel_map)
        (name,) = self.default_kernel_map
        self.kernel = self.kernel_map[name](batch, seq_len, heads, heads_kv, dim, self.rotary_dim,
                                            interleaved, self.frequencies, amplitude, dtype)
        self._shapes = (batch, seq_len, heads, dim), (batch, seq_len, heads_kv, dim)
        self._plans = Layouts()  # of the arguments that were found right
        self._apart = Layouts()  # in place: of q and k

    def forward(self, q: Optional[torch.Tensor], k: Optional[torch.Tensor],
                positions: Optional[torch.Tensor] = None):
        layout = layout_of(q, k, positions)
        plan = self._plans.get(layout)
        if plan is None:
            self._check(q, k, positions)
            if q is None and k is None:
                return None, None
            plan = self._plans.keep(layout, plan_of(self.kernel, q, k, positions, self.inplace))
        if self.inplace and q is not None and k is not None:
            apart = self._apart.get(layout) or self._apart.keep(layout, Apart(q, k))
            if not apart(q.data_ptr(), k.data_ptr()):
                raise ValueError(f"{self._names[0]} and {self._names[1]} share memory: they cannot "
                                 "both be rotated in place")
        if plan is NO_PLAN:
            return self.kernel(q, k, positions, self.inplace)
        return self.kernel.forward(q, k, positions, self.inplace, plan)

    def _check(self, q, k, positions) -> None:
        dev = getattr(k if q is None else q, "device", None)
        for name, t, shape in zip(self._names, (q, k), self._shapes):
            if t is not None or shape[2]:
                check_tensor(dev, name, t, shape, self.dtype)
                if self.inplace:
                    self._check_inplace(name, t)
        if positions is not None:
            backend = get_device_backend()
            if not backend.is_device_tensor(positions):
                raise ValueError(f"positions must be a {backend.name} tensor, got "
                                 f"{getattr(positions, 'device', type(positions).__name__)}")
            if positions.device != dev:
                raise ValueError(f"Expected positions on {dev}, got {positions.device}")
            if positions.shape not in ((self.seq_len,), (self.batch, self.seq_len)):
                raise ValueError(f"Expected positions.shape ({self.seq_len},) or ({self.batch}, "
                                 f"{self.seq_len}), got {tuple(positions.shape)}")
            if positions.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")

    @staticmethod
    def _check_inplace(name: str, t: torch.Tensor) -> None:
        if not channels_last(t):
            raise ValueError(f"{name} must have contiguous channels when it is rotated in place")
        if overlaps(t.shape, t.stride()):
            raise ValueError(f"{name} has elements that share memory: it cannot be rotated in place")

    def eval_roofline(self) -> tuple[int, int]:
        """``(3 * B * S * (H + Hkv) * rotary_dim, 2 * B * S * (H + Hkv) * dim * elem_bytes)``."""
        rows = self.batch * self.seq_len * (self.heads + self.heads_kv)
        return 3 * rows * self.rotary_dim, 2 * rows * self.dim * self.dtype.itemsize


class RotaryEmbeddingFwdOp(_RotaryEmbeddingOp):
    """Queries and keys rotated by their positions.

    Args:
        batch, seq_len, heads, heads_kv, dim: Problem shape.
        rotary_dim: Channels of a head that rotate, the first ones (default: all), even, up to 256.
        interleaved: Pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
        frequencies: The pairs' angles a token (default: ``rotary_frequencies(rotary_dim)``).
        amplitude: Factor on the rotated channels.
        dtype: float32, float16 or bfloat16.
        inplace: Write over q and k and return them.
        kernel_map: Optional override of ``"rotary_fwd"``.
    """

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"rotary_fwd": RotaryEmbeddingFwdKernel}


class RotaryEmbeddingBwdOp(_RotaryEmbeddingOp):
    """Gradients of the rotary positions: the transposed rotation of dq and dk.

    Args:
        batch, seq_len, heads, heads_kv, dim, rotary_dim, interleaved, frequencies, amplitude,
            dtype: Those of the forward op.
        inplace: Write over dq and dk and return them.
        kernel_map: Optional override of ``"rotary_bwd"``.
    """

    _names = ("dq", "dk")

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"rotary_bwd": RotaryEmbeddingBwdKernel}
