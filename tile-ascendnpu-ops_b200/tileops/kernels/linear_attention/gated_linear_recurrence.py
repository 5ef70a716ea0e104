"""Gated linear recurrence kernels: forward, backward and one decode step.

Shims over ``tileops_glr_fwd``, ``tileops_glr_bwd`` and
``tileops_glr_decode_fwd`` (formulas in ``csrc/recurrence.cu``).  Row inputs
may be views whose channels are contiguous (column slices of a projection's
output): their batch and token strides go to the kernel and nothing is copied.
"""

from __future__ import annotations

from typing import Optional

import torch

from tileops import _native
from tileops.kernels.kernel_base import Kernel, check_dtype

__all__ = ["GatedLinearRecurrenceBwdKernel", "GatedLinearRecurrenceDecodeKernel",
           "GatedLinearRecurrenceFwdKernel"]

SEGMENT = 32  # tokens between two saved states (TILEOPS_GLR_SEGMENT)


def _channels_last(t: torch.Tensor) -> torch.Tensor:
    """``t``, copied only when its channels are not contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows_like(t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
    """A dense output (``empty_like`` costs the host half of what ``empty`` does, but takes over
    the order of ``t``'s strides: rows that overlap, strides (1, 1), give a transposed one)."""
    if t.dtype is dtype and t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(shape, dtype=dtype, device=t.device)


class _GatedLinearRecurrenceKernel(Kernel):
    SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)

    def __init__(self, batch: int, seq_len: int, dim: int, decay_scale: float = 8.0,
                 dtype: torch.dtype = torch.bfloat16, config: Optional[dict] = None):
        super().__init__()
        check_dtype(self, dtype, self.SUPPORTED_DTYPES)
        if (min(batch, seq_len) < 0 or dim < 1 or batch > 65535 or seq_len > 2**31 - 2**16
                or dim > 2**31 - 1):
            raise ValueError(f"{type(self).__name__} supports batch 0..65535, seq_len "
                             f"0..2^31 - 2^16 and dim 1..2^31 - 1, got ({batch}, {seq_len}, {dim})")
        fp32 = torch.finfo(torch.float32)  # what the kernels compute with
        if not fp32.tiny <= decay_scale <= fp32.max:
            raise ValueError(f"decay_scale must be positive and a normal float32, got {decay_scale}")
        self.batch, self.seq_len, self.dim = batch, seq_len, dim
        self.decay_scale = float(decay_scale)
        self.dtype = dtype
        self._code = _native.dtype_code(dtype)
        self._ws_bytes: Optional[int] = None
        self.init_config(config)

    def _sequences(self, cu_seqlens, device):
        """Device int32 offsets (or None) and the number of sequences."""
        if cu_seqlens is None:
            return None, self.batch
        if cu_seqlens.dtype is torch.int64:  # saturated: a cast alone would wrap 2^32 + n to n
            cu_seqlens = cu_seqlens.clamp(-1, 2**31 - 1)
        return (cu_seqlens.to(device=device, dtype=torch.int32).contiguous(),
                cu_seqlens.numel() - 1)


class GatedLinearRecurrenceFwdKernel(_GatedLinearRecurrenceKernel):
    """Forward over whole sequences.

    Args:
        batch, seq_len, dim: problem shape.
        decay_scale: c in ``log a = -c softplus(decay_param) sigmoid(decay_gate)``.
        dtype: float32, float16 or bfloat16.
        config: Optional config dict (no tunables).
    """

    def forward(self, x, input_gate, decay_gate, decay_param, initial_state=None,
                cu_seqlens=None, save_states: bool = False):
        """Return ``(y, final_state, states)``; states is None unless asked for."""
        B, T, D, dev = self.batch, self.seq_len, self.dim, x.device
        cu, nseq = self._sequences(cu_seqlens, dev)
        if initial_state is not None:
            initial_state = initial_state.contiguous()
        y = _rows_like(x, self.dtype, (B, T, D))
        states = (torch.empty((B, -(-T // SEGMENT), D), dtype=torch.float32, device=dev)
                  if save_states else None)
        if B == 0 or T == 0 or nseq == 0:  # no token anywhere: every sequence ends where it began
            final = (torch.zeros((nseq, D), dtype=torch.float32, device=dev)
                     if initial_state is None else initial_state.detach().clone())
            return y, final, states
        final = (torch.empty((nseq, D), dtype=torch.float32, device=dev)
                 if initial_state is None else torch.empty_like(initial_state))
        x, input_gate, decay_gate = map(_channels_last, (x, input_gate, decay_gate))
        decay_param = decay_param.contiguous()
        _native.launch(
            "tileops_glr_fwd", dev, x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(),
            decay_param.data_ptr(), _native.data_ptr(initial_state), _native.data_ptr(cu), nseq,
            y.data_ptr(), final.data_ptr(), _native.data_ptr(states), B, T, D,
            x.stride(0), x.stride(1), input_gate.stride(0), input_gate.stride(1),
            decay_gate.stride(0), decay_gate.stride(1), self.decay_scale, self._code)
        return y, final, states


class GatedLinearRecurrenceBwdKernel(_GatedLinearRecurrenceKernel):
    """Gradients of the forward; the same arguments."""

    def forward(self, dy, x, input_gate, decay_gate, decay_param, states, initial_state=None,
                d_final_state=None, cu_seqlens=None):
        """Return ``(dx, d_input_gate, d_decay_gate, d_decay_param, d_initial_state)``."""
        B, T, D, dev = self.batch, self.seq_len, self.dim, x.device
        cu, nseq = self._sequences(cu_seqlens, dev)
        if initial_state is not None:
            initial_state = initial_state.contiguous()
        if d_final_state is not None:
            d_final_state = d_final_state.contiguous()
        dx, di, dr = (_rows_like(t, self.dtype, (B, T, D)) for t in (x, input_gate, decay_gate))
        if B == 0 or T == 0 or nseq == 0:
            d_initial = (torch.zeros((nseq, D), dtype=torch.float32, device=dev)
                         if d_final_state is None else d_final_state.detach().clone())
            return dx, di, dr, torch.zeros(D, dtype=torch.float32, device=dev), d_initial
        d_param = torch.empty(D, dtype=torch.float32, device=dev)
        d_initial = torch.empty((nseq, D), dtype=torch.float32, device=dev)
        if self._ws_bytes is None:
            self._ws_bytes = _native.lib().tileops_glr_bwd_workspace_bytes(B, T, D)
        ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=dev)
        dy, x, input_gate, decay_gate = map(_channels_last, (dy, x, input_gate, decay_gate))
        decay_param, states = decay_param.contiguous(), states.contiguous()
        _native.launch(
            "tileops_glr_bwd", dev, dy.data_ptr(), x.data_ptr(), input_gate.data_ptr(),
            decay_gate.data_ptr(), decay_param.data_ptr(), states.data_ptr(), _native.data_ptr(initial_state),
            _native.data_ptr(d_final_state), _native.data_ptr(cu), nseq, dx.data_ptr(), di.data_ptr(),
            dr.data_ptr(), d_param.data_ptr(), d_initial.data_ptr(), ws.data_ptr(), B, T, D,
            dy.stride(0), dy.stride(1), x.stride(0), x.stride(1), input_gate.stride(0),
            input_gate.stride(1), decay_gate.stride(0), decay_gate.stride(1), self.decay_scale,
            self._code)
        return dx, di, dr, d_param, d_initial


class GatedLinearRecurrenceDecodeKernel(_GatedLinearRecurrenceKernel):
    """One token of every sequence.

    Args:
        batch, dim: sequences and channels.
        decay_scale, dtype, config: as in the forward kernel.
    """

    def __init__(self, batch: int, dim: int, decay_scale: float = 8.0,
                 dtype: torch.dtype = torch.bfloat16, config: Optional[dict] = None):
        super().__init__(batch, 1, dim, decay_scale, dtype, config)

    def forward(self, x, input_gate, decay_gate, decay_param, state, inplace: bool = False):
        """Return ``(y, new_state)``; ``inplace`` writes the new state over ``state``."""
        B, D, dev = self.batch, self.dim, x.device
        x, input_gate = _channels_last(x), _channels_last(input_gate)
        decay_gate, decay_param = _channels_last(decay_gate), decay_param.contiguous()
        if not inplace:
            state = state.contiguous()
        y = _rows_like(x, self.dtype, (B, D))
        new_state = state if inplace else torch.empty_like(state)
        _native.launch(
            "tileops_glr_decode_fwd", dev, x.data_ptr(), input_gate.data_ptr(),
            decay_gate.data_ptr(), decay_param.data_ptr(), state.data_ptr(),
            y.data_ptr(), new_state.data_ptr(), B, D, x.stride(0), input_gate.stride(0),
            decay_gate.stride(0), self.decay_scale, self._code)
        return y, new_state
