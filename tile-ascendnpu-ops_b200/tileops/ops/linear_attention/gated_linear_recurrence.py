"""Gated linear recurrence ops: prefill / training forward, backward, decode.

A state per channel (GLA, GDN and SSD keep a matrix per head), for the
recurrent block behind a causal depthwise conv1d.  Per channel, with
``k = decay_scale * softplus(decay_param)``::

    a_t = exp(-k * sigmoid(decay_gate_t))
    h_t = a_t * h_{t-1} + sqrt(1 - a_t^2) * sigmoid(input_gate_t) * x_t
    y_t = h_t                                   (h in fp32, y rounded once)

A decay gate of -inf has a = 1 exactly and takes no input: a padded token (whose
x and input_gate are still read and must be finite, but have no say).  a stays
above zero however strong the decay: an infinite state stays infinite.

    GatedLinearRecurrenceFwdOp(batch, seq_len, dim, decay_scale=8.0, dtype=torch.bfloat16,
                               save_states=False, kernel_map=None)
    forward(x, input_gate, decay_gate, decay_param, initial_state=None, cu_seqlens=None)
        -> (y, final_state) or, with save_states, (y, final_state, states)

    GatedLinearRecurrenceBwdOp(batch, seq_len, dim, decay_scale=8.0, dtype=torch.bfloat16,
                               kernel_map=None)
    forward(dy, x, input_gate, decay_gate, decay_param, states, initial_state=None,
            d_final_state=None, cu_seqlens=None)
        -> (dx, d_input_gate, d_decay_gate, d_decay_param, d_initial_state)

    GatedLinearRecurrenceDecodeOp(batch, dim, decay_scale=8.0, dtype=torch.bfloat16,
                                  inplace=False, kernel_map=None)
    forward(x, input_gate, decay_gate, decay_param, state) -> (y, new_state)

x, input_gate, decay_gate, dy are (batch, seq_len, dim) -- (batch, dim) for
decode -- of ``dtype``; column slices of a wider tensor are read in place.
decay_param (dim,), the states (batch, dim) and ``states`` (batch,
ceil(seq_len / 32), dim) are float32.  Packed sequences follow the GDN op:
batch 1, ``cu_seqlens`` an integer device tensor of N + 1 offsets 0, ...,
seq_len, one initial and final state per sequence; offsets that break this
rule set the device error flag to 2 (with seq_len 0 nothing is launched and they
are not read).  A device's first packed call looks that flag up: make it outside
a graph's capture.  Like every op here, these build no
autograd graph: a training loop calls the two ops itself.
"""

from __future__ import annotations

from typing import Dict, Optional

import torch

from tileops.device import get_device_backend
from tileops.kernels.kernel_base import Kernel
from tileops.kernels.linear_attention import (
    GatedLinearRecurrenceBwdKernel,
    GatedLinearRecurrenceDecodeKernel,
    GatedLinearRecurrenceFwdKernel,
)
from tileops.ops.op_base import Op

__all__ = ["GatedLinearRecurrenceBwdOp", "GatedLinearRecurrenceDecodeOp",
           "GatedLinearRecurrenceFwdOp"]

_SEGMENT = 32


def _check(is_device_tensor, device: torch.device, name: str, t: torch.Tensor, shape: tuple,
           dtype: torch.dtype) -> None:
    if (is_device_tensor(t) and t.dtype is dtype and t.shape == shape and t.device == device):
        return
    backend = get_device_backend()
    if not backend.is_device_tensor(t):
        raise ValueError(f"{name} must be a {backend.name} tensor, "
                         f"got {getattr(t, 'device', type(t).__name__)}")
    if t.device != device:
        raise ValueError(f"Expected {name} on {device}, got {t.device}")
    if t.shape != shape:
        raise ValueError(f"Expected {name}.shape {shape}, got {tuple(t.shape)}")
    raise ValueError(f"Expected {name}.dtype {dtype}, got {t.dtype}")


def _num_seqs(batch: int, device: torch.device, cu_seqlens: Optional[torch.Tensor]) -> int:
    """Number of sequences; checks what the host can see of ``cu_seqlens``."""
    if cu_seqlens is None:
        return batch
    if not get_device_backend().is_device_tensor(cu_seqlens):
        raise ValueError(f"cu_seqlens must be a {get_device_backend().name} tensor, "
                         f"got {getattr(cu_seqlens, 'device', type(cu_seqlens).__name__)}")
    if cu_seqlens.device != device:
        raise ValueError(f"Expected cu_seqlens on {device}, got {cu_seqlens.device}")
    if batch != 1:
        raise ValueError(f"The batch size is expected to be 1 rather than {batch} when using "
                         "`cu_seqlens`. Please flatten variable-length inputs before processing.")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be a 1-D tensor of N + 1 offsets with N >= 1, got shape "
                         f"{tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
    return cu_seqlens.numel() - 1


class GatedLinearRecurrenceFwdOp(Op):
    """Gated linear recurrence over whole sequences.

    Args:
        batch, seq_len, dim: Batch size, tokens, channels.
        decay_scale: Decay rate per unit of ``softplus(decay_param)``, a positive normal float32.
        dtype: float32, float16 or bfloat16.
        save_states: Also return the states the backward op takes.
        kernel_map: Optional override of ``"glr_fwd"``.
    """

    def __init__(self, batch: int, seq_len: int, dim: int, decay_scale: float = 8.0,
                 dtype: torch.dtype = torch.bfloat16, save_states: bool = False,
                 kernel_map: Optional[Dict[str, Kernel]] = None) -> None:
        self.batch, self.seq_len, self.dim = batch, seq_len, dim
        self._nseq = batch  # sequences of the last call
        self.decay_scale = decay_scale
        self.dtype = dtype
        self.save_states = save_states
        self.dispatch_kernel(kernel_map)
        self.kernel = self.kernel_map["glr_fwd"](batch, seq_len, dim, decay_scale, dtype)

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"glr_fwd": GatedLinearRecurrenceFwdKernel}

    def forward(self, x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor,
                decay_param: torch.Tensor, initial_state: Optional[torch.Tensor] = None,
                cu_seqlens: Optional[torch.Tensor] = None):
        rows = (self.batch, self.seq_len, self.dim)
        dev, on_device = getattr(x, "device", None), get_device_backend().is_device_tensor
        _check(on_device, dev, "x", x, rows, self.dtype)
        _check(on_device, dev, "input_gate", input_gate, rows, self.dtype)
        _check(on_device, dev, "decay_gate", decay_gate, rows, self.dtype)
        _check(on_device, dev, "decay_param", decay_param, (self.dim,), torch.float32)
        nseq = self._nseq = _num_seqs(self.batch, dev, cu_seqlens)
        if initial_state is not None:
            _check(on_device, dev, "initial_state", initial_state, (nseq, self.dim), torch.float32)
        out = self.kernel(x, input_gate, decay_gate, decay_param, initial_state, cu_seqlens,
                          self.save_states)
        return out if self.save_states else out[:2]

    def eval_roofline(self) -> tuple[int, int]:
        """``(20 * B * T * D, 4 * B * T * D * elem_bytes + 2 * S * D * 4 + D * 4)``, S the sequences
        of the last call (B without packed ones).  What a forward pass cannot do without: the
        states for the backward op, 4 / 32 bytes an element, are not in it."""
        elems = self.batch * self.seq_len * self.dim
        nbytes = 4 * elems * self.dtype.itemsize + 8 * self._nseq * self.dim + 4 * self.dim
        return 20 * elems, nbytes


class GatedLinearRecurrenceBwdOp(Op):
    """Gradients of the gated linear recurrence.

    Args:
        batch, seq_len, dim, decay_scale, dtype: Those of the forward op.
        kernel_map: Optional override of ``"glr_bwd"``.
    """

    def __init__(self, batch: int, seq_len: int, dim: int, decay_scale: float = 8.0,
                 dtype: torch.dtype = torch.bfloat16,
                 kernel_map: Optional[Dict[str, Kernel]] = None) -> None:
        self.batch, self.seq_len, self.dim = batch, seq_len, dim
        self._nseq = batch  # sequences of the last call
        self.decay_scale = decay_scale
        self.dtype = dtype
        self.dispatch_kernel(kernel_map)
        self.kernel = self.kernel_map["glr_bwd"](batch, seq_len, dim, decay_scale, dtype)

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"glr_bwd": GatedLinearRecurrenceBwdKernel}

    def forward(self, dy: torch.Tensor, x: torch.Tensor, input_gate: torch.Tensor,
                decay_gate: torch.Tensor, decay_param: torch.Tensor, states: torch.Tensor,
                initial_state: Optional[torch.Tensor] = None,
                d_final_state: Optional[torch.Tensor] = None,
                cu_seqlens: Optional[torch.Tensor] = None):
        rows = (self.batch, self.seq_len, self.dim)
        dev, on_device = getattr(x, "device", None), get_device_backend().is_device_tensor
        _check(on_device, dev, "x", x, rows, self.dtype)
        _check(on_device, dev, "dy", dy, rows, self.dtype)
        _check(on_device, dev, "input_gate", input_gate, rows, self.dtype)
        _check(on_device, dev, "decay_gate", decay_gate, rows, self.dtype)
        _check(on_device, dev, "decay_param", decay_param, (self.dim,), torch.float32)
        _check(on_device, dev, "states", states, (self.batch, -(-self.seq_len // _SEGMENT), self.dim),
               torch.float32)
        nseq = self._nseq = _num_seqs(self.batch, dev, cu_seqlens)
        for name, t in (("initial_state", initial_state), ("d_final_state", d_final_state)):
            if t is not None:
                _check(on_device, dev, name, t, (nseq, self.dim), torch.float32)
        return self.kernel(dy, x, input_gate, decay_gate, decay_param, states, initial_state,
                           d_final_state, cu_seqlens)

    def eval_roofline(self) -> tuple[int, int]:
        """``(40 * B * T * D, 7 * B * T * D * elem_bytes + the fp32 states and gradients)``, of as
        many sequences as the last call had."""
        elems = self.batch * self.seq_len * self.dim
        saved = self.batch * -(-self.seq_len // _SEGMENT) * self.dim
        nbytes = (7 * elems * self.dtype.itemsize + 4 * saved + 8 * self._nseq * self.dim
                  + 8 * self.dim)
        return 40 * elems, nbytes


class GatedLinearRecurrenceDecodeOp(Op):
    """One token of the gated linear recurrence for every sequence of a batch.

    Args:
        batch, dim: Sequences, channels.
        decay_scale, dtype: Those of the forward op.
        inplace: Write the new state over ``state`` (then contiguous) and return it.
        kernel_map: Optional override of ``"glr_decode"``.
    """

    def __init__(self, batch: int, dim: int, decay_scale: float = 8.0,
                 dtype: torch.dtype = torch.bfloat16, inplace: bool = False,
                 kernel_map: Optional[Dict[str, Kernel]] = None) -> None:
        self.batch, self.dim = batch, dim
        self.decay_scale = decay_scale
        self.dtype = dtype
        self.inplace = inplace
        self.dispatch_kernel(kernel_map)
        self.kernel = self.kernel_map["glr_decode"](batch, dim, decay_scale, dtype)

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"glr_decode": GatedLinearRecurrenceDecodeKernel}

    def forward(self, x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor,
                decay_param: torch.Tensor,
                state: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        rows = (self.batch, self.dim)
        dev, on_device = getattr(x, "device", None), get_device_backend().is_device_tensor
        _check(on_device, dev, "x", x, rows, self.dtype)
        _check(on_device, dev, "input_gate", input_gate, rows, self.dtype)
        _check(on_device, dev, "decay_gate", decay_gate, rows, self.dtype)
        _check(on_device, dev, "decay_param", decay_param, (self.dim,), torch.float32)
        _check(on_device, dev, "state", state, rows, torch.float32)
        if self.inplace and not state.is_contiguous():
            raise ValueError("state must be contiguous when it is updated in place")
        return self.kernel(x, input_gate, decay_gate, decay_param, state, self.inplace)

    def eval_roofline(self) -> tuple[int, int]:
        """``(20 * B * D, 4 * B * D * elem_bytes + 2 * B * D * 4 + D * 4)``."""
        elems = self.batch * self.dim
        return 20 * elems, 4 * elems * self.dtype.itemsize + 8 * elems + 4 * self.dim
