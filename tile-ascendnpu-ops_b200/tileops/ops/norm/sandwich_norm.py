"""Sandwich norm ops: from the end of one block to the start of the next.

FusedAddLayerNormFwdOp adds a block's output to the residual stream and
normalises the sum for the next block; these ops also normalise the block's
output first, scale it by the block's gate and scale the stream::

    p = norm(x) * post_weight + post_bias         x: the block's output
    s = residual_scale * residual + gate * p      residual_out, rounded
    y = norm(s) * pre_weight + pre_bias           the next block's input

norm is RMS (``v / sqrt(mean(v^2) + eps)``) or LayerNorm, statistics in fp32;
the second one's are over the rounded s, as in FusedAddLayerNormFwdOp.

    FusedSandwichNormFwdOp(M=None, N=None, dtype=None, norm="rms", eps=1e-6,
                           residual_scale=1.0, kernel_map=None)
    forward(x, residual, post_weight, pre_weight, gate=None, post_bias=None, pre_bias=None)
        -> (y, residual_out)

    FusedSandwichNormBwdOp(the same)
    forward(dy, d_residual_out, x, residual_out, post_weight, pre_weight, gate=None,
            post_bias=None, pre_bias=None)
        -> (dx, d_residual, d_post_weight, d_pre_weight, d_gate, d_post_bias, d_pre_bias)

x, residual and the gradients of rows are (..., N) of ``dtype``.  Parameters
are (N,), all of ``dtype`` or all float32.  gate is (N,) or (G, N): the rows
are G equal consecutive groups (a batch of G samples) with a gate each; None
means 1.  A bias of None means 0.  The backward op takes the forward's x and
residual_out and the same parameters; ``d_residual_out`` may be None, and
gradients of what was None are None.  Gradients have their tensors' types,
summed in fp32 in a fixed order; the backward pass takes a workspace of two or
four fp32 rows for each gate row besides those of its CTAs.
"""

from __future__ import annotations

from typing import Dict, Optional

import torch

from tileops.device import get_device_backend
from tileops.kernels.kernel_base import Kernel
from tileops.kernels.norm import FusedSandwichNormBwdKernel, FusedSandwichNormFwdKernel

from ..op_base import Op

__all__ = ["FusedSandwichNormBwdOp", "FusedSandwichNormFwdOp"]


class _SandwichNormOp(Op):
    _op_name = ""

    def __init__(
        self,
        M: Optional[int] = None,
        N: Optional[int] = None,
        dtype: Optional[torch.dtype] = None,
        norm: str = "rms",
        eps: float = 1e-6,
        residual_scale: float = 1.0,
        kernel_map: Optional[Dict[str, Kernel]] = None,
    ):
        if norm not in ("rms", "layer"):
            raise ValueError(f"norm must be 'rms' or 'layer', got {norm!r}")
        self.M = M
        self.N = N
        self.dtype = dtype
        self._committed = (M, N, dtype)
        self.norm = norm
        self.eps = eps
        self.residual_scale = residual_scale
        self.dispatch_kernel(kernel_map)
        self._kernel_cache: Dict[tuple, Kernel] = {}
        self._last: Optional[tuple[int, int, int, int]] = None

    def _check(self, rows: tuple, params: tuple, gate: Optional[torch.Tensor]) -> Kernel:
        """Validate (name, tensor, name, tensor, ...) rows, x first, and parameters, the two
        weights first (only the biases and the gate may be None); returns the kernel of these
        sizes (the op's own attributes may be another thread's by then).

        A decode step is bound by the host: tensors are compared against x and the first
        parameter in one pass each, and told apart only when something is wrong."""
        is_device_tensor = get_device_backend().is_device_tensor
        for t in rows[1::2] + params[1:4:2]:
            if not is_device_tensor(t):
                self._refuse_device(rows + params[:4])
        for t in (params[5], params[7], gate):
            if t is not None and not is_device_tensor(t):
                self._refuse_device((*params[4:], "gate", gate), optional=True)
        x = rows[1]
        committed_m, committed_n, committed_dtype = self._committed
        dtype, shape, device = committed_dtype or x.dtype, x.shape, x.device
        N = shape[-1] if shape else 0
        if N < 1:
            raise ValueError(f"Expected x of shape (..., N) with N >= 1, got {tuple(shape)}")
        M = x.numel() // N
        affine = params[1].dtype
        if affine is not dtype and affine is not torch.float32:
            raise ValueError(f"Expected {params[0]}.dtype {dtype} or {torch.float32}, "
                             f"got {affine}")
        for i in range(1, len(rows), 2):
            t = rows[i]
            if not (t.dtype is dtype and t.shape == shape and t.device == device):
                self._refuse(rows[i - 1], t, dtype, shape, device)
        vectors, vector = 0, (N,)
        for i in range(1, len(params), 2):
            t = params[i]
            if t is not None:
                vectors += 1
                if not (t.dtype is affine and t.shape == vector and t.device == device):
                    self._refuse(params[i - 1], t, affine, vector, device)
        if gate is not None:
            if gate.dtype is not affine or gate.device != device:
                self._refuse("gate", gate, affine, gate.shape, device)
            gate_shape = gate.shape
            if (len(gate_shape) not in (1, 2) or gate_shape[-1] != N
                    or len(gate_shape) == 2 and (gate_shape[0] < 1 or M % gate_shape[0])):
                raise ValueError(f"Expected gate shape {(N,)} or (G, {N}) with G dividing the "
                                 f"{M} rows, got {tuple(gate_shape)}")
            vectors += gate.numel() // N
        if committed_n is not None and committed_n != N:
            raise ValueError(f"Expected hidden dim {committed_n}, got {N}")
        if committed_m is not None and committed_m != M:
            raise ValueError(f"Expected M={committed_m} (product of leading dims), got {M}")
        self.M, self.N, self.dtype = M, N, dtype
        self._last = (M, N, dtype.itemsize, vectors * affine.itemsize)
        key = (M, N, dtype, device.index)
        kernel = self._kernel_cache.get(key)
        if kernel is None:
            kernel = self._kernel_cache[key] = self.kernel_map[self._op_name](
                M, N, self.norm, self.eps, self.residual_scale, dtype)
        return kernel

    @staticmethod
    def _refuse_device(named: tuple, optional: bool = False) -> None:
        backend = get_device_backend()
        for name, t in zip(named[::2], named[1::2]):
            if not (optional and t is None or backend.is_device_tensor(t)):
                raise ValueError(f"{name} must be a {backend.name} tensor")

    @staticmethod
    def _refuse(name: str, t: torch.Tensor, dtype: torch.dtype, shape, device) -> None:
        if t.dtype is not dtype:
            raise ValueError(f"Expected {name}.dtype {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"Expected {name} shape {tuple(shape)}, got {tuple(t.shape)}")
        raise ValueError(f"Expected {name} on {device}, got {t.device}")

    def _work(self, flops: int, rows: int, passes: int) -> tuple[int, int]:
        if self._last is None:
            raise RuntimeError(f"{type(self).__name__}.eval_roofline() requires a prior "
                               "forward() call to bind input shape and dtype")
        M, N, eb, vectors = self._last
        return flops * M * N, rows * M * N * eb + passes * vectors * N


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


class FusedSandwichNormFwdOp(_SandwichNormOp):
    """Norm of a block's output, gate, scaled residual and the next block's norm.

    Args:
        M: Optional committed row count (product of the leading dims).
        N: Optional committed hidden dimension.
        dtype: float32, float16 or bfloat16 (inferred from ``x`` when None).
        norm: ``"rms"`` or ``"layer"``, for both norms.
        eps: Epsilon of both norms.
        residual_scale: Constant factor of the residual stream.
        kernel_map: Optional kernel override dictionary.
    """

    _op_name = "sandwich_norm_fwd"

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {self._op_name: FusedSandwichNormFwdKernel}

    def forward(self, x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                pre_weight: torch.Tensor, gate: Optional[torch.Tensor] = None,
                post_bias: Optional[torch.Tensor] = None,
                pre_bias: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Return ``(y, residual_out)``, both shaped like ``x``."""
        kernel = self._check(("x", x, "residual", residual),
                             ("post_weight", post_weight, "pre_weight", pre_weight,
                              "post_bias", post_bias, "pre_bias", pre_bias), gate)
        return kernel(
            x.contiguous(), residual.contiguous(), post_weight.contiguous(),
            pre_weight.contiguous(), _dense(gate), _dense(post_bias), _dense(pre_bias))

    def eval_roofline(self) -> tuple[int, int]:
        """``(14 * M * N, 4 * M * N * elem_bytes + the parameters once)`` of the last forward."""
        return self._work(14, 4, 1)


class FusedSandwichNormBwdOp(_SandwichNormOp):
    """Gradients of FusedSandwichNormFwdOp; the same constructor arguments."""

    _op_name = "sandwich_norm_bwd"

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {self._op_name: FusedSandwichNormBwdKernel}

    def forward(self, dy: torch.Tensor, d_residual_out: Optional[torch.Tensor], x: torch.Tensor,
                residual_out: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor,
                gate: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                pre_bias: Optional[torch.Tensor] = None):
        """Return ``(dx, d_residual, d_post_weight, d_pre_weight, d_gate, d_post_bias,
        d_pre_bias)``, None in the place of a gradient of what was None."""
        rows = ("x", x, "dy", dy, "residual_out", residual_out)
        if d_residual_out is not None:
            rows += ("d_residual_out", d_residual_out)
        kernel = self._check(rows,
                             ("post_weight", post_weight, "pre_weight", pre_weight,
                              "post_bias", post_bias, "pre_bias", pre_bias), gate)
        return kernel(
            dy.contiguous(), _dense(d_residual_out), x.contiguous(), residual_out.contiguous(),
            post_weight.contiguous(), pre_weight.contiguous(), _dense(gate), _dense(post_bias),
            _dense(pre_bias))

    def eval_roofline(self) -> tuple[int, int]:
        """``(30 * M * N, 6 * M * N * elem_bytes + the parameters and their gradients)``."""
        return self._work(30, 6, 2)
