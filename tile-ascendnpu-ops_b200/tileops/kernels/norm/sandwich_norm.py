"""Sandwich norm kernels: the norm after a block, its gate, the scaled residual
and the next block's norm, forward and backward.

Shims over ``tileops_sandwich_norm_fwd`` and ``tileops_sandwich_norm_bwd``
(formulas in ``csrc/sandwich_norm.cu``).
"""

from __future__ import annotations

from typing import Optional

import torch

from tileops import _native
from tileops.kernels.kernel_base import Kernel, check_dtype

__all__ = ["FusedSandwichNormBwdKernel", "FusedSandwichNormFwdKernel"]

NORMS = {"rms": 0, "layer": 1}  # TILEOPS_NORM_*


class _SandwichNormKernel(Kernel):
    SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)

    def __init__(self, M: int, N: int, norm: str, eps: float, residual_scale: float,
                 dtype: torch.dtype, config: Optional[dict] = None):
        super().__init__()
        check_dtype(self, dtype, self.SUPPORTED_DTYPES)
        if norm not in NORMS:
            raise ValueError(f"{type(self).__name__} supports norm in {tuple(NORMS)}, "
                             f"got {norm!r}")
        self.M, self.N, self.norm = M, N, norm
        self.eps, self.residual_scale = float(eps), float(residual_scale)
        self.dtype = dtype
        self._code, self._norm_code = _native.dtype_code(dtype), NORMS[norm]
        self._ws_bytes: dict = {}
        self.init_config(config)


class FusedSandwichNormFwdKernel(_SandwichNormKernel):
    """Forward kernel.

    Args:
        M, N: Rows and hidden dimension.
        norm: ``"rms"`` or ``"layer"``.
        eps: Epsilon of both norms.
        residual_scale: Factor of the residual stream.
        dtype: float32, float16 or bfloat16.
        config: Optional config dict (no tunables).
    """

    def forward(self, x, residual, post_weight, pre_weight, gate=None, post_bias=None,
                pre_bias=None):
        """``(y, residual_out)``, shaped like ``x``: contiguous, M rows of N."""
        y, residual_out = torch.empty_like(x), torch.empty_like(x)
        ptr = _native.data_ptr
        _native.launch(
            "tileops_sandwich_norm_fwd", x.device, x.data_ptr(), residual.data_ptr(),
            post_weight.data_ptr(), pre_weight.data_ptr(), ptr(gate), ptr(post_bias),
            ptr(pre_bias), y.data_ptr(), residual_out.data_ptr(), self.M, self.N,
            1 if gate is None else gate.numel() // self.N, self._norm_code, self.eps,
            self.residual_scale, self._code, _native.dtype_code(post_weight.dtype))
        return y, residual_out


class FusedSandwichNormBwdKernel(_SandwichNormKernel):
    """Backward kernel; the same arguments."""

    def forward(self, dy, d_residual_out, x, residual_out, post_weight, pre_weight, gate=None,
                post_bias=None, pre_bias=None):
        """``(dx, d_residual, d_post_weight, d_pre_weight, d_gate, d_post_bias, d_pre_bias)``,
        None in the place of a gradient of what was not given."""
        dx, d_residual = torch.empty_like(x), torch.empty_like(x)
        grads = [None if p is None else torch.empty_like(p)
                 for p in (post_weight, pre_weight, gate, post_bias, pre_bias)]
        if self.M == 0:
            return dx, d_residual, *(None if g is None else g.zero_() for g in grads)
        groups = 1 if gate is None else gate.numel() // self.N
        ptr = _native.data_ptr
        key = (groups, post_bias is not None or pre_bias is not None)
        size = self._ws_bytes.get(key)
        if size is None:
            size = self._ws_bytes[key] = _native.lib().tileops_sandwich_norm_bwd_workspace_bytes(
                self.M, self.N, *key)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        _native.launch(
            "tileops_sandwich_norm_bwd", x.device, dy.data_ptr(), ptr(d_residual_out),
            x.data_ptr(), residual_out.data_ptr(), post_weight.data_ptr(), pre_weight.data_ptr(),
            ptr(gate), ptr(post_bias), dx.data_ptr(), d_residual.data_ptr(), *map(ptr, grads),
            ws.data_ptr(), self.M, self.N, groups, self._norm_code, self.eps,
            self.residual_scale, self._code, _native.dtype_code(post_weight.dtype))
        return dx, d_residual, *grads
