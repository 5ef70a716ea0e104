from tileops.kernels.norm.fused_add_layer_norm import FusedAddLayerNormKernel
from tileops.kernels.norm.sandwich_norm import (
    FusedSandwichNormBwdKernel,
    FusedSandwichNormFwdKernel,
)

__all__ = ["FusedAddLayerNormKernel", "FusedSandwichNormBwdKernel", "FusedSandwichNormFwdKernel"]
