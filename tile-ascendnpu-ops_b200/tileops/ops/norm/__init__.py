from tileops.ops.norm.fused_add_layer_norm import FusedAddLayerNormFwdOp
from tileops.ops.norm.sandwich_norm import FusedSandwichNormBwdOp, FusedSandwichNormFwdOp

__all__ = ["FusedAddLayerNormFwdOp", "FusedSandwichNormBwdOp", "FusedSandwichNormFwdOp"]
