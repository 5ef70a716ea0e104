from tileops.ops.linear_attention.gla_decode import GLADecodeOp
from tileops.ops.linear_attention.gated_delta_net_prefill import (
    GatedDeltaNetPrefillFwdOp,
    chunk_gated_delta_rule,
)
from tileops.ops.linear_attention.gated_linear_recurrence import (
    GatedLinearRecurrenceBwdOp,
    GatedLinearRecurrenceDecodeOp,
    GatedLinearRecurrenceFwdOp,
)

__all__ = [
    "GLADecodeOp",
    "GatedDeltaNetPrefillFwdOp",
    "GatedLinearRecurrenceBwdOp",
    "GatedLinearRecurrenceDecodeOp",
    "GatedLinearRecurrenceFwdOp",
    "chunk_gated_delta_rule",
]
