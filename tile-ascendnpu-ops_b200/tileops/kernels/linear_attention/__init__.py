from tileops.kernels.linear_attention.gated_linear_recurrence import (
    GatedLinearRecurrenceBwdKernel,
    GatedLinearRecurrenceDecodeKernel,
    GatedLinearRecurrenceFwdKernel,
)
from tileops.kernels.linear_attention.gdn_prefill import GDNPrefillFwdKernel
from tileops.kernels.linear_attention.gla_decode import GLADecodeKernel

__all__ = [
    "GDNPrefillFwdKernel",
    "GLADecodeKernel",
    "GatedLinearRecurrenceBwdKernel",
    "GatedLinearRecurrenceDecodeKernel",
    "GatedLinearRecurrenceFwdKernel",
]
