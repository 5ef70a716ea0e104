from tileops.kernels.attention.multi_head_attention import GQAPrefillFwdKernel
from tileops.kernels.attention.paged_attention import (
    PagedAttentionDecodeKernel,
    PagedKVAppendKernel,
)
from tileops.kernels.attention.rotary_embedding import (
    RotaryEmbeddingBwdKernel,
    RotaryEmbeddingFwdKernel,
)

__all__ = [
    "GQAPrefillFwdKernel",
    "PagedAttentionDecodeKernel",
    "PagedKVAppendKernel",
    "RotaryEmbeddingBwdKernel",
    "RotaryEmbeddingFwdKernel",
]
