from tileops.ops.attention.multi_head_attention import MultiHeadAttentionFwdOp
from tileops.ops.attention.paged_attention import PagedAttentionDecodeOp, PagedKVAppendOp
from tileops.ops.attention.rotary_embedding import (
    RotaryEmbeddingBwdOp,
    RotaryEmbeddingFwdOp,
    rotary_frequencies,
)

__all__ = [
    "MultiHeadAttentionFwdOp",
    "PagedAttentionDecodeOp",
    "PagedKVAppendOp",
    "RotaryEmbeddingBwdOp",
    "RotaryEmbeddingFwdOp",
    "rotary_frequencies",
]
