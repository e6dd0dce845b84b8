from .attention import (
    FastBaseAttention,
    FastGroupedQueryAttention,
    FastMultiHeadAttention,
    FastMultiHeadSelfAttention,
    FastMultiQueryAttention,
    PackedSequences,
    packed_attn_func,
    shared_prefix_attn_func,
    triton_attn_func,
)
from .embeddings import FastALiBiPositionEmbedding, FastRoPEPositionEmbedding
