"""Public functional attention API (reference
``trinix/layers/attention/functional.py:8-140``), computed by the gfx950 HIP
kernels in ``libtrinix_attn.so``.
"""
from typing import Optional, Tuple

import torch

from ...kernels.attention_kernel import TritonAttentionKernel, attention
from ...kernels.packed_attention import PackedSequences, packed_attention
from ...kernels.shared_prefix import shared_prefix_attention


def triton_attn_func(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    attn_mask: Optional[torch.Tensor] = None,
    dropout_p: float = 0.0,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    window_size: Optional[Tuple[int, int]] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    *,
    rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None,
    return_lse: bool = False,
) -> torch.Tensor:
    """Scaled dot-product attention on the GPU.

    Args (same order and meaning as the reference):
        q: (batch, seq_len_q, num_heads, head_dim) GPU tensor (fp32/fp16/bf16).
        k, v: (batch, seq_len_k, num_kv_heads, head_dim); ``num_kv_heads``
            divides ``num_heads`` (equal to it in the reference).  Query head
            ``h`` reads KV head ``h // (num_heads // num_kv_heads)``.
        attn_mask: additive mask, 2-D (Sq, Sk), 3-D (B, Sq, Sk) or 4-D
            (B, 1|H, Sq, Sk); ``-inf`` removes a key.
        dropout_p: dropout probability on the attention weights.
        softmax_scale: defaults to ``head_dim ** -0.5``.
        causal: key j allowed only for j <= i (top-left aligned).
        window_size: (left, right): keys with -left <= j - i <= right.
        alibi_slopes: (H,), (1, H) or (B, H); adds ``-slope * |i - j|``.
    Keyword-only extensions:
        rotary_cos / rotary_sin: RoPE tables (rows = positions, in q.dtype,
            as ``FastRoPEPositionEmbedding.forward`` returns them); q is
            rotated inside the attention kernel, k by a pre-pass.
        return_lse: also return the fp32 (B, H, Sq) log-sum-exp.

    Returns:
        (batch, seq_len_q, num_heads, head_dim) tensor of q.dtype,
        differentiable through the HIP backward (dropout included; the
        reference's output is detached).

    Raises:
        ValueError: non-GPU tensors, inconsistent shapes, or a zero-sized
            batch, sequence or head dimension (``TRINIX_ERR_BAD_SHAPE``).
        RuntimeError: the HIP kernel library or a gfx950 GPU is unavailable.
    """
    if not q.is_cuda:
        raise ValueError("triton_attn_func only supports CUDA tensors")

    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(
            f"Expected 4D tensors (batch, seqlen, nheads, headdim), "
            f"got q: {q.shape}, k: {k.shape}, v: {v.shape}"
        )

    batch, seqlen_q, nheads, headdim = q.shape
    _, seqlen_k, nheads_k, _ = k.shape

    if nheads_k <= 0 or nheads % nheads_k != 0 or k.shape != (batch, seqlen_k, nheads_k, headdim):
        raise ValueError(f"k shape {k.shape} doesn't match expected shape")

    if v.shape != (batch, seqlen_k, nheads_k, headdim):
        raise ValueError(f"v shape {v.shape} doesn't match expected shape")

    if not TritonAttentionKernel.is_available():
        raise RuntimeError(
            "HIP attention kernel not available. "
            "Build it with `python -m trinix_amd.build` and run on an MI355X (gfx950)."
        )

    if softmax_scale is None:
        softmax_scale = headdim**-0.5

    return attention(
        q,
        k,
        v,
        attn_mask=attn_mask,
        causal=causal,
        scale=softmax_scale,
        dropout_p=dropout_p,
        window_size=window_size,
        alibi_slopes=alibi_slopes,
        rotary_cos=rotary_cos,
        rotary_sin=rotary_sin,
        return_lse=return_lse,
    )


def packed_attn_func(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    sequences: PackedSequences,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    window_size: Optional[Tuple[int, int]] = None,
    alibi_slopes: Optional[torch.Tensor] = None,
    *,
    return_lse: bool = False,
):
    """Attention over sequences of different lengths packed without padding.

    Args:
        q: (total_q, num_heads, head_dim) GPU tensor (fp32/fp16/bf16); head_dim
            up to 256.
        k, v: (total_k, num_kv_heads, head_dim); ``num_kv_heads`` divides
            ``num_heads``.
        sequences: ``PackedSequences`` with the boundaries of the rows of q, k
            and v; no row sees another sequence.
        softmax_scale: defaults to ``head_dim ** -0.5``.
        causal: with Lq queries and Lk keys in a sequence, query i sees keys
            j <= i + Lk - Lq: the queries are the sequence's last positions, so
            a chunk of a prompt attends to its cache and to itself.
        window_size: (left, right): keys with
            -left <= j - (i + Lk - Lq) <= right.
        alibi_slopes: (H,) or (1, H) constants; adds ``-slope * |i + Lk - Lq - j|``.
        return_lse: also return the fp32 (num_heads, total_q) log-sum-exp.

    Returns:
        (total_q, num_heads, head_dim) tensor of q.dtype, differentiable in q, k
        and v.  A row that sees no key (a sequence without keys, a query before
        the first key, padding behind the last sequence) gives 0 and a
        log-sum-exp of -inf, where ``triton_attn_func`` gives NaN: packed
        batches hold such rows by design. Rows that see no key, and keys that no
        row sees (before the window of a chunk's first query, say), may hold
        anything; NaN or infinity in a key or value that one row sees may reach
        the other rows of its sequence.

    A graph captured around the forward and its backward takes q, k and v that
    no living eager autograd graph holds as leaves (``detach()`` makes such), as
    any captured backward does.

    Raises:
        ValueError: non-GPU tensors, inconsistent shapes, types or devices,
            slopes that require a gradient.
        RuntimeError: the HIP kernel library or a gfx950 GPU is unavailable,
            the sequences were rebuilt between a forward and its backward, or a
            second derivative is asked for.
    """
    return packed_attention(q, k, v, sequences, softmax_scale, causal, window_size, alibi_slopes, return_lse)


def shared_prefix_attn_func(
    q: torch.Tensor,
    prefix_k: torch.Tensor,
    prefix_v: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    seq_lens: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    *,
    return_lse: bool = False,
):
    """Attention of a batch of requests that share a long prefix, whose keys and
    values are read once for all of them.

    Args:
        q: (batch, seq_len_q, num_heads, head_dim) GPU tensor (fp32/fp16/bf16);
            head_dim up to 256.  One row for a decode step, several for drafts
            or an appended turn.
        prefix_k, prefix_v: (prefix_len, num_kv_heads, head_dim), seen by every
            query; ``num_kv_heads`` divides ``num_heads``.
        k, v: (batch, capacity, num_kv_heads, head_dim): the requests' own
            caches, any strides (a (batch, num_kv_heads, capacity, head_dim)
            cache is passed as ``cache.transpose(1, 2)``).  RoPE is the caller's:
            own position j stands at prefix_len + j.
        seq_lens: (batch,) int32 or int64 GPU tensor: valid own keys, the queries'
            among them; query i sees the own keys j <= seq_lens[b] - seq_len_q + i.
            Rows of the cache behind them are not read.  Values are read on the
            GPU (a captured graph replays with new ones) and clamped into
            [0, capacity].  By default capacity.
        softmax_scale: defaults to ``head_dim ** -0.5``.
        return_lse: also return the fp32 (batch, num_heads, seq_len_q)
            log-sum-exp.

    Returns:
        (batch, seq_len_q, num_heads, head_dim) tensor of q.dtype, without a
        backward.  A row that sees no key (no prefix, nothing of its own) gives 0
        and a log-sum-exp of -inf.

    Raises:
        ValueError: non-GPU tensors, inconsistent shapes, types or devices, or
            inputs that require gradients.
        RuntimeError: the HIP kernel library or a gfx950 GPU is unavailable.
    """
    return shared_prefix_attention(q, prefix_k, prefix_v, k, v, seq_lens, softmax_scale, return_lse)
