"""Python-level counterparts of the reference's PyO3 functions for this path
(src/python/functional.rs:187-241 `sdpa`, src/python/nn.rs:390-428 `scaled_dot_product_attention`),
on torch tensors that live on the GPU.  Both are differentiable: the forward saves O and the per-row
log-sum-exp only, the backward recomputes the probabilities tile by tile in the HIP kernels.  The autograd node and
the dispatch between the fused kernels and the materialised path (src/sdpa.rs:483-587 of the reference) are native
(csrc/torch_host.cpp).

Nothing here falls back to torch arithmetic: without the HIP library the calls raise.
"""
from __future__ import annotations

from . import capi


def sdpa(q, k, v, attn_mask=None, is_causal=None, scale=None):
    """Scaled dot-product attention on [B,H,S,D] tensors.

    attn_mask: optional binary keep-mask broadcastable as [B|1, H|1, Sq, Sk] (values >= 0.5 attend; the
    reference's public mask convention, src/sdpa.rs:458-470).  Its buffer may be refilled before the backward: the
    recorded graph holds a copy.  With is_causal=True the mask argument is ignored, as in the reference, and the
    causal structure is applied natively (no mask tensor is built).
    Inputs of another dtype are promoted to bf16 and the result is cast back."""
    return capi.host().sdpa(q, k, v, attn_mask, is_causal is not None and bool(is_causal), scale)


def scaled_dot_product_attention(q, k, v, is_causal=None):
    """nn.scaled_dot_product_attention of the reference: bf16 [B,H,S,D], scale 1/sqrt(D), optional causal."""
    if q.dim() != 4:
        raise ValueError("SDPA expects 4-D input [B, H, S, D]")
    return sdpa(q, k, v, None, is_causal)


def sdpa_with_bias(q, k, v, bias=None, scale=None):
    """attention::sdpa_with_bias: softmax(scale * Q K^T + bias) V with an additive float bias (inference only)."""
    if bias is None:
        return sdpa(q, k, v, scale=scale)
    return capi.host().sdpa_with_bias(q, k, v, bias, scale)


def sdpa_packed(q, k, v, cu_seqlens, cu_seqlens_k=None, is_causal=None, scale=None):
    """Attention of sequences of different lengths packed one behind the other: q [rows, H, D], k/v [key rows, H_kv, D],
    H a multiple of H_kv (head h reads key head h // (H // H_kv)).  Differentiable, once: a backward with create_graph=True is
    refused.

    cu_seqlens (and cu_seqlens_k where the keys have other lengths): int32 [sequences + 1] on the device, rising from 0, the rows of
    sequence i being cu_seqlens[i] .. cu_seqlens[i + 1] - 1; a recorded graph holds them, so they may not be refilled before
    its backward.  is_causal=True: query i of a sequence attends to keys j <= i + (keys - queries), the last query to
    all of them.  Queries without a key and rows behind the last sequence come out as zeros, with zero gradients.
    Inputs of another dtype are promoted to bf16 and the result is cast back.
    Its backward may be captured into a graph; a leaf that q, k or v come from and that an eager graph recorded on another
    stream still holds is refused in the capture."""
    return capi.host().sdpa_packed(q, k, v, cu_seqlens, cu_seqlens_k, is_causal is not None and bool(is_causal), scale)


def sdpa_paged(q, k_cache, v_cache, page_table, kv_len, prefix_table=None, prefix_len=None, scale=None):
    """Attention of the last N tokens of every sequence, q [B, H, N, D], against a paged cache, bf16 [pages, H_kv, page, D]
    (inference only; flame_amd.paged_cache keeps such a cache).

    page_table: int32 [B, pages], the pages of a sequence's own keys in their order; kv_len: int32 [B], how many own keys,
    the N new ones among them.  prefix_table (int32 [pages]) and prefix_len (int32 [1]): keys that all sequences have in
    front of their own, read once for the batch.  Token i attends to the prefix and to own keys j <= kv_len - N + i (an infinity or
    NaN in a later token's V reaches it all the same: its weight of 0 multiplies it).
    q of another dtype is promoted to bf16 and the result is cast back."""
    return capi.host().sdpa_paged(q, k_cache, v_cache, page_table, kv_len, prefix_table, prefix_len, scale)
