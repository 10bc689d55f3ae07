"""Operators on the paged K/V cache itself: writing it, making it smaller, thinning it out.

* :func:`paged_kv_append` / :func:`paged_kv_read`: rows into 16-bit, fp8 and MX4
  caches, and back as values.
* :func:`paged_attention_decode_mx4`: the decode over MX4 caches (4.25 bits an
  element).
* :func:`paged_attention_decode_weights`: the decode that also adds every
  token's attention weight to its slot of a ``weights`` tensor.
* :func:`paged_kv_evict`: cuts sequences back to the newest and the heaviest
  tokens, in place.

MX4 caches (OCP Microscaling v1.0, MXFP4): ``uint8 [num_pages, page_size,
num_kv_heads, head_dim // 2]``, two e2m1 codes a byte (the even element in the
low nibble), and scales ``uint8 [num_pages, page_size, num_kv_heads, head_dim //
32]``: byte s stands for 2^(s - 127), 255 for NaN.  torch's
``float4_e2m1fn_x2`` and ``float8_e8m0fnu`` are taken as well.
:func:`mx4_cache` makes such a pair, :func:`kv_weights` the weights and
positions that eviction goes by, both with the rows of a kv head next to each
other within a page, which the kernels read best; any strides with a contiguous
last axis are taken.

Argument problems visible from metadata raise AssertionError, as in the decode
operators (the binding checks them: in Python that took longer than a small
call's kernels); others raise RuntimeError.  Nothing reads tensor values on
the host: a call never synchronises, runs on the current stream and can be
captured into a HIP graph.  The reference has no counterparts; its caches are
fp16 and filled by the caller (tests/kernel_test_utils.py).
"""

from __future__ import annotations

import torch

from ._native import ext

MX4_HEAD_DIMS = (64, 128, 256)


def mx4_cache(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device="cuda"):
    """An empty MX4 cache, ``(codes, scales)``, of zeros: one call for K and one for V."""
    assert head_dim in MX4_HEAD_DIMS, f"MX4 caches: head_dim must be one of {MX4_HEAD_DIMS}"
    made = [torch.zeros(num_pages, num_kv_heads, page_size, width, dtype=torch.uint8, device=device).transpose(1, 2)
            for width in (head_dim // 2, head_dim // 32)]
    return made[0], made[1]


def kv_weights(num_pages: int, page_size: int, num_kv_heads: int, device="cuda"):
    """``(weights, positions)`` of a cache: float32 and int32 ``[num_pages, page_size, num_kv_heads]``, of zeros."""
    shape = (num_pages, num_kv_heads, page_size)
    return (torch.zeros(shape, dtype=torch.float32, device=device).transpose(1, 2),
            torch.zeros(shape, dtype=torch.int32, device=device).transpose(1, 2))


def paged_kv_append(k, v, k_cache, v_cache, slots, k_scale=None, v_scale=None, weights=None, positions=None,
                    token_weights=None, token_positions=None):
    """Store the rows of new tokens in their slots of a paged cache.

    ``k`` / ``v`` fp16 or bfloat16 ``[tokens, num_kv_heads, head_dim]``; ``slots
    [tokens]`` (int32 or int64): page id * page_size + place in the page of each
    token; a negative slot, or one outside the cache, stores nothing (padding).
    Slots have to differ: one named twice holds parts of either row.

    The caches' type says how rows are kept: 16-bit (the rows' own type); fp8 with
    ``k_scale`` / ``v_scale`` floats (x / scale, to nearest even, held to the largest finite value);
    MX4 with ``k_scale`` / ``v_scale`` the scale tensors: per 32 elements the
    scale 2^(floor(log2 max|x|) - 2), codes to nearest even, at most 6 scales; a
    block with a NaN or an infinity becomes NaN.

    ``weights`` and ``positions`` (see :func:`kv_weights`), if given, are set for
    every stored token and kv head: to ``token_weights`` (float32 ``[tokens,
    num_kv_heads]``; 0 by default) and to ``token_positions`` (int32 ``[tokens]``,
    required with ``positions``).
    """
    ext().kv_append(k, v, k_cache, v_cache, slots, k_scale, v_scale, weights, positions, token_weights,
                    token_positions)


def paged_kv_read(k_cache, v_cache, slots, k_scale=None, v_scale=None, dtype=None):
    """``(k, v)``: the rows that ``slots`` hold, as values ``[tokens, num_kv_heads, head_dim]``.

    What an attention over a chunk of a prompt reads of the cached part.  ``dtype``
    float16 or bfloat16: the caches' own type if they are 16-bit (the default
    there), else float16 by default; values are rounded to it (every MX4 value in
    bfloat16's range is exact in bfloat16).  A negative slot, or one outside the
    cache, gives zeros.
    """
    return ext().kv_read(k_cache, v_cache, slots, k_scale, v_scale, dtype)


def paged_attention_decode_mx4(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, num_splits=None,
                               scale=None):
    """Decode over MX4 K/V caches: the same operator with a quarter of the cache bytes.

    The caches as :func:`paged_kv_append` fills them (the module's text gives the
    layout).  q and the output are fp16 or bfloat16; the result equals the
    operator on the caches' values, which are widened exactly in registers as long
    as q's type holds them.  head_dim 64, 128 or 256, any page size, groups of up
    to 16 query heads.
    """
    return ext().cache_decode(q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, None, scale, num_splits)


def paged_attention_decode_weights(q, k_cache, v_cache, weights, block_table, seq_lens, num_splits=None, scale=None,
                                   k_scale=None, v_scale=None):
    """Decode, and add every token's attention weight to its slot of ``weights``.

    ``weights`` float32 ``[num_pages, page_size, num_kv_heads]`` (see
    :func:`kv_weights`): each token of each sequence gains the softmax weights of
    the query heads that share the kv head, in 32 bits and in one order.  Other
    slots are left alone.  The caches are fp16 or bfloat16 (q's type), fp8 with
    ``k_scale`` / ``v_scale`` floats, or MX4 with the scale tensors.  Returns the
    decode's output.

    A page must belong to one sequence of the call: of two that share one, either's
    weights may be lost.
    """
    assert weights is not None, "weights must be a float32 tensor"
    return ext().cache_decode(q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, weights, scale, num_splits)


def paged_kv_evict(k_cache, v_cache, weights, positions, block_table, seq_lens, keep, recent: int = 0, k_scale=None,
                   v_scale=None):
    """Cut every sequence back to ``keep`` tokens, in place; returns the new lengths (int32 ``[batch]``).

    Per kv head, the tokens whose position is above the largest one less
    ``recent`` are kept first, then the others by weight (NaN before all), equal
    ones from the lowest slot.  Kept tokens within the new length stay in their
    slots and those beyond it move, with weight and position, into the slots of
    evicted ones, so a sequence's slots are no longer in the order of its text and
    a slot belongs to different tokens in different kv heads; the attention does
    not depend on the order, and ``positions`` keep it.  Slots from the new length
    on keep what they held: :func:`paged_kv_append` sets weight and position of
    the tokens stored there next.  Pages past the new length may be reused.

    ``keep``: an int, or int32 ``[batch]``; a sequence of at most ``keep`` tokens
    is left as it is.  Caches as for :func:`paged_attention_decode_weights` (fp8
    needs no scales here; MX4 passes the scale tensors, which move too).  A page
    must belong to one sequence of the call.
    """
    return ext().kv_evict(k_cache, v_cache, weights, positions, block_table, seq_lens, keep, recent, k_scale, v_scale)
