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
operators; the native layer raises RuntimeError.  Nothing reads tensor values on
the host: a call never synchronises, runs on the current stream and can be
captured into a HIP graph.  The reference has no counterparts; its caches are
fp16 and filled by the caller (tests/kernel_test_utils.py).
"""

from __future__ import annotations

import math

import torch

from ._native import ext
from .ops import ENGINE_MFMA, FP8_CACHE_DTYPES, MAX_GQA, SUPPORTED_HEAD_DIMS, _aligned_q, _cache_format

MX4_HEAD_DIMS = (64, 128, 256)
_ROW_DTYPES = (torch.float16, torch.bfloat16)
_CODE_DTYPES = (torch.uint8, torch.float4_e2m1fn_x2)
_SCALE_DTYPES = (torch.uint8, torch.float8_e8m0fnu)


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


def _disjoint(t):
    """No two elements in one place, as far as strides of 0 show it."""
    return all(s != 0 or n <= 1 for s, n in zip(t.stride(), t.shape))


def _is_mx4(cache):
    return cache.dtype in _CODE_DTYPES


def _check_caches(k_cache, v_cache, k_scale, v_scale):
    """(codes or rows of K, of V, MX4 scales of K, of V, fp8 scales, head_dim) of a pair of caches."""
    assert k_cache.is_cuda and v_cache.is_cuda, "the caches must be GPU tensors"
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, (
        "the caches must be [num_pages, page_size, num_kv_heads, head_dim], both alike"
    )
    assert k_cache.dtype == v_cache.dtype, "k_cache and v_cache must have the same dtype"
    assert k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "K/V caches need a contiguous head_dim"
    if not _is_mx4(k_cache):
        assert k_cache.dtype in _ROW_DTYPES + FP8_CACHE_DTYPES, (
            "caches must be float16, bfloat16, float8_e4m3fn, float8_e5m2 or MX4 codes (uint8)"
        )
        head_dim = k_cache.shape[3]
        if k_cache.dtype in FP8_CACHE_DTYPES:
            assert head_dim in MX4_HEAD_DIMS, f"fp8 caches: head_dim must be one of {MX4_HEAD_DIMS}"
            ks = 1.0 if k_scale is None else k_scale
            vs = 1.0 if v_scale is None else v_scale
            assert not isinstance(ks, torch.Tensor) and not isinstance(vs, torch.Tensor), (
                "fp8 caches take per-tensor scales, Python floats"
            )
            ks, vs = float(ks), float(vs)
            assert ks > 0 and vs > 0 and math.isfinite(ks) and math.isfinite(vs), (
                "k_scale and v_scale must be finite and positive"
            )
            return k_cache, v_cache, None, None, ks, vs, head_dim
        assert head_dim in SUPPORTED_HEAD_DIMS, f"head_dim must be one of {SUPPORTED_HEAD_DIMS}"
        assert not isinstance(k_scale, torch.Tensor) and not isinstance(v_scale, torch.Tensor) and (
            k_scale in (None, 1.0) and v_scale in (None, 1.0)
        ), "k_scale / v_scale apply to fp8 and MX4 caches only"
        return k_cache, v_cache, None, None, 1.0, 1.0, head_dim
    head_dim = 2 * k_cache.shape[3]
    assert head_dim in MX4_HEAD_DIMS, f"MX4 caches: head_dim must be one of {MX4_HEAD_DIMS}"
    for s in (k_scale, v_scale):
        assert isinstance(s, torch.Tensor) and s.dtype in _SCALE_DTYPES, "MX4 caches need uint8 scale tensors"
        assert s.is_cuda and tuple(s.shape) == (*k_cache.shape[:3], head_dim // 32), (
            "MX4 scales must be [num_pages, page_size, num_kv_heads, head_dim // 32] on the GPU"
        )
        assert s.stride(3) == 1, "MX4 scales need a contiguous last axis"
    return (k_cache.view(torch.uint8), v_cache.view(torch.uint8), k_scale.view(torch.uint8),
            v_scale.view(torch.uint8), 1.0, 1.0, head_dim)


def _check_state(t, k_cache, dtype, name):
    assert t.is_cuda and t.dtype == dtype and tuple(t.shape) == tuple(k_cache.shape[:3]), (
        f"{name} must be {dtype} [num_pages, page_size, num_kv_heads] on the GPU"
    )
    assert _disjoint(t), f"{name} must not be an expanded tensor"


def _check_index(block_table, seq_lens, batch=None):
    assert block_table.is_cuda and seq_lens.is_cuda, "block_table and seq_lens must be GPU tensors"
    assert block_table.dim() == 2 and seq_lens.dim() == 1 and seq_lens.shape[0] == block_table.shape[0], (
        "block_table must be [batch, max_pages] and seq_lens [batch]"
    )
    assert batch is None or block_table.shape[0] == batch, "block_table must be [batch, max_pages]"
    for t in (block_table, seq_lens):
        assert t.dtype in (torch.int32, torch.int64), "block_table and seq_lens must be int32 or int64"
    return block_table.to(torch.int32), seq_lens.to(torch.int32)


def _check_slots(slots, tokens):
    assert slots.is_cuda and slots.dim() == 1 and slots.dtype in (torch.int32, torch.int64), (
        "slots must be a 1-D int32 or int64 GPU tensor"
    )
    assert tokens is None or slots.shape[0] == tokens, "slots must name one slot per row"
    return slots.contiguous()


def _aligned_rows(x):
    """16-byte rows, as the kernels need; copied if they are not."""
    if x.stride(2) != 1 or x.stride(1) % 8 or x.stride(0) % 8 or x.data_ptr() % 16:
        return x.contiguous()
    return x


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
    kc, vc, ks, vs, ksc, vsc, head_dim = _check_caches(k_cache, v_cache, k_scale, v_scale)
    assert k.is_cuda and v.is_cuda, "k and v must be GPU tensors"
    assert k.dtype in _ROW_DTYPES and v.dtype == k.dtype, "k and v must both be float16 or both bfloat16"
    assert k.dim() == 3 and v.shape == k.shape and tuple(k.shape[1:]) == (k_cache.shape[2], head_dim), (
        "k and v must be [tokens, num_kv_heads, head_dim] of the caches"
    )
    assert k_cache.dtype not in _ROW_DTYPES or k_cache.dtype == k.dtype, "16-bit caches take rows of their own type"
    assert all(_disjoint(t) for t in (kc, vc, ks, vs) if t is not None), "the caches must not be expanded tensors"
    slots = _check_slots(slots, k.shape[0])
    if weights is not None:
        _check_state(weights, k_cache, torch.float32, "weights")
    if positions is not None:
        _check_state(positions, k_cache, torch.int32, "positions")
        assert token_positions is not None, "positions need token_positions"
    if token_weights is not None:
        assert weights is not None, "token_weights need weights"
        assert token_weights.is_cuda and token_weights.dtype == torch.float32 and (
            tuple(token_weights.shape) == tuple(k.shape[:2])
        ), "token_weights must be float32 [tokens, num_kv_heads] on the GPU"
        token_weights = token_weights.contiguous()
    if token_positions is not None:
        assert positions is not None, "token_positions need positions"
        assert token_positions.is_cuda and token_positions.dtype in (torch.int32, torch.int64) and (
            tuple(token_positions.shape) == tuple(k.shape[:1])
        ), "token_positions must be int32 or int64 [tokens] on the GPU"
        token_positions = token_positions.to(torch.int32).contiguous()
    ext().kv_append(_aligned_rows(k), _aligned_rows(v), kc, vc, slots, ks, vs, ksc, vsc, weights, positions,
                    token_weights, token_positions)


def paged_kv_read(k_cache, v_cache, slots, k_scale=None, v_scale=None, dtype=None):
    """``(k, v)``: the rows that ``slots`` hold, as values ``[tokens, num_kv_heads, head_dim]``.

    What an attention over a chunk of a prompt reads of the cached part.  ``dtype``
    float16 or bfloat16: the caches' own type if they are 16-bit (the default
    there), else float16 by default; values are rounded to it (every MX4 value in
    bfloat16's range is exact in bfloat16).  A negative slot, or one outside the
    cache, gives zeros.
    """
    kc, vc, ks, vs, ksc, vsc, head_dim = _check_caches(k_cache, v_cache, k_scale, v_scale)
    if dtype is None:
        dtype = k_cache.dtype if k_cache.dtype in _ROW_DTYPES else torch.float16
    assert dtype in _ROW_DTYPES, "dtype must be float16 or bfloat16"
    assert k_cache.dtype not in _ROW_DTYPES or k_cache.dtype == dtype, "16-bit caches are read in their own type"
    return ext().kv_read(kc, vc, _check_slots(slots, None), ks, vs, ksc, vsc, head_dim, dtype == torch.bfloat16)


def _decode(q, k_cache, v_cache, block_table, seq_lens, num_splits, scale, k_scale, v_scale, weights):
    assert q.is_cuda and q.dtype in _ROW_DTYPES, "q must be a float16 or bfloat16 GPU tensor"
    assert q.dim() == 3, "q must be [batch, num_q_heads, head_dim]"
    kc, vc, ks, vs, ksc, vsc, head_dim = _check_caches(k_cache, v_cache, k_scale, v_scale)
    batch, num_q_heads = q.shape[:2]
    num_kv_heads = k_cache.shape[2]
    assert q.shape[2] == head_dim, "q head_dim must match the KV cache head_dim"
    assert num_kv_heads > 0 and num_q_heads % num_kv_heads == 0, (
        "num_q_heads must be divisible by num_kv_heads (GQA)"
    )
    assert num_q_heads // num_kv_heads <= MAX_GQA, f"GQA group larger than {MAX_GQA}"
    if ks is None:
        _cache_format(q, k_cache, v_cache, head_dim, ENGINE_MFMA, k_scale, v_scale)
    block_table, seq_lens = _check_index(block_table, seq_lens, batch)
    num_splits = 0 if num_splits is None else int(num_splits)
    assert num_splits >= 0, "num_splits must be >= 1"
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(head_dim)
    return ext().cache_decode(_aligned_q(q), kc, vc, block_table, seq_lens, ks, vs, weights, scale, ksc, vsc,
                              num_splits)


def paged_attention_decode_mx4(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, num_splits=None,
                               scale=None):
    """Decode over MX4 K/V caches: the same operator with a quarter of the cache bytes.

    The caches as :func:`paged_kv_append` fills them (the module's text gives the
    layout).  q and the output are fp16 or bfloat16; the result equals the
    operator on the caches' values, which are widened exactly in registers as long
    as q's type holds them.  head_dim 64, 128 or 256, any page size, groups of up
    to 16 query heads.
    """
    assert _is_mx4(k_cache), "MX4 caches are uint8 (or float4_e2m1fn_x2) codes"
    assert num_splits is None or int(num_splits) >= 1, "num_splits must be >= 1"
    return _decode(q, k_cache, v_cache, block_table, seq_lens, num_splits, scale, k_scale, v_scale, None)


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
    assert num_splits is None or int(num_splits) >= 1, "num_splits must be >= 1"
    assert k_cache.dim() == 4, "bad cache shapes"
    _check_state(weights, k_cache, torch.float32, "weights")
    return _decode(q, k_cache, v_cache, block_table, seq_lens, num_splits, scale, k_scale, v_scale, weights)


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
    kc, vc, ks, vs, _, _, head_dim = _check_caches(k_cache, v_cache, k_scale, v_scale)
    assert all(_disjoint(t) for t in (kc, vc, ks, vs) if t is not None), "the caches must not be expanded tensors"
    _check_state(weights, k_cache, torch.float32, "weights")
    _check_state(positions, k_cache, torch.int32, "positions")
    block_table, seq_lens = _check_index(block_table, seq_lens)
    recent = int(recent)
    assert 0 <= recent < 2**31, "recent must be at least 0"
    keeps = None
    if isinstance(keep, torch.Tensor):
        assert keep.is_cuda and keep.dtype in (torch.int32, torch.int64) and keep.shape == seq_lens.shape, (
            "keep must be an int, or int32 [batch] on the GPU"
        )
        keeps, keep = keep.to(torch.int32).contiguous(), 0
    else:
        keep = int(keep)
        assert 1 <= keep < 2**31, "keep must be at least 1"
    return ext().kv_evict(kc, vc, weights, positions, block_table, seq_lens, ks, vs, keeps, keep, recent, head_dim)
