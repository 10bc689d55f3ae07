/*
 * pa_cache.h - C ABI of the cache operators of libpa_decode.so: storing rows in
 * a paged K/V cache (16-bit, fp8, MX4), reading them back, decoding over MX4
 * caches, decoding with accumulated attention weights, and eviction.
 *
 * MX4 caches (OCP Microscaling v1.0, MXFP4).  Every 32 consecutive elements of a
 * row share a scale 2^(s - 127), one byte s (255: NaN); an element is an e2m1
 * code (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two
 * a byte, the even element in the low nibble.  Codes are uint8 [num_pages,
 * page_size, num_kv_heads, head_dim / 2], scales uint8 [num_pages, page_size,
 * num_kv_heads, head_dim / 32]; the last axis is contiguous, the other strides
 * are free (head-major pages, [num_pages, num_kv_heads, page_size, ...] in
 * memory, read best).  head_dim 64, 128 or 256.
 *
 * Weights (fp32) and positions (int32) are [num_pages, page_size, num_kv_heads]
 * with any strides: what each token has received from the queries so far, and its
 * place in the text.  A page belongs to one sequence where a call writes to it
 * (weights, eviction); two sequences that share one lose updates.
 *
 * Everything is asynchronous on `stream`, allocates nothing and can be captured.
 * Page ids outside [0, num_pages) read page 0 and are not written to; slots
 * outside the cache are skipped (append) or read as zeros (read).
 * Return codes are pa_decode.h's pad_status.  The operators have no
 * counterparts in the reference, whose callers fill fp16 caches themselves
 * (tests/kernel_test_utils.py).
 */
#ifndef PA_CACHE_H_
#define PA_CACHE_H_

#include "pa_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache formats besides pa_decode.h's: MX4 with fp16 q and out, or bfloat16. */
#define PAD_KV_MX4 6
#define PAD_KV_MX4_BF16 7

/* A decode over MX4 caches, or one that adds up attention weights, or both.
 *   call: as for pad_decode_launch_call(), with the dense page index, no work
 *     list, engine 0, and kv_format one of pa_decode.h's or the two above.  Over
 *     MX4 caches k_cache and v_cache are the codes and dims' k_stride and
 *     v_stride count bytes (rows 16-byte aligned, 8 at head_dim 64; page and slot
 *     strides below 2^32, as the scales'); k_scale and
 *     v_scale are not read.
 *   k_scales, v_scales, ks_stride, vs_stride: MX4 scale bytes; strides of page,
 *     slot and kv head.
 *   weights, w_stride: NULL, or where the softmax weights of every token, summed
 *     over the query heads of its kv head, are added (strides in elements).
 *   logits, logits_bytes: scratch of pad_cache_logits_bytes(), with weights (a
 *     table row's tokens times the group of query heads: below 2^30).
 * Scratch (workspace, counters): pad_cache_scratch(); with less than that a call
 * may run another kernel, or return PAD_ERR_WORKSPACE. */
typedef struct pad_cache_call {
  pad_decode_call call;
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  int64_t ks_stride[3];
  int64_t vs_stride[3];
  float* weights;
  int64_t w_stride[3];
  void* logits;
  size_t logits_bytes;
} pad_cache_call;

/* Workspace bytes and counters (zeroed once, left at zero) of a
 * pad_cache_decode() over caches of kv_format; num_cus <= 0 means 256.  Host
 * only. */
int pad_cache_scratch(const pad_decode_dims* dims, int kv_format,
                      int num_splits, int num_cus, size_t* bytes,
                      int64_t* count);

/* Bytes of the scores of one decode: 4 per (query head, token of a table row),
 * and 4 per (sequence, query head).  Host only. */
int pad_cache_logits_bytes(const pad_decode_dims* dims, size_t* bytes);

int pad_cache_decode(const pad_cache_call* call, const pad_decode_dims* dims,
                     void* stream);

/* One layer's caches.  kv_format: PAD_KV_FP16, PAD_KV_BF16, PAD_KV_FP8_E4M3FN,
 * PAD_KV_FP8_E5M2 or PAD_KV_MX4; strides (page, slot, kv head; 0 to 2^32 - 1) in
 * elements of the cache, which are bytes of codes for MX4.  k_scale, v_scale: fp8 caches hold
 * K / k_scale and V / v_scale.  k_scales, v_scales: MX4 only.  weights and
 * positions may be NULL in append and read, not in evict. */
typedef struct pad_kv_cache {
  void* k;
  void* v;
  uint8_t* k_scales;
  uint8_t* v_scales;
  float* weights;
  int32_t* positions;
  int64_t k_stride[3], v_stride[3];
  int64_t ks_stride[3], vs_stride[3];
  int64_t w_stride[3], p_stride[3];
  int64_t num_pages;
  int32_t page_size;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t kv_format;
  float k_scale;
  float v_scale;
} pad_kv_cache;

/* Rows [tokens, num_kv_heads, head_dim] (fewer than 2^31 rows) of an append or a read: fp16, or
 * bfloat16 (bf16 = 1), with strides of token and kv head in elements (rows
 * contiguous and 16-byte aligned).  slots: page * page_size + slot of every
 * token, int64 (slots64 = 1) or int32, contiguous. */
typedef struct pad_kv_rows {
  void* k;
  void* v;
  int64_t k_stride[2], v_stride[2];
  const void* slots;
  int64_t tokens;
  int32_t slots64;
  int32_t bf16;
} pad_kv_rows;

/* Stores rows: 16-bit caches as they are (the rows' type); fp8 caches
 * x / scale rounded to the nearest, ties to even, and held to the largest finite value (NaN
 * stays); MX4 caches by the format's rule: the scale is 2^(floor(log2 max|x|) - 2),
 * at least 2^-127, codes round to the nearest value, ties to the even code, 6 at
 * most; a block that holds a NaN or an infinity becomes NaN.
 * With cache->weights every stored token's weights become token_weights
 * [tokens, num_kv_heads] (contiguous), or 0 where that is NULL; with
 * cache->positions its positions become token_positions [tokens] (required
 * then).  Slots have to differ: a slot named twice holds parts of either row. */
int pad_kv_append(const pad_kv_cache* cache, const pad_kv_rows* rows,
                  const float* token_weights, const int32_t* token_positions,
                  void* stream);

/* The rows that the slots hold, as values (fp8 times its scale), rounded to the
 * rows' type; zeros for a slot outside the cache. */
int pad_kv_read(const pad_kv_cache* cache, const pad_kv_rows* rows,
                void* stream);

/* Cuts every sequence to `keep` tokens, per kv head: kept are the tokens whose
 * position is greater than the sequence's largest less `recent`, then those of
 * the largest weight (NaN before all others), and of equal ones the lowest slots.
 * Kept tokens in slots below the new length stay where they are; the i-th kept
 * token above it moves, with its weight and position, to the i-th slot below
 * that held an evicted one.  Slots from the new length on keep what they held.
 * A sequence of at most `keep` tokens is left as it is.
 *   keep: `keeps` (int32 [batch] on the device) or, where that is NULL, keep;
 *   new_lens: int32 [batch], the new lengths (not seq_lens itself);
 *   workspace: pad_kv_evict_workspace_bytes(). */
typedef struct pad_kv_evict_call {
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* keeps;
  int32_t* new_lens;
  void* workspace;
  size_t workspace_bytes;
  int64_t bt_stride[2];
  int64_t sl_stride;
  int32_t batch;
  int32_t max_pages;
  int32_t keep;
  int32_t recent;
} pad_kv_evict_call;

int pad_kv_evict_workspace_bytes(int64_t batch, int64_t num_kv_heads,
                                 int64_t max_pages, int64_t page_size,
                                 size_t* bytes);
int pad_kv_evict(const pad_kv_cache* cache, const pad_kv_evict_call* call,
                 void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* PA_CACHE_H_ */
