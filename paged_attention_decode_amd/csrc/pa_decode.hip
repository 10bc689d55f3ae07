// pa_decode.hip - gfx950 (MI355X) paged-attention decode: the per-unit kernel (its
// code is in pa_phase1.h) over 16-bit and fp8 caches, and the C ABI.
//
// Operator contract: the reference oracle paged_attention_decode_reference
// (src/reference.py:8-54) evaluated on fp16 inputs, output in fp16.
// Work decomposition: split-K over the sequence ("FlashDecoding"), the same
// merge algebra as analysis/split_k_derivation.md:16-86, restated here:
//
//   phase 1, per (sequence b, kv head, split s) over its tokens:
//     m_s = max score,  l_s = sum exp(score - m_s),
//     O_s = sum exp(score - m_s) * V                  (not divided by l_s)
//   phase 2, per (b, q head):
//     m = max_s m_s,  w_s = exp(m_s - m) (0 for an empty split),
//     out = (sum_s w_s O_s) / (sum_s w_s l_s)
//
// Scores are kept in base-2 units (score * scale * log2 e) so every
// exponential is a single v_exp_f32 (exp(x) = 2^(x log2 e)).
//
// Design (MI355X-first, not a translation of the reference's kernels):
//  * Splits are page-aligned: split s of a sequence covers logical pages
//    [s*pages_per_split, (s+1)*pages_per_split), so each page and each
//    block_table entry is read by exactly one workgroup.  The reference
//    split by tokens (cuda/kernel_v4_split_k.cu:73-75).
//  * A phase-1 workgroup is 1-8 wave64s; each wave walks 16-token blocks of
//    its split and keeps its own online-softmax state; the waves' states are
//    merged through LDS at the end (one fp32 partial per workgroup).
//  * Engine 0 (MFMA): scores are computed transposed, S^T = K . Q^T, with
//    v_mfma_f32_16x16x16_f16 (16 tokens x 16 padded GQA rows, K = head_dim),
//    and the output as O^T = V^T . P^T.  With S^T every lane already holds
//    P^T in the B-operand layout of the PV product, so P never moves between
//    lanes.  K and V are read as whole token rows (16 lanes cover a row
//    with 16-byte loads); the head_dim index inside each PV tile is
//    permuted so that these V registers are the MFMA A operand as loaded,
//    and K goes through a padded LDS tile into the A layout of S^T.  One
//    K/V tile is shared by the whole GQA group through the B operand.
//  * Engine 1 (VALU): 16 lanes per token, fp16x2 dot products
//    (v_dot2_f32_f16) reduced across the 16 lanes with 4 DPP steps, fp32
//    online softmax and FMA accumulation of P.V.  Kept for the measured
//    comparison against engine 0.
//  * Phase 2 is fused into the same launch: every workgroup of a split
//    sequence publishes its fp32 partial with device-scope stores and counts
//    itself in with an atomic; the last one to arrive folds all partials of
//    its (sequence, kv head) into the fp16 output and resets the counter
//    (past 48 splits in two levels, groups of 16 splits first).  A sequence
//    held by one split is normalised directly.  One kernel launch per call.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <mutex>

#include "pa_cache.h"
#include "pa_decode.h"
#include "pa_device.h"
#include "pa_ext.h"
#include "pa_range.h"
#include "pa_decode_timeline.h"  // slot constants; its functions exist only with -DPAD_TIMELINE

namespace pad {

#ifdef PAD_TIMELINE
// Phase timeline, compiled only into the measurement library
// (libpa_decode_tl.so, -DPAD_TIMELINE): thread 0 of every workgroup stores
// s_memrealtime stamps (100 MHz) at fixed points of its path, for the last
// PAD_TL_LAUNCHES launches (a ring indexed by a host-side launch count).
// Slot meanings are the PAD_TL_* constants of pa_decode_timeline.h.
__device__ unsigned long long tl_buf[PAD_TL_LAUNCHES * PAD_TL_MAX_GROUPS * PAD_TL_SLOTS];
static int tl_launches = 0;
static int tl_fold_polls = 0;  // pad_timeline_set_fold_polls()
#define PAD_TL_AT(lin, slot, value)                                                                      \
  do {                                                                                                   \
    if (threadIdx.x == 0 && (lin) < PAD_TL_MAX_GROUPS)                                                   \
      ::pad::tl_buf[((size_t)a.tl_launch * PAD_TL_MAX_GROUPS + (lin)) * PAD_TL_SLOTS + (slot)] = (value); \
  } while (0)
#define PAD_TL(lin, slot) PAD_TL_AT(lin, slot, __builtin_amdgcn_s_memrealtime())
#endif

}  // namespace pad

#include "pa_phase1.h"

namespace pad {

// Work-list planner: one wave per workgroup slot of the decode grid, run
// once per decode step (the sequence lengths and page ids it reads must not
// change before the launches that use the list).  Lane i < 32 writes word i
// of the record; slot 0 also writes the header.
__global__ __launch_bounds__(64) void pad_plan_kernel(const Phase1Args a, int32_t* wl) {
  int s, h, bz, lin;
  grid_pos(a, s, h, bz, lin);
  const int lane = threadIdx.x;
  const int g = s + a.num_splits * (h + a.hkv * bz);
  const int G = a.num_splits * a.hkv * a.batch;
  const int32_t* static_row = a.bt + (int64_t)bz * a.sbb;
  const SeqRaw raw = issue_seq_table(a, lane);
  const int static_len = load_uniform_i32(a.csr ? a.indptr : a.sl + (int64_t)bz * a.ssl);
  const WorkItem it = resolve_workgroup(a, raw, s, h, bz, g, G, lin, static_row, static_len, lane);
  int v = 0;
  switch (lane) {
    case 0: v = it.b; break;
    case 1: v = it.kvh; break;
    case 2: v = it.p_begin; break;
    case 3: v = it.p_end; break;
    case 4: v = it.L; break;
    case 5: v = it.nsplit; break;
    case 6: v = it.slot0; break;
    case 7: v = it.col_max; break;
    case 8: v = it.valid; break;
    case 9: v = a.csr ? (int)(it.ids_row - a.bt) : 0; break;
    default: break;
  }
  // A slot without an item gets an all-zero record (valid = 0), so lists
  // planned from the same inputs are identical word for word.
  if (!it.valid) v = 0;
  // The first page id of wave w's first block, as the decode kernel's
  // first_page_id() reads it (whole-page blocks only).
  const int w = lane - 16;
  if (w >= 0 && w < a.nw && it.valid && it.col_max >= 0 && a.ps % kBlockTokens == 0) {
    const int col = min(it.p_begin + block_page(a, w), it.col_max);
    v = it.ids_row[(int64_t)col * it.ids_stride];
  }
  int32_t* r = wl + kWlHeaderInts + (int64_t)kWlRecordInts * g;
  if (lane < kWlRecordInts) r[lane] = v;
  if (g == 0 && lane < kWlHeaderInts) wl[lane] = lane == 0 ? kWlMagic : (lane == 1 ? a.wl_key : (lane == 2 ? G : 0));
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

static bool head_dim_supported(int d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 256; }

static int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// VALU engine instantiations exist for these (head_dim, group) pairs.
static bool valu_supported(int d, int gqa) { return (d == 64 || d == 128) && gqa <= 8; }

// Dynamic LDS of a workgroup: wave (m, l) [nw][16], wave O [nw][gqa][D + 4],
// and for the MFMA engine one padded 16-row K staging tile per wave plus,
// for head_dim 256, one padded 16-row copy of Q^T.
// A range workgroup holds one Q^T copy per kv head of its group (nh).
static size_t group_lds_bytes(int nw, int gqa, int d, int engine, int nh = 1) {
  const size_t stage = engine == 0 ? (size_t)16 * (d * 2 + 16) : 0;
  const size_t q_stage = (engine == 0 && d >= 256) ? stage * nh : 0;
  return (size_t)nw * (16 * sizeof(float2) + (size_t)gqa * (d + 4) * sizeof(float) + stage) + q_stage;
}

static int lds_wave_cap(int gqa, int d, int engine) {
  const size_t per_wave = group_lds_bytes(1, gqa, d, engine) - group_lds_bytes(0, gqa, d, engine);
  int cap = (int)((kLdsBudget - group_lds_bytes(0, gqa, d, engine)) / per_wave);
  if (cap > max_group_waves(d)) cap = max_group_waves(d);
  if (cap < 1) cap = 1;
  return cap;
}

static int validate_dims(const pad_decode_dims* d) {
  if (!d) return PAD_ERR_NULL_POINTER;
  if (d->batch < 0 || d->num_q_heads <= 0 || d->num_kv_heads <= 0 || d->head_dim <= 0 ||
      d->page_size <= 0 || d->max_pages < 0 || d->num_pages < 0)
    return PAD_ERR_INVALID_SHAPE;
  if (!head_dim_supported(d->head_dim)) return PAD_ERR_UNSUPPORTED_HEAD_DIM;
  if (d->num_q_heads % d->num_kv_heads != 0) return PAD_ERR_UNSUPPORTED_GQA;
  if (d->num_q_heads / d->num_kv_heads > PAD_MAX_GQA) return PAD_ERR_UNSUPPORTED_GQA;
  if (d->q_stride[2] != 1 || d->k_stride[3] != 1 || d->v_stride[3] != 1 || d->out_stride[2] != 1)
    return PAD_ERR_STRIDE;
  return PAD_OK;
}

// Workspace layout (from the first 256-byte boundary of the buffer); the
// workspace holds no state between launches.  One slot per workgroup of the
// (S, Hkv, B) grid, G = B * Hkv * S slots:
//   o_part   fp32  [G, gqa, D] unnormalised split outputs
//   ml_part  fp32x2 [G, gqa]   (m in base-2 units, l)
// Returns the bytes needed (including 256 bytes of alignment slack) and,
// when `ws` is given, the region pointers.
static size_t workspace_layout(const pad_decode_dims* d, int S, void* ws, float** o_part, float2** ml_part) {
  const int gqa = d->num_q_heads / d->num_kv_heads;
  const size_t rows = (size_t)d->batch * d->num_kv_heads * (size_t)S * gqa;
  const size_t o_bytes = rows * (size_t)d->head_dim * sizeof(float);
  if (ws) {
    const uintptr_t base = ((uintptr_t)ws + 255u) & ~(uintptr_t)255u;
    *o_part = reinterpret_cast<float*>(base);
    *ml_part = reinterpret_cast<float2*>(base + o_bytes);
  }
  return 256 + o_bytes + rows * sizeof(float2);
}

// Splits per unit on an oversubscribed grid (see oversubscribed_shape), at
// least; and at least this many workgroups per CU.
constexpr int kOversubscribeSplits = 4;
constexpr int kOversubscribeGroupsPerCu = 8;

// A bandwidth-bound shape with a batch the in-kernel planner handles and
// either more than one (sequence, kv head) unit per two CUs, where the
// power-of-two rule gives one split per unit, or more than one per four CUs
// where its two splits per unit leave CUs idle.  The static splits are
// enough for uniform lengths (measured: C2 batch 128 81.4 us with one split
// against 93.9 us with 4 static splits), but ragged ones leave their longest
// units running alone at the end (C5: 2930 us with one workgroup per unit,
// 2656 us with kOversubscribeSplits planned items per unit, 2767 us with 8;
// C3's lengths at batch 66-127, 132-254 units: 101-113 us with one
// workgroup per unit, 58-100 us planned over oversubscribe_splits items per
// unit; at batch 33-48, 66-96 units: 51-53 us with two splits per unit,
// 34-46 us planned).  The launch therefore sizes the grid for several items
// per unit and the kernel decides from the lengths: all at full capacity,
// the static splits on the first workgroups; otherwise equal page chunks.
// fp8 caches (kv_bytes 1) keep the regime from one unit per CU up: their
// items carry half the bytes, and the grids below that (and the 8-per-CU
// floor of oversubscribe_splits) measured slower for them than the static
// splits (12/2 heads, lengths up to 4096, batch 40 / 96: 25.7 / 41.1 us
// against 18.8 / 31.4 us).
static bool oversubscribed_shape(const pad_decode_dims* d, int num_splits, int num_cus, bool latency_bound,
                                 int kv_bytes = 2) {
  const int64_t units = (int64_t)(d->batch > 0 ? d->batch : 1) * d->num_kv_heads;
  const bool many = kv_bytes == 1 ? units >= num_cus
                                  : units * 2 > num_cus || (units * 4 > num_cus && units * 2 < num_cus);
  return num_splits == 0 && !latency_bound && many && d->batch <= kPlanMaxBatch && d->max_pages < (1 << 23);
}

// Items per unit of an oversubscribed grid: kOversubscribeSplits, or more
// below two units per CU, so that the grid holds kOversubscribeGroupsPerCu
// workgroups per CU and a ragged batch's long units end in several smaller
// items (up to 16 items just above one unit per two CUs).  Measured on C5's
// lengths (batch 256, page 16, 512-32768 tokens) with 4 / 8 / 16 items per
// unit: 256 units (one GPU's share of C5 over 8 GPUs by kv heads, 8/1
// heads) 426 / 391 / 403 us; 512 units 759 / 750 / 803 us; 1024 units
// 1463 / 1509 / 1606 us; the whole C5, 2048 units, 2833 / 2916 / 3164 us.
// On C3's lengths (1-8192 tokens, page 32) this rule and a flat 4 items
// tie: 132 / 160 / 192 / 254 units 59.6 / 70.4 / 79.3 / 99.7 us against
// 58.1 / 72.0 / 76.3 / 104.9 us.
static int64_t oversubscribe_splits(int64_t units, int num_cus) {
  const int64_t want = ((int64_t)kOversubscribeGroupsPerCu * num_cus + units - 1) / units;
  return want > kOversubscribeSplits ? want : kOversubscribeSplits;
}

// Pages of one sequence the plan assumes: the dense table's row width, or
// for a CSR index (max_pages = entries of `indices`, the whole batch's
// pages) the mean per sequence, which is exact for equal lengths; ragged
// CSR batches are re-planned in-kernel from indptr anyway.
static int plan_pages_per_seq(const pad_decode_dims* d, bool csr) {
  if (d->max_pages <= 0) return 1;
  if (!csr || d->batch <= 1) return d->max_pages;
  return ceil_div(d->max_pages, d->batch);
}

static bool latency_bound_shape(const pad_decode_dims* d, int num_cus, bool csr) {
  const int max_pages = plan_pages_per_seq(d, csr);
  const int64_t units = (int64_t)(d->batch > 0 ? d->batch : 1) * d->num_kv_heads;
  const int64_t blocks_per_seq = ((int64_t)max_pages * d->page_size + kBlockTokens - 1) / kBlockTokens;
  return units * blocks_per_seq <= 16 * (int64_t)num_cus;
}

// A range launch (pa_range.hip) of a shape, or groups == 0 if the shape does
// not take one.
struct RangeShape {
  int groups;    // workgroups of the grid
  int nh_shift;  // log2 of the kv heads per workgroup
  int nw;        // waves per workgroup
  int unit_extra;  // positions a unit counts beyond its pages
  int min_chunk;   // pages per range, at least
  size_t workspace_bytes;
  int64_t counters;
};

// Partials of a range launch: two slots per workgroup, each of the rows of a
// head group (pa_range.hip's entry_slot).
static size_t range_layout(const pad_decode_dims* d, const RangeShape& r, void* ws, float** o_part, float2** ml_part) {
  const size_t rows = (size_t)2 * r.groups * (d->num_q_heads / d->num_kv_heads << r.nh_shift);
  const size_t o_bytes = rows * (size_t)d->head_dim * sizeof(float);
  if (ws) {
    const uintptr_t base = ((uintptr_t)ws + 255u) & ~(uintptr_t)255u;
    *o_part = reinterpret_cast<float*>(base);
    *ml_part = reinterpret_cast<float2*>(base + o_bytes);
  }
  return 256 + o_bytes + rows * sizeof(float2);
}

// kv_bytes: bytes per K/V element (2 for fp16, 1 for fp8 caches).
// pps_full, if given, receives the pages per split of the static splits
// (the power-of-two rule), which an oversubscribed grid runs when every
// sequence is at full capacity.
static int plan_units(const pad_decode_dims* d, int num_splits, int num_cus, int engine, bool csr,
                      pad_decode_plan_t* p, int kv_bytes = 2, int* pps_full = nullptr) {
  const int st = validate_dims(d);
  if (st != PAD_OK) return st;
  if (num_splits < 0 || num_splits > PAD_MAX_SPLITS) return PAD_ERR_NUM_SPLITS;
  if (num_cus <= 0) num_cus = 256;
  const int gqa = d->num_q_heads / d->num_kv_heads;
  const int max_pages = plan_pages_per_seq(d, csr);
  const int64_t units = (int64_t)(d->batch > 0 ? d->batch : 1) * d->num_kv_heads;

  // Regimes (fitted to measured split sweeps of C2 batch 1-64, C3 and C4 on
  // MI355X).  Bandwidth-bound shapes run one 4-wave workgroup per CU: that
  // streamed faster than two (batch 64: 44.0 vs 46.8 us; C4: 86 vs 94 us),
  // and fewer, longer splits shorten the merge.  Latency-bound shapes (at
  // most 16 blocks of work per CU) run 8-wave workgroups on at most half the
  // CUs: fewer splits to merge, each streamed by more waves (batch 8: 11.9
  // vs 13.2 us).
  const int64_t blocks_per_seq = ((int64_t)max_pages * d->page_size + kBlockTokens - 1) / kBlockTokens;
  const bool latency_bound = latency_bound_shape(d, num_cus, csr);
  int S;
  int pps;
  if (num_splits > 0) {
    // Caller's split count, page-aligned: pages_per_split = ceil(max_pages/S).
    // Splits past a sequence's last page are empty (never read).
    S = num_splits;
    pps = ceil_div(max_pages, S);
    if (pps_full) *pps_full = pps;
  } else {
    // A power-of-two split count (the splits of a power-of-two page count
    // are then equal) with at least kMinBlocks 16-token blocks per split, so
    // each workgroup's fixed costs (q load, wave merge, partial publish)
    // stay small against its streaming.  Where the largest count that fits
    // the workgroup budget is at least 1.5 times that, it is taken instead:
    // the power of two would leave a third of the budget idle (C2, uniform:
    // batch 40, 80 units, 35.1 us with 2 splits against 31.2 us with 3;
    // batch 20 20.8 against 19.2 us with 6; batch 5 12.3 against 11.7 us with
    // 12), while smaller steps lose to the longer merge (batch 7, 8 -> 9
    // splits, and batch 12, 8 -> 10: +2%).
    // A unit that shares its fold (kSharedFoldElements) at one workgroup per
    // CU pays no longer merge for more splits and takes all CUs (8 x 8192,
    // 16/1 heads of 256: 21.0 us against 23.4 us on half).
    const int64_t s_all = num_cus / units;
    const bool shared_fold = engine == 0 && s_all <= kTwoLevelSplits &&
                             s_all * gqa * (d->head_dim / 4) >= kSharedFoldElements;
    const int64_t max_groups = latency_bound && !shared_fold ? num_cus / 2 : num_cus;
    int64_t s_want = 1;
    while (s_want * 2 * units <= max_groups) s_want *= 2;
    const int64_t s_fit = max_groups / units;
    if (2 * s_fit >= 3 * s_want) s_want = s_fit;
    int64_t s_static = s_want;
    if (oversubscribed_shape(d, num_splits, num_cus, latency_bound, kv_bytes)) {
      s_want = kv_bytes == 1 ? kOversubscribeSplits : oversubscribe_splits(units, num_cus);
      // Rows of at most 128 bytes run 8-wave workgroups (below): half as
      // many items, so that each wave streams as many blocks as in a 4-wave
      // workgroup (fp16 head_dim 64, 32/8 heads, lengths up to 4096, batch
      // 20: 30.1 us with the full item count, 25.9 us with half).
      if (d->head_dim * kv_bytes <= 128 && units <= num_cus && kv_bytes == 2) s_want /= 2;
    }
    int64_t s_cap = blocks_per_seq / kMinBlocks;
    // Latency-bound short sequences: a wave's serial chain of blocks costs
    // more than a merge of up to 16 splits (one round trip), so splits may
    // go down to 4 blocks (C1, 1024 tokens: 9.2 us at 16 splits against
    // 10.3 us at the 4 that 16-block splits allow).
    if (latency_bound) {
      const int64_t short_cap = blocks_per_seq / kMinBlocksShort < 16 ? blocks_per_seq / kMinBlocksShort : 16;
      if (s_cap < short_cap) s_cap = short_cap;
    }
    if (s_cap < 1) s_cap = 1;
    if (s_want > s_cap) s_want = s_cap;
    if (s_want > PAD_MAX_SPLITS) s_want = PAD_MAX_SPLITS;
    if (s_static > s_want) s_static = s_want;
    if (pps_full) *pps_full = ceil_div(max_pages, s_static);
    if (csr) {
      // Never more splits (hence scratch) than the dense plan of the same
      // dims, so pad_decode_workspace_bytes() also sizes a CSR launch.
      pad_decode_plan_t dense;
      plan_units(d, 0, num_cus, engine, false, &dense);
      if (s_want > dense.num_splits) s_want = dense.num_splits;
    }
    pps = ceil_div(max_pages, s_want);
    S = ceil_div(max_pages, pps);
  }
  // Waves per workgroup: never more than the split has blocks or the wave
  // workgroup LDS budget allows.
  const int64_t split_tokens = (int64_t)pps * d->page_size;
  int nw = (int)((split_tokens + kBlockTokens - 1) / kBlockTokens);
  // Bandwidth-bound shapes run 4 waves per workgroup, except rows of at
  // most 128 bytes (fp16 head_dim <= 64, fp8 head_dim <= 128) with at most
  // one (sequence, kv head) unit per CU: their 16-token tiles are half the
  // bytes or less, and 8 waves keep as many bytes in flight per CU (32/8 d64
  // batch 32: 25.8 against 29.9 us; 16/4 d32: 17.8 against 21.9 us).  With
  // more units than CUs, 4-wave workgroups let several units share a CU
  // (16/16 d64 batch 32: 46.9 against 47.9 us).  The split count depends on
  // kv_bytes only through the oversubscribed regime, which gives fp8 caches
  // fewer items than fp16 ones, never more, so the fp16 plan's scratch
  // sizes always cover the fp8 plan's.
  const bool narrow_rows = d->head_dim * kv_bytes <= 128 && units <= num_cus;
  const int nw_max = (latency_bound || narrow_rows) ? kMaxWaves : kMaxWaves / 2;
  if (nw > nw_max) nw = nw_max;
  const int cap = lds_wave_cap(gqa, d->head_dim, engine);
  if (nw > cap) nw = cap;
  if (nw < 1) nw = 1;

  p->num_splits = S;
  p->pages_per_split = pps;
  p->waves_per_group = nw;
  p->single_pass = (S == 1) ? 1 : 0;
  p->engine = engine;
  p->reserved = 0;
  p->counters = 0;
  p->workspace_bytes = p->single_pass ? 0 : workspace_layout(d, S, nullptr, nullptr, nullptr);
  // One arrival counter per unit and, where a unit may get more than
  // kTwoLevelSplits items, one per item slot for the merge's groups.
  const int64_t units64 = (int64_t)d->batch * d->num_kv_heads;
  p->counters = p->single_pass ? 0 : units64 + (units64 * S > kTwoLevelSplits ? units64 * S : 0);
  return PAD_OK;
}

// Fewest K/V bytes per range: what a workgroup streams against its fixed costs
// (q and the first K/V loads, merge, partial).
constexpr int64_t kRangeMinBytes = 192 * 1024;
// What a workgroup streams in the time it takes from one unit of its range to
// the next: its waves' states merged and written, the next unit's first
// loads.  64 x [1, 8192] tokens of 32/8 heads (fp8) with 0 / 40 / 80 / 160 /
// 240 KB: 103.7 / 99.4 / 97.9 / 96.8 / 97.1 us; 24 x [1, 4096] at head_dim 64:
// 30.8 / 26.1 / 24.8 / 22.5 / 23.1 us; 48 x [1, 4096] at page size 1, four
// layers: 343 / 323 / 314 / 302 / 298 us.
constexpr int64_t kRangeUnitBytes = 160 * 1024;
// Fewest K/V bytes of a full table row in one head group, as 16-bit caches
// hold them (fp8 rows turn at the same token counts: 200 x [1, n] of 32/8
// heads, n = 384 / 512 / 640, 0.83 / 1.26 / 1.32 times the per-unit kernel's
// speed with fp8 and 0.95 / 1.14 / 1.12 with 16-bit caches).  A workgroup takes
// short units one after the other, several microseconds each, where the
// per-unit grid runs two or three side by side on a CU.  Speed against it at
// rows of 0.5 / 0.75 / 1 / 1.5 / 2 MB: 200 x [1, n] of 32/8 0.85 / 0.95 / 1.14
// / 1.16 / 1.15, 128 of 64/8 - / 0.78 / 1.04 / 1.05 / 1.09, 400 of 16/1 at
// head_dim 256 0.78 / 0.90 / 0.95 / 1.08 / 1.06 (128 of it 0.88-1.03 up to 3).
// The table's width is what the host knows of a dense call.  Short sequences
// in a wide table gain where they are many (200 x [1, 300] of 32/8 1.3, the
// per-unit grid being oversubscribed in vain) and lose where they are few or
// have one kv head (20 of 32/8 0.8, with fp8 caches 0.6; 100-256 of 8/1 0.8),
// most above the per-unit planner's batch (300 x [1, 300] of 8/1 10.7 us per
// unit, 19.6 here; filled to 4096 tokens 76 and 59).
constexpr int64_t kRangeRowBytes = 3 << 19;
// Fewest 16-bit K/V bytes of all rows: below, the per-unit grid's shorter way
// to the first load and its smaller merges count for more.  Speed against it
// at 70 / 100 / 134 / 170 / 210 / 270 MB, means of ragged and full tables of 9
// to 300 sequences: 32/8 heads 0.86 / 0.88 / 0.94 / 0.98 / 1.02 / 1.05, 24/6
// 0.89 / 0.93 / 0.97 / 1.01 / 1.05 / 1.07, 32/8 at head_dim 64 1.04 / 1.10 /
// 1.16 / 1.17 / 1.19 / 1.21, 64/8 0.75 / 0.79 / 0.84 / 0.89 / 0.94 / 0.98 (few
// units among them, which range_shape leaves out; 17 sequences 0.83 / 0.86 /
// 0.91 / 1.03 / 1.05 / 1.08).
constexpr int64_t kRangeCallBytes = 1 << 27;

// Takes the calls that the per-unit kernel plans on an oversubscribed grid
// (more units than a few per CU's worth of splits would balance, see
// oversubscribed_shape), and batches past its planner, in one workgroup per
// CU.  Against it (us, one box): 256 x [512, 32768] of 64/8 heads 2830 ->
// 2710; 64 x [1, 8192] of 32/8 with fp8 caches 114 -> 97; 24 x [1, 4096] at
// head_dim 64 28.1 -> 22.5; 17 x 4096 of 32/8 67.3 -> 51.7; 300 x [1, 4096] of
// 8/1 76.1 -> 59.0; 100 x [1, 8192] of 16/1 at head_dim 256 150 -> 89.  Two
// kv heads stay per unit: their token rows are 512 bytes, which two
// workgroups read no worse than one (the probe: 6.5 TB/s either way), and
// calls with few units keep the per-unit kernel's shorter merge (32/8 heads,
// 4 x 8192: 26.3 against 28.6-32 us).
static RangeShape range_shape(const pad_decode_dims* d, int num_splits, int num_cus, int engine, bool csr,
                              int kv_bytes, bool mx4 = false) {
  RangeShape r = {0, 0, 0, 0, 0, 0, 0};
#ifdef PAD_TIMELINE
  return r;  // the phase stamps are the per-unit kernel's
#endif
  if (num_cus <= 0) num_cus = 256;
  const int64_t units = (int64_t)d->batch * d->num_kv_heads;
  if (num_splits != 0 || engine != 0 || d->batch <= 0 || d->batch > kRangeMaxBatch) return r;
  if (d->num_kv_heads == 2 && !mx4) return r;
  r.nh_shift = d->num_kv_heads % 4 == 0 ? 2 : (d->num_kv_heads % 2 == 0 ? 1 : 0);
  // Rows of at most 128 bytes: 8 waves keep as many bytes in flight as 4 of
  // wider rows (fp8, 64 x [1, 8192]: 93.3 us with 8, 93.8 with 4; head_dim 64,
  // 24 x [1, 4096]: 22.5 and 23.1 us).
  r.nw = d->head_dim * kv_bytes <= 128 ? kMaxWaves : kMaxWaves / 2;
  // Units: above a quarter of one per CU, as the oversubscribed grid, and not
  // at one per two CUs, whose splits the per-unit grid deals evenly.  Groups of
  // four heads need more, as a workgroup's waves then stream a head each (one
  // wave, or two of fp8 rows) and a call of few units waits for that: speed
  // against the per-unit kernel at 72 / 96 / 136 units, 9 / 12 / 17 x [1, n]
  // of 64/8 heads: n = 3632 0.68 / 0.76 (3456) / 0.95 (3872), full tables of
  // 4096 0.82 / 0.89 / 1.22; 17 and 24 x [1, 1920] of 16/4 at 256 0.82, 0.88;
  // fp8, 9 and 12 x [1, 4096] of 32/8 0.91, 1.28, full 0.93, 1.03.  One and two
  // heads per workgroup gain from 70 units on (70 x [1, 4736] of 8/1 1.11, 12 x
  // [1, 4608] of 24/6 1.05), and so does head_dim 64 (9 x [1, 7264] 1.32).
  if (units * 4 <= num_cus || units * 2 == num_cus || latency_bound_shape(d, num_cus, csr)) return r;
  if (r.nh_shift == 2 && (r.nw == kMaxWaves / 2 ? units * 2 < num_cus : kv_bytes == 1 && units * 3 <= num_cus)) return r;
  // MX4 rows are short: a per-unit workgroup's share of them does not pay for its
  // fixed costs, so two kv heads take ranges as well, and groups of four from
  // rows of 512 tokens (of 128) on.  us, per unit / ranges: 48 x [1, 4096] of 12/2
  // 17.5 / 15.9, 66 23.2 / 18.1, 200 48.2 / 31.4 (33 13.4 / 15.8); 200 x [1, 512]
  // of 32/8 45.2 / 26.5, full 35.7 / 31.5, 120 27.6 / 20.0 (120 x [1, 416] 16.9 /
  // 19.2).
  if (mx4 && units * 3 <= num_cus) return r;
  const int64_t least_row = mx4 && r.nh_shift == 2 ? kRangeRowBytes * 2 / 3 : kRangeRowBytes;
  const int64_t page_bytes = ((int64_t)d->page_size * d->head_dim * (mx4 ? 1 : kv_bytes * 2)) << r.nh_shift;
  const int64_t row_bytes = plan_pages_per_seq(d, csr) * (((int64_t)d->page_size * d->head_dim * 4) << r.nh_shift);
  if (row_bytes < least_row || (units >> r.nh_shift) * row_bytes < kRangeCallBytes) return r;
  // Positions are counted in 32 bits (twice the pages at most, and unit_extra).
  if (d->batch * (2 * (int64_t)d->max_pages + 4096) > (1 << 30) / d->num_kv_heads) return r;
  // A work list holds a record per workgroup and two sequences per record.
  pad_decode_plan_t p;
  plan_units(d, 0, num_cus, 0, csr, &p);
  const int64_t records = units * p.num_splits;
  const int groups = (int)(records < num_cus ? records : num_cus);
  if (d->batch > 2 * groups) return r;
  r.groups = groups;
  r.unit_extra = ceil_div(kRangeUnitBytes, page_bytes);
  r.min_chunk = ceil_div(kRangeMinBytes, page_bytes);
  r.workspace_bytes = range_layout(d, r, nullptr, nullptr, nullptr);
  r.counters = (units >> r.nh_shift) + 2 * (int64_t)groups;
  return r;
}

// What pad_decode_plan() reports: the per-unit plan, with scratch for the range
// launch too if the shape takes one (a launch with less runs the per-unit
// kernel).  It sizes the scratch of 16-bit and fp8 launches: an fp8 launch may
// take the range kernel where a 16-bit one does not.
static int plan_impl(const pad_decode_dims* d, int num_splits, int num_cus, int engine, bool csr,
                     pad_decode_plan_t* p) {
  const int st = plan_units(d, num_splits, num_cus, engine, csr, p);
  if (st != PAD_OK) return st;
  const bool fp8_dim = d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256;
  for (int kv_bytes = 2; kv_bytes >= (fp8_dim ? 1 : 2); --kv_bytes) {
    const RangeShape r = range_shape(d, num_splits, num_cus, engine, csr, kv_bytes);
    if (r.groups == 0) continue;
    p->single_pass = 0;
    if (p->workspace_bytes < r.workspace_bytes) p->workspace_bytes = r.workspace_bytes;
    if (p->counters < r.counters) p->counters = r.counters;
  }
  return PAD_OK;
}

static int g_num_cus[64];

static int device_cus(int* out) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return PAD_ERR_DEVICE;
  if (dev < 0 || dev >= 64) return PAD_ERR_DEVICE;
  if (g_num_cus[dev] <= 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      return PAD_ERR_DEVICE;
    g_num_cus[dev] = n;
  }
  *out = g_num_cus[dev];
  return PAD_OK;
}

// fp8 caches (head_dim 64, 128 or 256) and bfloat16 (every head_dim), MFMA
// engine.
template <int KVF>
static hipError_t dispatch_kvf_dim(const Phase1Args& a, int head_dim, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if constexpr (KVF == kKvBF16) {
    if (head_dim == 32) return dispatch_kvf<32, KVF>(a, grid, nw, lds, st);
    if (head_dim == 96) return dispatch_kvf<96, KVF>(a, grid, nw, lds, st);
  }
  switch (head_dim) {
    case 64: return dispatch_kvf<64, KVF>(a, grid, nw, lds, st);
    case 128: return dispatch_kvf<128, KVF>(a, grid, nw, lds, st);
    case 256: return dispatch_kvf<256, KVF>(a, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

template <int D, int MODE>
static hipError_t dispatch_engine(const Phase1Args& a, dim3 grid, int nw, size_t lds, int engine,
                                  hipStream_t st) {
  if (engine == 1) {
    if constexpr ((D == 64 || D == 128) && MODE <= kModeUniform) {
      if (a.gqa == 1) return launch_p1<D, MODE, 1, 1>(a, grid, nw, lds, st);
      if (a.gqa == 2) return launch_p1<D, MODE, 1, 2>(a, grid, nw, lds, st);
      if (a.gqa <= 4) return launch_p1<D, MODE, 1, 4>(a, grid, nw, lds, st);
      if (a.gqa <= 6) return launch_p1<D, MODE, 1, 6>(a, grid, nw, lds, st);
      return launch_p1<D, MODE, 1, 8>(a, grid, nw, lds, st);
    }
    return hipErrorInvalidValue;
  }
  return launch_p1<D, MODE, 0, 0>(a, grid, nw, lds, st);
}

// Block-addressing mode from the page size (the VALU engine has the uniform
// and generic modes only).
template <int D>
static hipError_t dispatch_phase1(const Phase1Args& a, dim3 grid, int nw, size_t lds, int engine,
                                  hipStream_t st) {
  if (a.ps % kBlockTokens == 0) return dispatch_engine<D, kModeUniform>(a, grid, nw, lds, engine, st);
  if (engine == 0) {
    switch (a.ps) {
      case 1: return dispatch_engine<D, kModeSubpage + 0>(a, grid, nw, lds, engine, st);
      case 2: return dispatch_engine<D, kModeSubpage + 1>(a, grid, nw, lds, engine, st);
      case 4: return dispatch_engine<D, kModeSubpage + 2>(a, grid, nw, lds, engine, st);
      case 8: return dispatch_engine<D, kModeSubpage + 3>(a, grid, nw, lds, engine, st);
      default: break;
    }
  }
  return dispatch_engine<D, kModeGeneric>(a, grid, nw, lds, engine, st);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Everything one decode launch needs: kernel arguments, plan, grid, LDS.
struct Launch {
  RangeArgs a;
  bool range;  // pa_range.hip's kernel, else pad_phase1_kernel
  pad_decode_plan_t plan;
  dim3 grid;
  int nw;
  size_t lds;
  bool empty;  // batch 0: nothing to launch
};

// Key of a launch's plan, stored in a work list's header: the fields that
// decide the grid and which item each workgroup gets (FNV-1a).
static int plan_key(const RangeArgs& a) {
  const int f[] = {a.batch, a.hkv, a.max_pages, a.num_splits, a.nw, a.csr, a.balance,
                   a.ps, a.pps, a.gqa, a.pair_heads, a.min_chunk, a.groups, a.nh_shift};
  uint32_t h = 2166136261u;
  for (int x : f) {
    h ^= (uint32_t)x;
    h *= 16777619u;
  }
  return (int)(h & 0x7fffffff);
}

// Bytes of a work list: header plus one record per workgroup (of either
// kernel's grid), and of the per-unit grid of this plan.
static_assert(kRlHeaderInts == kWlHeaderInts && kRlRecordInts == kWlRecordInts, "one size for both kernels' lists");
static size_t worklist_bytes_of(int64_t groups) {
  return sizeof(int32_t) * (size_t)(kWlHeaderInts + kWlRecordInts * groups);
}
static size_t worklist_bytes_for(const pad_decode_plan_t& plan, const pad_decode_dims* d) {
  return worklist_bytes_of((int64_t)plan.num_splits * d->num_kv_heads * d->batch);
}

// Dense page table: bt = block_table, sl = seq_lens, indptr = lpl = NULL.
// CSR: bt = indices, indptr / lpl given, sl unused (dims->max_pages is the
// number of entries in indices).  io: also check q/k/v/out and the scratch
// (a work-list plan reads only the index arrays).  list_bytes: size of the
// work list the launch reads or the plan writes, if there is one.  mx4: MX4
// caches (kv_bytes 1).
static int setup_launch(const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* sl,
                        const int32_t* indptr, const int32_t* lpl, void* out, void* ws, size_t ws_bytes,
                        int32_t* counters, int64_t num_counters, const pad_decode_dims* d, float scale,
                        int num_splits, int engine, bool io, Launch* L, int kv_bytes = 2,
                        size_t list_bytes = SIZE_MAX, bool mx4 = false) {
  if (engine != 0 && engine != 1) return PAD_ERR_INVALID_SHAPE;
  // Page ids are bounds-checked against num_pages on the device (an id
  // outside [0, num_pages) reads page 0), so a launch that reads pages needs
  // the real cache size.
  if (d && d->batch > 0 && d->max_pages > 0 && d->num_pages <= 0) return PAD_ERR_INVALID_SHAPE;
  int cus = 0;
  int st = device_cus(&cus);
  if (st != PAD_OK) return st;
  const bool csr = indptr != nullptr || lpl != nullptr;
  pad_decode_plan_t& plan = L->plan;
  int pps_full = 0;
  st = plan_units(d, num_splits, cus, engine, csr, &plan, kv_bytes, &pps_full);
  if (st != PAD_OK) return st;
  const RangeShape rs = range_shape(d, num_splits, cus, engine, csr, kv_bytes, mx4);
  // The range kernel runs where its scratch and its list fit (an fp8 launch's
  // own grid may have fewer workgroups than the range launch, and a list of
  // that size stays good for it).
  L->range = rs.groups > 0 && list_bytes >= worklist_bytes_of(rs.groups) &&
             (!io || (ws && ws_bytes >= rs.workspace_bytes && counters && num_counters >= rs.counters));
  const int gqa = d->num_q_heads / d->num_kv_heads;
  if (engine == 1 && !valu_supported(d->head_dim, gqa)) return PAD_ERR_UNSUPPORTED_GQA;
  L->empty = d->batch == 0;
  if (L->empty) return PAD_OK;
  // The page-id array may be NULL only when it has no entries (a [batch, 0]
  // table, or an empty CSR index): then no sequence has a page to read.
  if ((!bt && d->max_pages > 0) || (csr ? (!indptr || !lpl) : !sl)) return PAD_ERR_NULL_POINTER;
  if (io) {
    if (!q || !k || !v || !out) return PAD_ERR_NULL_POINTER;
    // 16-byte rows: every K/V/q/out row start must be 16-byte aligned.
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return PAD_ERR_ALIGNMENT;
    if ((d->q_stride[0] | d->q_stride[1]) % 8 || (d->out_stride[0] | d->out_stride[1]) % 8 ||
        (d->k_stride[0] | d->k_stride[1] | d->k_stride[2]) % 8 ||
        (d->v_stride[0] | d->v_stride[1] | d->v_stride[2]) % 8)
      return PAD_ERR_ALIGNMENT;
    if (!L->range && !plan.single_pass && (!ws || ws_bytes < plan.workspace_bytes)) return PAD_ERR_WORKSPACE;
    if (!L->range && !plan.single_pass && (!counters || num_counters < plan.counters)) return PAD_ERR_WORKSPACE;
  }

  const int S = plan.num_splits;
  float* o_part = nullptr;
  float2* ml_part = nullptr;
  if (io && L->range)
    range_layout(d, rs, ws, &o_part, &ml_part);
  else if (io && !plan.single_pass)
    workspace_layout(d, S, ws, &o_part, &ml_part);

  RangeArgs& a = L->a;
  a.q = static_cast<const _Float16*>(q);
  a.k = static_cast<const _Float16*>(k);
  a.v = static_cast<const _Float16*>(v);
  a.bt = bt;
  a.sl = sl;
  a.indptr = indptr;
  a.lpl = lpl;
  a.worklist = nullptr;
  a.out = static_cast<_Float16*>(out);
  a.o_part = o_part;
  a.ml_part = ml_part;
  a.counters = counters;
  a.sqb = d->q_stride[0];
  a.sqh = d->q_stride[1];
  a.skp = d->k_stride[0];
  a.sks = d->k_stride[1];
  a.skh = d->k_stride[2];
  a.svp = d->v_stride[0];
  a.svs = d->v_stride[1];
  a.svh = d->v_stride[2];
  a.sbb = csr ? 0 : d->bt_stride[0];
  a.sbp = csr ? 1 : d->bt_stride[1];
  a.ssl = d->sl_stride;
  a.sob = d->out_stride[0];
  a.soh = d->out_stride[1];
  a.num_pages = d->num_pages;
  a.gqa = gqa;
  a.ps = d->page_size;
  a.pps = plan.pages_per_split;
  a.num_splits = S;
  a.hkv = d->num_kv_heads;
  a.max_pages = d->max_pages;
  a.batch = d->batch;
  a.csr = csr ? 1 : 0;
  // The in-kernel planner evens out ragged batches; an explicit split count
  // keeps its meaning (that many page-aligned splits per sequence).
  a.balance = 0;
  if (num_splits == 0 && !plan.single_pass && d->batch <= kPlanMaxBatch && d->max_pages < (1 << 23))
    a.balance = oversubscribed_shape(d, num_splits, cus, latency_bound_shape(d, cus, csr), kv_bytes) ? 2 : 1;
  a.min_chunk = ceil_div(kMinBlocks * kBlockTokens, d->page_size);
  a.pair_heads = ((d->head_dim * 2) % 128 != 0 && d->num_kv_heads % 2 == 0 &&
                  ((int64_t)S * d->num_kv_heads * d->batch) % 16 == 0) ? 1 : 0;
  if (a.balance == 2) {
    // An oversubscribed grid runs the static splits when every sequence is
    // at full capacity: pps is theirs (the grid's own split is the planner's
    // business), and balance = 1 + their count s0 per unit.  More than one
    // unit per four CUs leaves at most 3 (the budget over the units); with
    // more than one they take the first workgroups in order, unit-major,
    // so head pairing stays off.
    const int s0 = pps_full > 0 && d->max_pages > pps_full ? ceil_div(d->max_pages, pps_full) : 1;
    if (s0 <= 3) {
      a.pps = pps_full;
      a.balance = 1 + s0;
      if (s0 > 1) a.pair_heads = 0;
    } else {
      a.balance = 1;  // not reached; the planner of the grid as it is
    }
  }
  a.ps_shift = -1;
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == d->page_size) a.ps_shift = sh;
  a.scale_log2 = scale * kLog2e;
  a.v_fix = 1.0f;
  a.ks = a.vs = nullptr;
  a.sksp = a.skss = a.sksh = a.svsp = a.svss = a.svsh = 0;
  a.logits = a.lse = nullptr;
  a.slog = 0;
  a.hq = d->num_q_heads;
  a.fold_polls = 0;
  // The shared fold waits for a unit's other workgroups: only where the whole
  // grid can run at once, each unit has group counters, and a unit can get
  // the splits (the planner may give one more than S).
  const int total4 = gqa * (d->head_dim / 4);
  const int most_splits = a.balance ? (kTwoLevelSplits > total4 / 16 ? kTwoLevelSplits : total4 / 16) : S;
  if (!L->range && plan.counters > (int64_t)d->batch * d->num_kv_heads && engine == 0 &&
      most_splits * total4 >= kSharedFoldElements && (int64_t)S * d->num_kv_heads * d->batch <= cus)
    a.fold_polls = 32 + (int)((int64_t)plan.pages_per_split * d->page_size / 8);
#ifdef PAD_TIMELINE
  if (a.fold_polls > 0 && tl_fold_polls > 0) a.fold_polls = tl_fold_polls;
#endif
  a.nw = L->range ? rs.nw : plan.waves_per_group;
  a.groups = 0;
  a.unit_extra = 0;
  a.nh_shift = 0;
  a.rows = gqa;
  a.gqa_rcp = (65536u + gqa - 1) / gqa;
  if (L->range) {
    a.groups = rs.groups;
    a.nh_shift = rs.nh_shift;
    a.rows = gqa << rs.nh_shift;
    a.hkv = d->num_kv_heads >> rs.nh_shift;
    a.num_splits = a.pps = a.pair_heads = 0;
    a.balance = 1;
    a.min_chunk = rs.min_chunk;
    a.unit_extra = rs.unit_extra;
  }
  a.wl_key = plan_key(a);
#ifdef PAD_TIMELINE
  a.tl_launch = 0;
#endif
  L->nw = a.nw;
  L->lds = group_lds_bytes(L->nw, gqa, d->head_dim, engine, 1 << a.nh_shift);
  L->grid = dim3(S, d->num_kv_heads, d->batch);
  return PAD_OK;
}

// A known format; bfloat16 and fp8 on the MFMA engine; fp8 with head_dim
// 64/128/256 and finite positive scales (the scales are read for fp8 only).
static bool kv_format_fp8(int f) {
  return f == PAD_KV_FP8_E4M3FN || f == PAD_KV_FP8_E5M2 || f == PAD_KV_FP8_E4M3FN_BF16 || f == PAD_KV_FP8_E5M2_BF16;
}

// The kernels' element format (kKv*) of a PAD_KV_* code.
static int range_format(int kv_format) {
  switch (kv_format) {
    case PAD_KV_FP8_E4M3FN: return kKvE4M3;
    case PAD_KV_FP8_E5M2: return kKvE5M2;
    case PAD_KV_BF16: return kKvBF16;
    case PAD_KV_FP8_E4M3FN_BF16: return kKvE4M3B;
    case PAD_KV_FP8_E5M2_BF16: return kKvE5M2B;
    default: return kKvF16;
  }
}

static int check_kv_format(int kv_format, int engine, const pad_decode_dims* d, float k_scale, float v_scale) {
  if (kv_format == PAD_KV_FP16) return PAD_OK;
  if (kv_format == PAD_KV_BF16) return engine == 0 ? PAD_OK : PAD_ERR_KV_FORMAT;
  if (!kv_format_fp8(kv_format)) return PAD_ERR_KV_FORMAT;
  if (engine != 0) return PAD_ERR_KV_FORMAT;
  if (d && d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return PAD_ERR_UNSUPPORTED_HEAD_DIM;
  if (!(k_scale > 0.0f) || !(v_scale > 0.0f) || k_scale > 1.0e30f || v_scale > 1.0e30f) return PAD_ERR_KV_FORMAT;
  return PAD_OK;
}

// kv_format: PAD_KV_FP16, or an fp8 format with per-tensor scales k_scale,
// v_scale (the caches hold K / k_scale and V / v_scale).
static int launch_impl(const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* sl,
                       const int32_t* indptr, const int32_t* lpl, void* out, void* ws, size_t ws_bytes,
                       int32_t* counters, int64_t num_counters, const pad_decode_dims* d, float scale,
                       int num_splits, int engine, void* const* events, void* stream,
                       const void* worklist = nullptr, size_t worklist_bytes = 0, int kv_format = PAD_KV_FP16,
                       float k_scale = 1.0f, float v_scale = 1.0f) {
  int st = check_kv_format(kv_format, engine, d, k_scale, v_scale);
  if (st != PAD_OK) return st;
  Launch L;
  const bool fp8 = kv_format_fp8(kv_format);
  st = setup_launch(q, k, v, bt, sl, indptr, lpl, out, ws, ws_bytes, counters, num_counters, d, scale,
                    num_splits, engine, true, &L, fp8 ? 1 : 2, worklist ? worklist_bytes : SIZE_MAX);
  if (st != PAD_OK || L.empty) return st;
  if (fp8) {
    // The caches hold K / k_scale and V / v_scale: k_scale multiplies every
    // score, v_scale every output row.
    L.a.scale_log2 *= k_scale;
    L.a.v_fix = v_scale;
  }
  if (worklist != nullptr) {
    if (worklist_bytes < worklist_bytes_for(L.plan, d)) return PAD_ERR_WORKSPACE;
    L.a.worklist = static_cast<const int32_t*>(worklist);
  }
#ifdef PAD_TIMELINE
  L.a.tl_launch = tl_launches++ % PAD_TL_LAUNCHES;
#endif
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  if (events && events[0] && hipEventRecord(reinterpret_cast<hipEvent_t>(events[0]), hs) != hipSuccess)
    return PAD_ERR_LAUNCH;
  hipError_t e;
#ifndef PAD_TIMELINE
  if (L.range) {
    e = launch_range(L.a, d->head_dim, range_format(kv_format), L.nw, L.lds, hs);
  } else
#endif
  if (kv_format == PAD_KV_FP8_E4M3FN) {
    e = dispatch_kvf_dim<kKvE4M3>(L.a, d->head_dim, L.grid, L.nw, L.lds, hs);
  } else if (kv_format == PAD_KV_FP8_E5M2) {
    e = dispatch_kvf_dim<kKvE5M2>(L.a, d->head_dim, L.grid, L.nw, L.lds, hs);
  } else if (kv_format == PAD_KV_BF16) {
    e = dispatch_kvf_dim<kKvBF16>(L.a, d->head_dim, L.grid, L.nw, L.lds, hs);
  } else if (kv_format == PAD_KV_FP8_E4M3FN_BF16) {
    e = dispatch_kvf_dim<kKvE4M3B>(L.a, d->head_dim, L.grid, L.nw, L.lds, hs);
  } else if (kv_format == PAD_KV_FP8_E5M2_BF16) {
    e = dispatch_kvf_dim<kKvE5M2B>(L.a, d->head_dim, L.grid, L.nw, L.lds, hs);
  } else switch (d->head_dim) {
    case 32: e = dispatch_phase1<32>(L.a, L.grid, L.nw, L.lds, engine, hs); break;
    case 64: e = dispatch_phase1<64>(L.a, L.grid, L.nw, L.lds, engine, hs); break;
    case 96: e = dispatch_phase1<96>(L.a, L.grid, L.nw, L.lds, engine, hs); break;
    case 128: e = dispatch_phase1<128>(L.a, L.grid, L.nw, L.lds, engine, hs); break;
    default: e = dispatch_phase1<256>(L.a, L.grid, L.nw, L.lds, engine, hs); break;
  }
  if (e != hipSuccess) return PAD_ERR_LAUNCH;
  if (events && events[1] && hipEventRecord(reinterpret_cast<hipEvent_t>(events[1]), hs) != hipSuccess)
    return PAD_ERR_LAUNCH;
  if (events && events[2] && hipEventRecord(reinterpret_cast<hipEvent_t>(events[2]), hs) != hipSuccess)
    return PAD_ERR_LAUNCH;
  return PAD_OK;
}

#ifndef PAD_TIMELINE
// Floats of a query head's scores: a table row's tokens, in whole vectors of four.
static int64_t logit_row_floats(const pad_decode_dims* d) { return ((int64_t)d->max_pages * d->page_size + 3) & ~3ll; }

static size_t logits_bytes_of(const pad_decode_dims* d) {
  const size_t rows = (size_t)d->batch * d->num_q_heads;
  return 256 + rows * sizeof(float) * ((size_t)logit_row_floats(d) + 1);
}

// A decode over MX4 caches, or one that adds up attention weights, or both.
static int launch_cache_call(const pad_cache_call* cc, const pad_decode_dims* d, hipStream_t hs) {
  const pad_decode_call& c = cc->call;
  const bool mx4 = c.kv_format == PAD_KV_MX4 || c.kv_format == PAD_KV_MX4_BF16;
  const bool fp8 = kv_format_fp8(c.kv_format);
  int st = validate_dims(d);
  if (st != PAD_OK) return st;
  if (c.indptr || c.last_page_len || c.worklist) return PAD_ERR_INVALID_SHAPE;
  if (!mx4 && !cc->weights) return PAD_ERR_KV_FORMAT;  // pad_decode_launch_call()'s
  if (mx4) {
    if (c.engine != 0) return PAD_ERR_KV_FORMAT;
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return PAD_ERR_UNSUPPORTED_HEAD_DIM;
    if (d->batch > 0 && (!cc->k_scales || !cc->v_scales)) return PAD_ERR_NULL_POINTER;
    // Strides are multiplied as unsigned 32-bit values.
    for (int i = 0; i < 2; ++i)
      for (int64_t x : {d->k_stride[i], d->v_stride[i], cc->ks_stride[i], cc->vs_stride[i]})
        if (x < 0 || x > UINT32_MAX) return PAD_ERR_STRIDE;
    // A lane reads 16 bytes of a row at once, 8 at head_dim 64.
    if (d->head_dim >= 128 && ((d->k_stride[0] | d->k_stride[1] | d->k_stride[2] | d->v_stride[0] | d->v_stride[1] |
                                d->v_stride[2]) & 15))
      return PAD_ERR_ALIGNMENT;
  } else {
    st = check_kv_format(c.kv_format, c.engine, d, c.k_scale, c.v_scale);
    if (st != PAD_OK) return st;
    if (c.engine != 0) return PAD_ERR_KV_FORMAT;
    // A block's rows are addressed with 32-bit offsets.
    for (int64_t x : {d->k_stride[1], d->v_stride[1]})
      if (x < 0 || x > UINT32_MAX / 32 - 64) return PAD_ERR_STRIDE;
  }
  // The launch counts the tokens of a table row in 32 bits.
  if ((int64_t)d->max_pages * d->page_size > INT32_MAX - 4096) return PAD_ERR_INVALID_SHAPE;
  // A kv head's scores are one buffer with 32-bit offsets.
  if (cc->weights && logit_row_floats(d) * (d->num_q_heads / d->num_kv_heads) >= (1ll << 30) - 1024)
    return PAD_ERR_INVALID_SHAPE;
  Launch L;
  st = setup_launch(c.q, c.k_cache, c.v_cache, c.block_table, c.seq_lens, nullptr, nullptr, c.out, c.workspace,
                    c.workspace_bytes, c.counters, c.num_counters, d, c.scale, c.num_splits, 0, true, &L,
                    mx4 || fp8 ? 1 : 2, SIZE_MAX, mx4);
  if (st != PAD_OK || L.empty) return st;
  if (fp8) {
    L.a.scale_log2 *= c.k_scale;
    L.a.v_fix = c.v_scale;
  }
  int kvf = mx4 ? (c.kv_format == PAD_KV_MX4 ? kKvMx4 : kKvMx4B) : range_format(c.kv_format);
  L.a.ks = cc->k_scales;
  L.a.vs = cc->v_scales;
  L.a.sksp = cc->ks_stride[0];
  L.a.skss = cc->ks_stride[1];
  L.a.sksh = cc->ks_stride[2];
  L.a.svsp = cc->vs_stride[0];
  L.a.svss = cc->vs_stride[1];
  L.a.svsh = cc->vs_stride[2];
  if (cc->weights) {
    if (!cc->logits || cc->logits_bytes < logits_bytes_of(d)) return PAD_ERR_WORKSPACE;
    L.a.slog = logit_row_floats(d);
    L.a.logits = reinterpret_cast<float*>(((uintptr_t)cc->logits + 255u) & ~(uintptr_t)255u);
    L.a.lse = L.a.logits + (size_t)d->batch * d->num_q_heads * L.a.slog;
    L.a.fold_polls = 0;  // these instantiations have no shared fold
  }
  hipError_t e;
  if (mx4)
    e = launch_mx4(L.a, L.range, d->head_dim, kvf | (cc->weights ? kKvWeights : 0), L.grid, L.nw, L.lds, hs);
  else if (fp8)
    e = launch_weights_fp8(L.a, L.range, d->head_dim, kvf, L.grid, L.nw, L.lds, hs);
  else
    e = launch_weights(L.a, L.range, d->head_dim, kvf, L.grid, L.nw, L.lds, hs);
  if (e != hipSuccess) return PAD_ERR_LAUNCH;
  if (cc->weights && d->max_pages > 0 && launch_accumulate(L.a, cc->weights, cc->w_stride, hs) != hipSuccess)
    return PAD_ERR_LAUNCH;
  return PAD_OK;
}
#endif

// Writes the work list of a launch with these dims and indices (one wave per
// workgroup slot of the decode grid).
// kv_bytes: bytes per K/V element of the launch the list is for (the wave
// count, and so the list's plan key, depends on it).
static int plan_worklist_impl(const int32_t* bt, const int32_t* sl, const int32_t* indptr, const int32_t* lpl,
                              const pad_decode_dims* d, int num_splits, void* worklist, size_t worklist_bytes,
                              void* stream, int kv_bytes = 2) {
  Launch L;
  int st = setup_launch(nullptr, nullptr, nullptr, bt, sl, indptr, lpl, nullptr, nullptr, 0, nullptr, 0, d, 1.0f,
                        num_splits, 0, false, &L, kv_bytes, worklist_bytes);
  if (st != PAD_OK) return st;
  if (!worklist) return PAD_ERR_NULL_POINTER;
  if (worklist_bytes < worklist_bytes_for(L.plan, d)) return PAD_ERR_WORKSPACE;
  if (L.empty) return PAD_OK;
#ifndef PAD_TIMELINE
  if (L.range)
    return launch_range_plan(L.a, static_cast<int32_t*>(worklist), reinterpret_cast<hipStream_t>(stream)) == hipSuccess
               ? PAD_OK
               : PAD_ERR_LAUNCH;
#endif
  hipLaunchKernelGGL(pad_plan_kernel, L.grid, dim3(64), 0, reinterpret_cast<hipStream_t>(stream), L.a,
                     static_cast<int32_t*>(worklist));
  return hipGetLastError() == hipSuccess ? PAD_OK : PAD_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
// Allocation-free launches (pad_decode_launch_noalloc): the split scratch is
// a file-scope device array instead of caller memory.  Layout: the int32
// arrival counters first (PAD_NOALLOC_COUNTERS of them), then the partials
// workspace (PAD_NOALLOC_WORKSPACE_BYTES).  Every GPU the library runs on
// holds its own copy until the process ends.  In host code `scratch` names a
// host-side stand-in, not device memory: the per-device address comes from
// hipGetSymbolAddress once per device and only that address is used.
// ---------------------------------------------------------------------------
constexpr size_t kNoallocCounterBytes = (size_t)PAD_NOALLOC_COUNTERS * sizeof(int32_t);
static __device__ __align__(256) unsigned char scratch[kNoallocCounterBytes + PAD_NOALLOC_WORKSPACE_BYTES];

constexpr int kMaxDevices = 64;
static void* g_scratch_ptr[kMaxDevices];
static std::mutex g_scratch_mu;

// Zeroes n int32 values with vector stores (used for the counters once per
// device; a kernel rather than hipMemsetAsync so that a call made under
// stream capture records a kernel node).
__global__ void pad_zero_i32_kernel(int32_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    p[i] = 0;
}

// The current device's scratch address; the first call on a device looks it
// up (with that device current) and queues a clear of its counters on
// `stream`, ahead of the caller's launch.  The array is zero when the code
// object loads, and every launch leaves the counters zero again, so the
// clear only makes that state explicit.
static int noalloc_scratch(hipStream_t stream, unsigned char** out) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return PAD_ERR_DEVICE;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* ptr = nullptr;
    if (hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)) != hipSuccess || !ptr) return PAD_ERR_DEVICE;
    hipLaunchKernelGGL(pad_zero_i32_kernel, dim3(64), dim3(256), 0, stream, static_cast<int32_t*>(ptr),
                       (int64_t)PAD_NOALLOC_COUNTERS);
    if (hipGetLastError() != hipSuccess) return PAD_ERR_LAUNCH;
    g_scratch_ptr[dev] = ptr;
  }
  *out = static_cast<unsigned char*>(g_scratch_ptr[dev]);
  return PAD_OK;
}

static int launch_noalloc(const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* sl,
                          void* out, const pad_decode_dims* d, float scale, int num_splits, void* stream) {
  if (d && d->batch > 0 && d->max_pages > 0 && d->num_pages <= 0) return PAD_ERR_INVALID_SHAPE;
  int cus = 0;
  int st = device_cus(&cus);
  if (st != PAD_OK) return st;
  // What the launch needs at least: one whose range launch does not fit the
  // static scratch runs the per-unit kernel.
  pad_decode_plan_t plan;
  st = plan_units(d, num_splits, cus, 0, false, &plan);
  if (st != PAD_OK) return st;
  if (plan.workspace_bytes > PAD_NOALLOC_WORKSPACE_BYTES || plan.counters > PAD_NOALLOC_COUNTERS)
    return PAD_ERR_SCRATCH_LIMIT;
  unsigned char* base = nullptr;
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  st = noalloc_scratch(hs, &base);
  if (st != PAD_OK) return st;
  return launch_impl(q, k, v, bt, sl, nullptr, nullptr, out, base + kNoallocCounterBytes,
                     PAD_NOALLOC_WORKSPACE_BYTES, reinterpret_cast<int32_t*>(base), PAD_NOALLOC_COUNTERS, d, scale,
                     num_splits, 0, nullptr, stream);
}

}  // namespace pad

extern "C" {

int pad_decode_plan(const pad_decode_dims* dims, int num_splits, int num_cus, pad_decode_plan_t* plan) {
  if (!plan) return PAD_ERR_NULL_POINTER;
  return pad::plan_impl(dims, num_splits, num_cus, 0, false, plan);
}

int pad_decode_plan_csr(const pad_decode_dims* dims, int num_splits, int num_cus, pad_decode_plan_t* plan) {
  if (!plan) return PAD_ERR_NULL_POINTER;
  return pad::plan_impl(dims, num_splits, num_cus, 0, true, plan);
}

int pad_decode_workspace_bytes(const pad_decode_dims* dims, int num_splits, int num_cus, size_t* bytes) {
  if (!bytes) return PAD_ERR_NULL_POINTER;
  pad_decode_plan_t p;
  const int st = pad::plan_impl(dims, num_splits, num_cus, 0, false, &p);
  if (st != PAD_OK) return st;
  *bytes = p.workspace_bytes;
  return PAD_OK;
}

int pad_decode_counters_needed(const pad_decode_dims* dims, int num_splits, int num_cus, int64_t* count) {
  if (!count) return PAD_ERR_NULL_POINTER;
  pad_decode_plan_t p;
  const int st = pad::plan_impl(dims, num_splits, num_cus, 0, false, &p);
  if (st != PAD_OK) return st;
  *count = p.counters;
  return PAD_OK;
}

int pad_decode_least_scratch(const pad_decode_dims* dims, int num_splits, int num_cus, int csr, size_t* bytes,
                             int64_t* count) {
  if (!bytes || !count) return PAD_ERR_NULL_POINTER;
  pad_decode_plan_t p;
  const int st = pad::plan_units(dims, num_splits, num_cus, 0, csr != 0, &p);
  if (st != PAD_OK) return st;
  *bytes = p.workspace_bytes;
  *count = p.counters;
  return PAD_OK;
}

int pad_decode_launch(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                      const int32_t* seq_lens, void* out, void* workspace, size_t workspace_bytes,
                      int32_t* counters, int64_t num_counters, const pad_decode_dims* dims, float scale,
                      int num_splits, void* stream) {
  return pad::launch_impl(q, k_cache, v_cache, block_table, seq_lens, nullptr, nullptr, out, workspace,
                          workspace_bytes, counters, num_counters, dims, scale, num_splits, 0, nullptr, stream);
}

int pad_decode_launch_csr(const void* q, const void* k_cache, const void* v_cache, const int32_t* indices,
                          const int32_t* indptr, const int32_t* last_page_len, void* out, void* workspace,
                          size_t workspace_bytes, int32_t* counters, int64_t num_counters,
                          const pad_decode_dims* dims, float scale, int num_splits, int engine, void* stream) {
  if (!indptr || !last_page_len) return PAD_ERR_NULL_POINTER;
  return pad::launch_impl(q, k_cache, v_cache, indices, nullptr, indptr, last_page_len, out, workspace,
                          workspace_bytes, counters, num_counters, dims, scale, num_splits, engine, nullptr, stream);
}

int pad_decode_launch_ex(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                         const int32_t* seq_lens, void* out, void* workspace, size_t workspace_bytes,
                         int32_t* counters, int64_t num_counters, const pad_decode_dims* dims, float scale,
                         int num_splits, int engine, void* const* events, void* stream) {
  return pad::launch_impl(q, k_cache, v_cache, block_table, seq_lens, nullptr, nullptr, out, workspace,
                          workspace_bytes, counters, num_counters, dims, scale, num_splits, engine, events, stream);
}

int pad_decode_launch_kv8(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                          const int32_t* seq_lens, void* out, void* workspace, size_t workspace_bytes,
                          int32_t* counters, int64_t num_counters, const pad_decode_dims* dims, float scale,
                          int kv_format, float k_scale, float v_scale, int num_splits, void* stream) {
  // fp16 caches: pad_decode_launch; bfloat16: pad_decode_launch_call
  if (!pad::kv_format_fp8(kv_format)) return PAD_ERR_KV_FORMAT;
  return pad::launch_impl(q, k_cache, v_cache, block_table, seq_lens, nullptr, nullptr, out, workspace,
                          workspace_bytes, counters, num_counters, dims, scale, num_splits, 0, nullptr, stream,
                          nullptr, 0, kv_format, k_scale, v_scale);
}

int pad_decode_launch_noalloc(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                              const int32_t* seq_lens, void* out, const pad_decode_dims* dims, float scale,
                              int num_splits, void* stream) {
  return pad::launch_noalloc(q, k_cache, v_cache, block_table, seq_lens, out, dims, scale, num_splits, stream);
}

int pad_decode_worklist_bytes(const pad_decode_dims* dims, int num_splits, int num_cus, int csr, size_t* bytes) {
  if (!bytes) return PAD_ERR_NULL_POINTER;
  pad_decode_plan_t p;
  const int st = pad::plan_impl(dims, num_splits, num_cus, 0, csr != 0, &p);
  if (st != PAD_OK) return st;
  *bytes = pad::worklist_bytes_for(p, dims);
  return PAD_OK;
}

int pad_decode_plan_worklist(const int32_t* block_table, const int32_t* seq_lens, const pad_decode_dims* dims,
                             int num_splits, void* worklist, size_t worklist_bytes, void* stream) {
  return pad::plan_worklist_impl(block_table, seq_lens, nullptr, nullptr, dims, num_splits, worklist, worklist_bytes,
                                 stream);
}

int pad_decode_plan_worklist_csr(const int32_t* indices, const int32_t* indptr, const int32_t* last_page_len,
                                 const pad_decode_dims* dims, int num_splits, void* worklist, size_t worklist_bytes,
                                 void* stream) {
  if (!indptr || !last_page_len) return PAD_ERR_NULL_POINTER;
  return pad::plan_worklist_impl(indices, nullptr, indptr, last_page_len, dims, num_splits, worklist,
                                 worklist_bytes, stream);
}

int pad_decode_launch_worklist(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                               const int32_t* seq_lens, void* out, void* workspace, size_t workspace_bytes,
                               int32_t* counters, int64_t num_counters, const pad_decode_dims* dims, float scale,
                               int num_splits, const void* worklist, size_t worklist_bytes, void* stream) {
  if (!worklist) return PAD_ERR_NULL_POINTER;
  return pad::launch_impl(q, k_cache, v_cache, block_table, seq_lens, nullptr, nullptr, out, workspace,
                          workspace_bytes, counters, num_counters, dims, scale, num_splits, 0, nullptr, stream,
                          worklist, worklist_bytes);
}

int pad_decode_launch_worklist_csr(const void* q, const void* k_cache, const void* v_cache, const int32_t* indices,
                                   const int32_t* indptr, const int32_t* last_page_len, void* out, void* workspace,
                                   size_t workspace_bytes, int32_t* counters, int64_t num_counters,
                                   const pad_decode_dims* dims, float scale, int num_splits, const void* worklist,
                                   size_t worklist_bytes, void* stream) {
  if (!indptr || !last_page_len || !worklist) return PAD_ERR_NULL_POINTER;
  return pad::launch_impl(q, k_cache, v_cache, indices, nullptr, indptr, last_page_len, out, workspace,
                          workspace_bytes, counters, num_counters, dims, scale, num_splits, 0, nullptr, stream,
                          worklist, worklist_bytes);
}

int pad_decode_launch_call(const pad_decode_call* c, const pad_decode_dims* dims, void* stream) {
  if (!c) return PAD_ERR_NULL_POINTER;
  const bool csr = c->indptr != nullptr || c->last_page_len != nullptr;
  if (csr && (!c->indptr || !c->last_page_len)) return PAD_ERR_NULL_POINTER;
  if (c->worklist && c->engine != 0) return PAD_ERR_INVALID_SHAPE;  // work lists serve the MFMA engine
  return pad::launch_impl(c->q, c->k_cache, c->v_cache, c->block_table, csr ? nullptr : c->seq_lens, c->indptr,
                          c->last_page_len, c->out, c->workspace, c->workspace_bytes, c->counters, c->num_counters,
                          dims, c->scale, c->num_splits, c->engine, nullptr, stream, c->worklist, c->worklist_bytes,
                          c->kv_format, c->k_scale, c->v_scale);
}

int pad_decode_plan_worklist_call(const pad_decode_call* c, const pad_decode_dims* dims, void* worklist,
                                  size_t worklist_bytes, void* stream) {
  if (!c) return PAD_ERR_NULL_POINTER;
  const bool csr = c->indptr != nullptr || c->last_page_len != nullptr;
  if (csr && (!c->indptr || !c->last_page_len)) return PAD_ERR_NULL_POINTER;
  if (c->engine != 0) return PAD_ERR_INVALID_SHAPE;  // work lists serve the MFMA engine
  const int st = pad::check_kv_format(c->kv_format, 0, dims, c->k_scale, c->v_scale);
  if (st != PAD_OK) return st;
  const bool fp8 = pad::kv_format_fp8(c->kv_format);
  return pad::plan_worklist_impl(c->block_table, csr ? nullptr : c->seq_lens, c->indptr, c->last_page_len, dims,
                                 c->num_splits, worklist, worklist_bytes, stream, fp8 ? 1 : 2);
}

int pad_decode_counters_init(int32_t* counters, int64_t num_counters, void* stream) {
  if (!counters) return PAD_ERR_NULL_POINTER;
  if (num_counters <= 0) return PAD_OK;
  // A fill kernel, not hipMemsetAsync: under stream capture this records a
  // kernel node, which replays correctly.
  const int64_t blocks = (num_counters + 255) / 256;
  hipLaunchKernelGGL(pad::pad_zero_i32_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), counters, num_counters);
  return hipGetLastError() == hipSuccess ? PAD_OK : PAD_ERR_LAUNCH;
}

int pad_device_num_cus(int* num_cus) {
  if (!num_cus) return PAD_ERR_NULL_POINTER;
  return pad::device_cus(num_cus);
}

const char* pad_status_string(int status) {
  switch (status) {
    case PAD_OK: return "ok";
    case PAD_ERR_NULL_POINTER: return "a required pointer is NULL";
    case PAD_ERR_INVALID_SHAPE: return "invalid shape (non-positive or inconsistent sizes)";
    case PAD_ERR_UNSUPPORTED_HEAD_DIM: return "unsupported head_dim (supported: 32, 64, 96, 128, 256)";
    case PAD_ERR_UNSUPPORTED_GQA:
      return "unsupported GQA group (num_q_heads must be a multiple of num_kv_heads, ratio <= 16)";
    case PAD_ERR_STRIDE: return "head_dim must be contiguous (stride 1) for q, k_cache, v_cache and out";
    case PAD_ERR_ALIGNMENT: return "q/k_cache/v_cache/out rows must be 16-byte aligned";
    case PAD_ERR_WORKSPACE:
      return "workspace/counters NULL or smaller than pad_decode_workspace_bytes()/pad_decode_counters_needed()";
    case PAD_ERR_NUM_SPLITS: return "num_splits must be in [0, 1024]";
    case PAD_ERR_LAUNCH: return "kernel launch failed";
    case PAD_ERR_DEVICE: return "no usable HIP device";
    case PAD_ERR_SCRATCH_LIMIT:
      return "the call needs more split scratch than pad_decode_launch_noalloc's static buffer holds "
             "(PAD_NOALLOC_WORKSPACE_BYTES of partials, PAD_NOALLOC_COUNTERS counters); use pad_decode_launch";
    case PAD_ERR_KV_FORMAT:
      return "unsupported K/V cache format or scale (fp8: PAD_KV_FP8_E4M3FN / _E5M2 (fp16 q) or _BF16 (bfloat16 "
             "q), MFMA engine, head_dim 64/128/256, finite positive k_scale and v_scale; PAD_KV_BF16: MFMA engine)";
    default: return "unknown status";
  }
}

int pad_decode_abi_version(void) { return PAD_ABI_VERSION; }

#ifdef PAD_TIMELINE
int pad_timeline_read(void* host, size_t bytes) {
  if (!host) return PAD_ERR_NULL_POINTER;
  const size_t n = bytes < sizeof(pad::tl_buf) ? bytes : sizeof(pad::tl_buf);
  return hipMemcpyFromSymbol(host, HIP_SYMBOL(pad::tl_buf), n, 0, hipMemcpyDeviceToHost) == hipSuccess
             ? PAD_OK
             : PAD_ERR_DEVICE;
}

int pad_timeline_reset(void) {
  void* p = nullptr;
  if (hipGetSymbolAddress(&p, HIP_SYMBOL(pad::tl_buf)) != hipSuccess) return PAD_ERR_DEVICE;
  if (hipMemset(p, 0, sizeof(pad::tl_buf)) != hipSuccess || hipDeviceSynchronize() != hipSuccess)
    return PAD_ERR_DEVICE;
  pad::tl_launches = 0;
  return PAD_OK;
}

int pad_timeline_set_fold_polls(int polls) {
  pad::tl_fold_polls = polls > 0 ? polls : 0;
  return PAD_OK;
}
#endif

#ifndef PAD_TIMELINE
int pad_cache_logits_bytes(const pad_decode_dims* dims, size_t* bytes) {
  const int st = pad::validate_dims(dims);
  if (st != PAD_OK) return st;
  if (!bytes) return PAD_ERR_NULL_POINTER;
  *bytes = pad::logits_bytes_of(dims);
  return PAD_OK;
}

int pad_cache_scratch(const pad_decode_dims* dims, int kv_format, int num_splits, int num_cus, size_t* bytes,
                      int64_t* count) {
  if (!bytes || !count) return PAD_ERR_NULL_POINTER;
  const bool mx4 = kv_format == PAD_KV_MX4 || kv_format == PAD_KV_MX4_BF16;
  if (!mx4 && pad::check_kv_format(kv_format, 0, dims, 1.0f, 1.0f) != PAD_OK) return PAD_ERR_KV_FORMAT;
  const int kv_bytes = mx4 || pad::kv_format_fp8(kv_format) ? 1 : 2;
  pad_decode_plan_t p;
  const int st = pad::plan_units(dims, num_splits, num_cus, 0, false, &p, kv_bytes);
  if (st != PAD_OK) return st;
  const pad::RangeShape r = pad::range_shape(dims, num_splits, num_cus, 0, false, kv_bytes, mx4);
  *bytes = r.groups > 0 && r.workspace_bytes > p.workspace_bytes ? r.workspace_bytes : p.workspace_bytes;
  *count = r.groups > 0 && r.counters > p.counters ? r.counters : p.counters;
  return PAD_OK;
}

int pad_cache_decode(const pad_cache_call* call, const pad_decode_dims* dims, void* stream) {
  if (!call || !dims) return PAD_ERR_NULL_POINTER;
  return pad::launch_cache_call(call, dims, reinterpret_cast<hipStream_t>(stream));
}
#endif

}  // extern "C"
