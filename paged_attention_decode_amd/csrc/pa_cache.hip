// pa_cache.hip - gfx950 kernels that write, read and thin out a paged K/V cache:
// append, read, the accumulation of attention weights, and eviction
// (include/pa_cache.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pa_cache.h"
#include "pa_device.h"
#include "pa_ext.h"

namespace pad {

typedef float f2_t __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------------------
// Append and read.  A thread has eight elements of a row of K and of V (16 bytes
// of 16-bit values each); the four lanes of an MX4 block find its largest value
// together.  Bound by memory: the rows are read (or written) once, the cache's
// the other way.  (One of K and V a thread and 64-bit index arithmetic: 16000
// MX4 rows of 8 heads 23.4 + 19.0 us; so 20.8 + 17.0.)
// ---------------------------------------------------------------------------
constexpr int kRows16 = 0, kRowsE4M3 = 1, kRowsE5M2 = 2, kRowsMx4 = 3;  // kinds of cache rows

struct RowArgs {
  pad_kv_cache c;
  pad_kv_rows r;
  const float* token_weights;
  const int32_t* token_positions;
  uint32_t rows;  // tokens * kv heads
  int row8;       // head_dim / 8
  int row8_shift, ps_shift, head_shift;  // log2 where a power of two, else -1
  int same;       // K and V (and their scales) have the same strides
};

__device__ __forceinline__ uint32_t divide(uint32_t x, int shift, uint32_t by) { return shift >= 0 ? x >> shift : x / by; }

__device__ __forceinline__ int64_t slot_of(const RowArgs& a, uint32_t token) {
  return a.r.slots64 ? static_cast<const int64_t*>(a.r.slots)[token] : static_cast<const int32_t*>(a.r.slots)[token];
}

// The thread's row and eight elements of it; false past the last row.
struct RowPart {
  uint32_t row, token, h, e8;
};
__device__ __forceinline__ bool row_part(const RowArgs& a, RowPart& p) {
  // Workgroups have whole rows (256 is a multiple of row8 but at head_dim 96:
  // 252 threads of 21 rows).
  const uint32_t per = a.row8_shift >= 0 ? 256u >> a.row8_shift : 256u / (uint32_t)a.row8;
  const uint32_t sub = divide(threadIdx.x, a.row8_shift, a.row8);
  if (sub >= per) return false;
  p.row = blockIdx.x * per + sub;
  p.e8 = threadIdx.x - sub * a.row8;
  p.token = divide(p.row, a.head_shift, a.c.num_kv_heads);
  p.h = p.row - p.token * a.c.num_kv_heads;
  return p.row < a.rows;
}

// Strides are below 2^32 (check_cache), so that each product is one instruction.
__device__ __forceinline__ uint64_t offset_of(const int64_t* st, uint32_t page, uint32_t at, uint32_t h) {
  return (uint64_t)page * (uint32_t)st[0] + (uint64_t)at * (uint32_t)st[1] + (uint64_t)h * (uint32_t)st[2];
}

// Page and place of a slot; false for one outside the cache.
__device__ __forceinline__ bool place_of(const RowArgs& a, int64_t s, uint32_t& page, uint32_t& at) {
  if (s < 0) return false;
  int64_t p;
  if (a.ps_shift >= 0) {
    p = s >> a.ps_shift;
  } else if (s < (1ll << 32)) {
    p = (uint32_t)s / (uint32_t)a.c.page_size;
  } else {
    p = s / a.c.page_size;
  }
  if (p >= a.c.num_pages) return false;
  page = (uint32_t)p;
  at = (uint32_t)(s - p * a.c.page_size);
  return true;
}

template <bool BF16>
__device__ __forceinline__ void unpack8(u4_t w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const h2_t h = __builtin_bit_cast(h2_t, (uint32_t)w[i]);
      x[2 * i] = (float)h.x;
      x[2 * i + 1] = (float)h.y;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ u4_t pack8(const float (&x)[8]) {
  u4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2_t{x[2 * i], x[2 * i + 1]}, b2_t));
    } else {
      w[i] = __builtin_bit_cast(uint32_t, h2_t{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
    }
  }
  return w;
}

// Four values / scale as fp8 codes, held to the largest finite value (a
// comparison with NaN is false, so NaN stays).
template <int KIND>
__device__ __forceinline__ uint32_t fp8x4(const float* x, float scale) {
  constexpr float kMax = KIND == kRowsE4M3 ? 448.f : 57344.f;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float v = x[i] / scale;
    y[i] = v > kMax ? kMax : (v < -kMax ? -kMax : v);
  }
  int w = 0;
  if constexpr (KIND == kRowsE4M3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], w, true);
  }
  return (uint32_t)w;
}

// One row's eight elements into a cache, at element (byte) `off` of the row's place.
template <int KIND, bool BF16>
__device__ __forceinline__ void store_part(u4_t w, void* cache, uint8_t* scales, uint64_t off, uint64_t scale_off,
                                           float scale, uint32_t e8) {
  char* base = static_cast<char*>(cache);
  if constexpr (KIND == kRows16) {
    *reinterpret_cast<u4_t*>(base + (off + e8 * 8) * 2) = w;
  } else {
    float x[8];
    unpack8<BF16>(w, x);
    if constexpr (KIND == kRowsMx4) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));  // the block's four lanes
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
      const int e = (int)(top >> 23);  // biased; 255: NaN or infinity
      const uint32_t s = e == 255 ? 255u : (uint32_t)max(e - 2, 0);
      // v_cvt_scalef32_pk_fp4_f32 divides by the scale, rounds to nearest even
      // and saturates (exponent byte 0 stands for 2^-127).
      const float by = __uint_as_float(s << 23);
      uint32_t codes = 0;
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], by, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], by, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], by, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], by, 3);
      *reinterpret_cast<uint32_t*>(base + off + e8 * 4) = e == 255 ? 0u : codes;
      if ((e8 & 3) == 0) scales[scale_off + (e8 >> 2)] = (uint8_t)s;
    } else {
      *reinterpret_cast<u2_t*>(base + off + e8 * 8) = u2_t{fp8x4<KIND>(x, scale), fp8x4<KIND>(x + 4, scale)};
    }
  }
}

template <int KIND, bool BF16>
__global__ __launch_bounds__(256) void pad_append_kernel(const RowArgs a) {
  RowPart p;
  if (!row_part(a, p)) return;
  const _Float16* ks = static_cast<const _Float16*>(a.r.k) + (int64_t)p.token * a.r.k_stride[0] +
                       (int64_t)p.h * a.r.k_stride[1] + p.e8 * 8;
  const _Float16* vs = static_cast<const _Float16*>(a.r.v) + (int64_t)p.token * a.r.v_stride[0] +
                       (int64_t)p.h * a.r.v_stride[1] + p.e8 * 8;
  const u4_t k = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(ks));
  const u4_t v = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(vs));
  // A row's threads (and so an MX4 block's four lanes) go on or leave together.
  uint32_t page, at;
  if (!place_of(a, slot_of(a, p.token), page, at)) return;
  const uint64_t koff = offset_of(a.c.k_stride, page, at, p.h);
  const uint64_t voff = a.same ? koff : offset_of(a.c.v_stride, page, at, p.h);
  uint64_t ksoff = 0, vsoff = 0;
  if constexpr (KIND == kRowsMx4) {
    ksoff = offset_of(a.c.ks_stride, page, at, p.h);
    vsoff = a.same ? ksoff : offset_of(a.c.vs_stride, page, at, p.h);
  }
  store_part<KIND, BF16>(k, a.c.k, a.c.k_scales, koff, ksoff, a.c.k_scale, p.e8);
  store_part<KIND, BF16>(v, a.c.v, a.c.v_scales, voff, vsoff, a.c.v_scale, p.e8);
  if (p.e8 == 0) {
    if (a.c.weights)
      a.c.weights[offset_of(a.c.w_stride, page, at, p.h)] = a.token_weights ? a.token_weights[p.row] : 0.f;
    if (a.c.positions) a.c.positions[offset_of(a.c.p_stride, page, at, p.h)] = a.token_positions[p.token];
  }
}

// Eight elements of a row as 16-bit values; the cache's words are loaded first
// (load_part), so that K's and V's are in flight together.
template <int KIND>
struct Part {
  u4_t w;
  uint32_t scale;
};
template <int KIND>
__device__ __forceinline__ Part<KIND> load_part(const void* cache, const uint8_t* scales, uint64_t off,
                                                uint64_t scale_off, uint32_t e8) {
  const char* base = static_cast<const char*>(cache);
  Part<KIND> p = {};
  if constexpr (KIND == kRows16) {
    p.w = *reinterpret_cast<const u4_t*>(base + (off + e8 * 8) * 2);
  } else if constexpr (KIND == kRowsMx4) {
    p.w[0] = *reinterpret_cast<const uint32_t*>(base + off + e8 * 4);
    p.scale = scales[scale_off + (e8 >> 2)];
  } else {
    const u2_t w = *reinterpret_cast<const u2_t*>(base + off + e8 * 8);
    p.w[0] = w[0];
    p.w[1] = w[1];
  }
  return p;
}
template <int KIND, bool BF16>
__device__ __forceinline__ u4_t values_of(const Part<KIND>& p, float scale) {
  float x[8];
  if constexpr (KIND == kRows16) {
    return p.w;
  } else if constexpr (KIND == kRowsMx4) {
    const float by = __uint_as_float(p.scale << 23);
    const uint32_t w = p.w[0];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f2_t y = j == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, by, 0)
                     : j == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, by, 1)
                     : j == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, by, 2)
                              : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, by, 3);
      x[2 * j] = y.x;
      x[2 * j + 1] = y.y;
    }
    return pack8<BF16>(x);
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f2_t lo, hi;
      if constexpr (KIND == kRowsE4M3) {
        lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)p.w[j], false);
        hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)p.w[j], true);
      } else {
        lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)p.w[j], false);
        hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)p.w[j], true);
      }
      x[4 * j] = lo.x * scale;
      x[4 * j + 1] = lo.y * scale;
      x[4 * j + 2] = hi.x * scale;
      x[4 * j + 3] = hi.y * scale;
    }
    return pack8<BF16>(x);
  }
}

template <int KIND, bool BF16>
__global__ __launch_bounds__(256) void pad_read_kernel(const RowArgs a) {
  RowPart p;
  if (!row_part(a, p)) return;
  u4_t k = (u4_t)0u, v = (u4_t)0u;
  uint32_t page, at;
  if (place_of(a, slot_of(a, p.token), page, at)) {
    const uint64_t koff = offset_of(a.c.k_stride, page, at, p.h);
    const uint64_t voff = a.same ? koff : offset_of(a.c.v_stride, page, at, p.h);
    uint64_t ksoff = 0, vsoff = 0;
    if constexpr (KIND == kRowsMx4) {
      ksoff = offset_of(a.c.ks_stride, page, at, p.h);
      vsoff = a.same ? ksoff : offset_of(a.c.vs_stride, page, at, p.h);
    }
    const Part<KIND> kp = load_part<KIND>(a.c.k, a.c.k_scales, koff, ksoff, p.e8);
    const Part<KIND> vp = load_part<KIND>(a.c.v, a.c.v_scales, voff, vsoff, p.e8);
    k = values_of<KIND, BF16>(kp, a.c.k_scale);
    v = values_of<KIND, BF16>(vp, a.c.v_scale);
  }
  _Float16* kd = static_cast<_Float16*>(a.r.k) + (int64_t)p.token * a.r.k_stride[0] + (int64_t)p.h * a.r.k_stride[1];
  _Float16* vd = static_cast<_Float16*>(a.r.v) + (int64_t)p.token * a.r.v_stride[0] + (int64_t)p.h * a.r.v_stride[1];
  __builtin_nontemporal_store(k, reinterpret_cast<u4_t*>(kd + p.e8 * 8));
  __builtin_nontemporal_store(v, reinterpret_cast<u4_t*>(vd + p.e8 * 8));
}

// ---------------------------------------------------------------------------
// weights[slot] += sum over the group's rows of 2^(score - lse): the second
// half of a kKvWeights decode.  A workgroup walks tokens of one (sequence, kv
// head) unit; each weight is updated by one thread, so the sums have one order.
// ---------------------------------------------------------------------------
struct AccumulateArgs {
  const float* logits;
  const float* lse;
  const int32_t* bt;
  const int32_t* sl;
  float* weights;
  int64_t slog, sbb, sbp, ssl, swp, sws, swh, num_pages;
  int gqa, hkv, ps, ps_shift, max_pages;
};

// Round trips bound it: the first page id is loaded before the length is known
// (the table reaches as far as any length), and up to 4096 workgroups share the
// tokens (with four times as many, a stretch of 256 tokens each, 14.4 against 10.9 us
// at 48 x [1, 6000] of 32/8 heads).  Scores wait for the length: read up to the
// table's width they took longer than the wait.
__global__ __launch_bounds__(256) void pad_accumulate_kernel(const AccumulateArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const uint32_t cap = (uint32_t)a.max_pages * (uint32_t)a.ps;
  const int64_t row0 = ((int64_t)b * a.hkv + h) * a.gqa;
  const float* lse = a.lse + row0;
  float* wh = a.weights + (int64_t)h * a.swh;
  auto page_at = [&](uint32_t t) { return a.ps_shift >= 0 ? t >> a.ps_shift : t / (uint32_t)a.ps; };
  uint32_t t = blockIdx.x * 256 + threadIdx.x;
  int id = a.bt[b * a.sbb + (int64_t)page_at(min(t, cap - 1)) * a.sbp];
  const uint32_t L = min((uint32_t)max(a.sl[(int64_t)b * a.ssl], 0), cap);
  while (t < L) {
    const float* x = a.logits + row0 * a.slog + (int64_t)(t >> 2) * a.gqa * 4 + (t & 3);
    float* w = wh + clamp_page(id, a.num_pages) * a.swp + (int64_t)(t - page_at(t) * (uint32_t)a.ps) * a.sws;
    const float old = *w;
    float sum = 0.f;
#pragma unroll 4
    for (int r = 0; r < a.gqa; ++r) sum += exp2_fast(x[4 * r] - lse[r]);
    if (id >= 0 && id < a.num_pages) *w = old + sum;  // (not to page 0 for an id that is none)
    t += gridDim.x * 256;
    if (t < L) id = a.bt[b * a.sbb + (int64_t)page_at(t) * a.sbp];
  }
}

hipError_t launch_accumulate(const Phase1Args& p, float* weights, const int64_t* w_stride, hipStream_t st) {
  AccumulateArgs a = {};
  a.logits = p.logits;
  a.lse = p.lse;
  a.bt = p.bt;
  a.sl = p.sl;
  a.weights = weights;
  a.slog = p.slog;
  a.sbb = p.sbb;
  a.sbp = p.sbp;
  a.ssl = p.ssl;
  a.swp = w_stride[0];
  a.sws = w_stride[1];
  a.swh = w_stride[2];
  a.num_pages = p.num_pages;
  a.gqa = p.gqa;
  a.hkv = p.hq / p.gqa;  // (a range launch's hkv counts head groups)
  a.ps = p.ps;
  a.ps_shift = p.ps_shift;
  a.max_pages = p.max_pages;
  const int64_t units = (int64_t)p.batch * a.hkv;
  const int64_t chunks = ((int64_t)p.max_pages * p.ps + 255) / 256;
  const int64_t most = 4096 / units > 1 ? 4096 / units : 1;
  hipLaunchKernelGGL(pad_accumulate_kernel, dim3((unsigned)(chunks < most ? chunks : most), a.hkv, p.batch), dim3(256),
                     0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Eviction.  Per (sequence, kv head): the keep-th largest key by radix selection
// (four digits of 8 bits of an order-preserving integer of the weight), ties by
// slot order, then the moves: the i-th kept slot at or above the new length goes
// to the i-th evicted slot below it.  Sources lie at or above the new length and
// targets below it, so no move can overwrite what another reads, and moves run
// in any order.
//
// A workgroup selects for one unit; round trips and barriers bound it, so every
// wave scans the 256 counts of a digit by itself (one barrier a digit), and keys
// stay in registers: they are read once, a round trip for the page ids and one
// for weights and positions.  64 x 2049 slots of 2 heads, one token to go: 11.3 us
// with the move (20.8 + 4.8 with keys read again in each of three passes; 512
// threads 12.6 for 12.2 of 1024).  16 x 5120 of 8 heads, 1024 to go: 16.9 us, and
// the moves 28.8 us (33.3 one at a time), 4.7 TB/s, what a copy reaches.
// ---------------------------------------------------------------------------
struct EvictArgs {
  pad_kv_cache c;
  pad_kv_evict_call e;
  int2* moves;     // [units][most] (source slot, target slot)
  int* num_moves;  // [units]: those left to the move kernel
  int64_t most;
  int ps_shift;
  int row_units;   // vector units of a K (or V) row
  int elem_bytes;  // bytes per element of the rows' strides
  int scale_bytes; // MX4 scale bytes of a row, else 0
  int wide;        // 1: units of 16 bytes, 0: of 8
};

// Moves that the selecting workgroup makes itself, without a second kernel.
constexpr int kOwnMoves = 128;
constexpr uint32_t kKeyNewest = 0xffffffffu;
constexpr uint32_t kKeyNan = 0xfffffffeu;

// Order-preserving integer of a weight (-0 counts as 0); 0 is below all.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return kKeyNan;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_page(const EvictArgs& a, int slot) {
  return a.ps_shift >= 0 ? slot >> a.ps_shift : (int)((uint32_t)slot / (uint32_t)a.c.page_size);
}

// Where a slot of sequence b lies.
struct Place {
  int64_t page, at;
  bool real;  // the table's id is a page (else page 0 is read, and nothing written)
};
__device__ __forceinline__ Place evict_place(const EvictArgs& a, int b, int slot) {
  const int page = evict_page(a, slot);
  Place p;
  const int id = a.e.block_table[(int64_t)b * a.e.bt_stride[0] + (int64_t)page * a.e.bt_stride[1]];
  p.page = clamp_page(id, a.c.num_pages);
  p.real = p.page == id;
  p.at = slot - (int64_t)page * a.c.page_size;
  return p;
}

// Moves first, first + step, ... of m by `threads` threads, 2 * row_units for
// a move: K's vector units, then V's (the first ones take the scales, weight and
// position along).
template <typename U>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int b, int h, const int2* list, int m, int block,
                                          int blocks, int tid, int threads) {
  const int tp = 2 * a.row_units;
  const int per = threads / tp;
  const int mine = tid / tp;
  if (mine >= per) return;
  const int task = tid - mine * tp;
  const bool is_v = task >= a.row_units;
  const int c = is_v ? task - a.row_units : task;
  const int64_t* st = is_v ? a.c.v_stride : a.c.k_stride;
  const int64_t* ss = is_v ? a.c.vs_stride : a.c.ks_stride;
  char* base = static_cast<char*>(is_v ? a.c.v : a.c.k) + (int64_t)h * st[2] * a.elem_bytes + c * sizeof(U);
  // Four moves at a time: a round trip for the list, the page ids and the rows each.
  constexpr int N = 4;
  const int step = blocks * per;
  for (int i0 = block * per + mine; i0 < m; i0 += N * step) {
    int2 mv[N];
    Place s[N], d[N];
    U row[N];
#pragma unroll
    for (int j = 0; j < N; ++j) mv[j] = list[min(i0 + j * step, m - 1)];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      s[j] = evict_place(a, b, mv[j].x);
      d[j] = evict_place(a, b, mv[j].y);
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      row[j] = *reinterpret_cast<const U*>(base + (s[j].page * st[0] + s[j].at * st[1]) * a.elem_bytes);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (i0 + j * step >= m) break;
      if (!s[j].real || !d[j].real) continue;
      *reinterpret_cast<U*>(base + (d[j].page * st[0] + d[j].at * st[1]) * a.elem_bytes) = row[j];
      if (c < a.scale_bytes) {
        uint8_t* sb = (is_v ? a.c.v_scales : a.c.k_scales) + (int64_t)h * ss[2] + c;
        sb[d[j].page * ss[0] + d[j].at * ss[1]] = sb[s[j].page * ss[0] + s[j].at * ss[1]];
      }
      if (c == 0) {
        const int64_t* ws = is_v ? a.c.p_stride : a.c.w_stride;  // 32-bit words either way
        uint32_t* w = (is_v ? reinterpret_cast<uint32_t*>(a.c.positions) : reinterpret_cast<uint32_t*>(a.c.weights)) +
                      (int64_t)h * ws[2];
        w[d[j].page * ws[0] + d[j].at * ws[1]] = w[s[j].page * ws[0] + s[j].at * ws[1]];
      }
    }
  }
}

// Adds one to hist[bin] for every lane with `in`: the lanes that share the first
// one's bin in one addition (weights of a digit fall into few bins).
__device__ __forceinline__ void count_bin(int* hist, int bin, bool in, int lane) {
  const uint64_t active = __builtin_amdgcn_ballot_w64(in);
  if (active == 0) return;
  const int lead = (int)__builtin_ctzll(active);
  const int common = __builtin_amdgcn_readlane(bin, lead);
  const uint64_t same = __builtin_amdgcn_ballot_w64(in && bin == common);
  if (lane == lead) atomicAdd(&hist[common], (int)__builtin_popcountll(same));
  if (in && bin != common) atomicAdd(&hist[bin], 1);
}

// NR: slots of a thread, whose keys are in registers; 0: any number, read again
// in every pass.
template <int NR, int THREADS>
__global__ __launch_bounds__(THREADS) void pad_evict_select_kernel(const EvictArgs a) {
  constexpr int WAVES = THREADS / 64;
  const int h = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = (int64_t)b * a.c.num_kv_heads + h;
  const int64_t cap = (int64_t)a.e.max_pages * a.c.page_size;
  const int L = (int)min((int64_t)max(a.e.seq_lens[(int64_t)b * a.e.sl_stride], 0), cap);
  const int n = min(max(a.e.keeps ? a.e.keeps[b] : a.e.keep, 0), L);
  if (tid == 0 && h == 0) a.e.new_lens[b] = n;
  if (n == L || n == 0) {
    if (tid == 0) a.num_moves[unit] = 0;
    return;
  }
  __shared__ int hist[4][256];
  __shared__ int2 sm[2][WAVES];
  __shared__ int2 own[kOwnMoves];
  for (int i = tid; i < 4 * 256; i += THREADS) hist[0][i] = 0;

  // A wave has consecutive slots, 64 at a time.
  const int steps = (L + THREADS - 1) / THREADS;
  const int first = wave * steps * 64 + lane;
  const char* wbase = reinterpret_cast<const char*>(a.c.weights + (int64_t)h * a.c.w_stride[2]);
  const char* pbase = reinterpret_cast<const char*>(a.c.positions + (int64_t)h * a.c.p_stride[2]);
  auto weight_of = [&](const Place& p) {
    return *reinterpret_cast<const float*>(wbase + (p.page * a.c.w_stride[0] + p.at * a.c.w_stride[1]) * 4);
  };
  auto position_of = [&](const Place& p) {
    return *reinterpret_cast<const int32_t*>(pbase + (p.page * a.c.p_stride[0] + p.at * a.c.p_stride[1]) * 4);
  };
  constexpr int N = NR > 0 ? NR : 1;
  uint32_t keys[N];
  int64_t border;
  {
    int newest = INT32_MIN;
    int positions[N];
    if constexpr (NR > 0) {
      // Slots past the end read the last one's words (and get key 0 below): no
      // branch holds a load back.
      constexpr int BATCH = NR < 8 ? NR : 8;
#pragma unroll
      for (int i0 = 0; i0 < NR; i0 += BATCH) {
        if (i0 < steps) {
          Place p[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) p[i] = evict_place(a, b, min(first + (i0 + i) * 64, L - 1));
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            positions[i0 + i] = position_of(p[i]);
            keys[i0 + i] = __float_as_uint(weight_of(p[i]));
          }
#pragma unroll
          for (int i = 0; i < BATCH; ++i) newest = max(newest, positions[i0 + i]);
        }
      }
    } else {
      for (int i = 0; i < steps; ++i) {
        const int slot = first + i * 64;
        if (slot < L) newest = max(newest, position_of(evict_place(a, b, slot)));
      }
    }
    newest = wave_max_i32(newest);
    if (lane == 0) sm[0][wave].x = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) newest = max(newest, sm[0][w].x);
    border = (int64_t)newest - a.e.recent;
    if constexpr (NR > 0) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const bool in = i < steps && first + i * 64 < L;
        const uint32_t k = (int64_t)positions[i] > border ? kKeyNewest : weight_key(__uint_as_float(keys[i]));
        keys[i] = in ? k : 0u;
      }
    }
  }
  auto key_at = [&](int i) -> uint32_t {
    if constexpr (NR > 0) {
      return keys[i];
    } else {
      const int slot = first + i * 64;
      if (slot >= L) return 0u;
      const Place p = evict_place(a, b, slot);
      const int32_t at = position_of(p);
      const float w = weight_of(p);
      return (int64_t)at > border ? kKeyNewest : weight_key(w);
    }
  };
  // f(i, key) for each of the thread's slots; whole waves call it.
  auto each = [&](auto f) {
    if constexpr (NR > 0) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
        if (i < steps) f(i, keys[i]);
    } else {
      for (int i = 0; i < steps; ++i) f(i, key_at(i));
    }
  };

  // The n-th largest key.
  uint32_t prefix = 0;
  int left = n;  // of the keys with this prefix, how many from the top
  int equal = 0;  // keys with this prefix
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    each([&](int, uint32_t k) {
      const bool in = k != 0 && (pass == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
      count_bin(hist[pass], (int)((k >> shift) & 255u), in, lane);
    });
    __syncthreads();
    // Lane l has bins 255 - 4l and the three below, from the top.
    const i4_t c = *reinterpret_cast<const i4_t*>(&hist[pass][252 - 4 * lane]);
    const int sum = c[0] + c[1] + c[2] + c[3];
    int above = wave_incl_scan_i32(sum, lane) - sum;
    int bin = -1;
    int above_bin = 0, in_bin = 0;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      if (above < left && left <= above + c[j]) {
        bin = 252 - 4 * lane + j;
        above_bin = above;
        in_bin = c[j];
      }
      above += c[j];
    }
    const int who = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(bin >= 0));  // the keys counted are at least `left`
    prefix |= (uint32_t)__builtin_amdgcn_readlane(bin, who) << shift;
    left -= __builtin_amdgcn_readlane(above_bin, who);
    equal = __builtin_amdgcn_readlane(in_bin, who);
  }

  // `left` of the keys equal to it are kept, the lowest slots first: where not
  // all are, their order over the waves counts.
  const uint64_t below = (1ull << lane) - 1;
  int tie0 = 0;
  if (equal != left) {
    int ties = 0;
    each([&](int, uint32_t k) { ties += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(k == prefix)); });
    if (lane == 0) sm[1][wave] = make_int2(ties, 0);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) tie0 += w < wave ? sm[1][w].x : 0;
  }
  int tie = tie0, movers = 0, holes = 0;
  auto classify = [&](int i, uint32_t k, uint64_t& moves, uint64_t& opens) {
    const int slot = first + i * 64;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(k == prefix);
    const bool kept = k > prefix || (k == prefix && tie + (int)__builtin_popcountll(eq & below) < left);
    tie += (int)__builtin_popcountll(eq);
    moves = __builtin_amdgcn_ballot_w64(kept && slot >= n);
    opens = __builtin_amdgcn_ballot_w64(!kept && slot < n);
  };
  each([&](int i, uint32_t k) {
    uint64_t mv, op;
    classify(i, k, mv, op);
    movers += (int)__builtin_popcountll(mv);
    holes += (int)__builtin_popcountll(op);
  });
  // (Places in turn: every wave has passed a barrier since it read this one.)
  if (lane == 0) sm[0][wave] = make_int2(movers, holes);
  __syncthreads();
  int mover = 0, hole = 0, num_moves = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int2 x = sm[0][w];
    mover += w < wave ? x.x : 0;
    hole += w < wave ? x.y : 0;
    num_moves += x.x;
  }
  num_moves = (int)min((int64_t)num_moves, a.most);
  const bool mine = num_moves <= kOwnMoves;
  int2* list = mine ? own : a.moves + unit * a.most;
  tie = tie0;
  each([&](int i, uint32_t k) {
    uint64_t mv, op;
    classify(i, k, mv, op);
    const int slot = first + i * 64;
    const int m = mover + (int)__builtin_popcountll(mv & below), o = hole + (int)__builtin_popcountll(op & below);
    if ((mv >> lane & 1) && m < num_moves) list[m].x = slot;
    if ((op >> lane & 1) && o < num_moves) list[o].y = slot;
    mover += (int)__builtin_popcountll(mv);
    hole += (int)__builtin_popcountll(op);
  });
  if (tid == 0) a.num_moves[unit] = mine ? 0 : num_moves;
  if (!mine) return;
  __syncthreads();
  if (a.wide)
    move_rows<u4_t>(a, b, h, own, num_moves, 0, 1, tid, THREADS);
  else
    move_rows<u2_t>(a, b, h, own, num_moves, 0, 1, tid, THREADS);
}

template <typename U>
__global__ __launch_bounds__(256) void pad_evict_move_kernel(const EvictArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t unit = (int64_t)b * a.c.num_kv_heads + h;
  move_rows<U>(a, b, h, a.moves + unit * a.most, a.num_moves[unit], blockIdx.x, gridDim.x, threadIdx.x, 256);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
static int shift_of(int ps) {
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == ps) return sh;
  return -1;
}

static int row_kind(int kv_format) {
  switch (kv_format) {
    case PAD_KV_FP16:
    case PAD_KV_BF16: return kRows16;
    case PAD_KV_FP8_E4M3FN: return kRowsE4M3;
    case PAD_KV_FP8_E5M2: return kRowsE5M2;
    case PAD_KV_MX4: return kRowsMx4;
    default: return -1;
  }
}

// Bytes of a row in the cache, and of a stride's element.
static int row_bytes(const pad_kv_cache* c) {
  const int kind = row_kind(c->kv_format);
  return kind == kRows16 ? 2 * c->head_dim : kind == kRowsMx4 ? c->head_dim / 2 : c->head_dim;
}
static int stride_bytes(const pad_kv_cache* c) { return row_kind(c->kv_format) == kRows16 ? 2 : 1; }

// Rows' alignment: the largest power of two (up to 16) that every row starts at.
static int row_alignment(const pad_kv_cache* c) {
  uint64_t x = (uint64_t)(uintptr_t)c->k | (uint64_t)(uintptr_t)c->v | 16u;
  for (int i = 0; i < 3; ++i)
    x |= (uint64_t)c->k_stride[i] * stride_bytes(c) | (uint64_t)c->v_stride[i] * stride_bytes(c);
  return (int)(x & (~x + 1));
}

static int check_cache(const pad_kv_cache* c) {
  if (!c || !c->k || !c->v) return PAD_ERR_NULL_POINTER;
  const int kind = row_kind(c->kv_format);
  if (kind < 0) return PAD_ERR_KV_FORMAT;
  if (c->page_size <= 0 || c->num_kv_heads <= 0 || c->num_kv_heads > 65535 || c->num_pages <= 0 ||
      c->num_pages > INT32_MAX)
    return PAD_ERR_INVALID_SHAPE;
  const int d = c->head_dim;
  if (d != 64 && d != 128 && d != 256 && (kind != kRows16 || (d != 32 && d != 96))) return PAD_ERR_UNSUPPORTED_HEAD_DIM;
  if (kind == kRowsMx4 && (!c->k_scales || !c->v_scales)) return PAD_ERR_NULL_POINTER;
  if ((kind == kRowsE4M3 || kind == kRowsE5M2) &&
      (!(c->k_scale > 0.f) || !(c->v_scale > 0.f) || c->k_scale > 1e30f || c->v_scale > 1e30f))
    return PAD_ERR_KV_FORMAT;
  // Offsets are sums of 32 by 32 bit products.
  const int64_t* strides[] = {c->k_stride, c->v_stride, c->ks_stride, c->vs_stride, c->w_stride, c->p_stride};
  const bool used[] = {true, true, kind == kRowsMx4, kind == kRowsMx4, c->weights != nullptr, c->positions != nullptr};
  for (int j = 0; j < 6; ++j)
    for (int i = 0; used[j] && i < 3; ++i)
      if (strides[j][i] < 0 || strides[j][i] > UINT32_MAX) return PAD_ERR_STRIDE;
  const int need = kind == kRows16 ? 16 : 8;
  return row_alignment(c) < need ? PAD_ERR_ALIGNMENT : PAD_OK;
}

static int check_rows(const pad_kv_cache* c, const pad_kv_rows* r) {
  const int st = check_cache(c);
  if (st != PAD_OK) return st;
  if (!r) return PAD_ERR_NULL_POINTER;
  if (r->tokens < 0) return PAD_ERR_INVALID_SHAPE;
  if (r->tokens == 0) return PAD_OK;
  if (!r->k || !r->v || !r->slots) return PAD_ERR_NULL_POINTER;
  if (r->tokens > INT32_MAX / c->num_kv_heads) return PAD_ERR_INVALID_SHAPE;  // rows are counted in 32 bits
  if ((((uintptr_t)r->k | (uintptr_t)r->v) & 15u) != 0 ||
      ((r->k_stride[0] | r->k_stride[1] | r->v_stride[0] | r->v_stride[1]) & 7) != 0)
    return PAD_ERR_ALIGNMENT;
  if (row_kind(c->kv_format) == kRows16 && (c->kv_format == PAD_KV_BF16) != (r->bf16 != 0)) return PAD_ERR_KV_FORMAT;
  return PAD_OK;
}

template <template <int, bool> class K>
static void launch_rows(const RowArgs& a, hipStream_t st) {
  const uint32_t per = 256u / (uint32_t)a.row8;
  const dim3 grid((a.rows + per - 1) / per);
  const bool bf16 = a.r.bf16 != 0;
  switch (row_kind(a.c.kv_format)) {
    case kRows16: K<kRows16, false>::launch(a, grid, st); break;  // moved as bits
    case kRowsE4M3: bf16 ? K<kRowsE4M3, true>::launch(a, grid, st) : K<kRowsE4M3, false>::launch(a, grid, st); break;
    case kRowsE5M2: bf16 ? K<kRowsE5M2, true>::launch(a, grid, st) : K<kRowsE5M2, false>::launch(a, grid, st); break;
    default: bf16 ? K<kRowsMx4, true>::launch(a, grid, st) : K<kRowsMx4, false>::launch(a, grid, st); break;
  }
}

template <int KIND, bool BF16>
struct Append {
  static void launch(const RowArgs& a, dim3 grid, hipStream_t st) {
    hipLaunchKernelGGL((pad_append_kernel<KIND, BF16>), grid, dim3(256), 0, st, a);
  }
};
template <int KIND, bool BF16>
struct Read {
  static void launch(const RowArgs& a, dim3 grid, hipStream_t st) {
    hipLaunchKernelGGL((pad_read_kernel<KIND, BF16>), grid, dim3(256), 0, st, a);
  }
};

static RowArgs row_args(const pad_kv_cache* c, const pad_kv_rows* r) {
  RowArgs a = {};
  a.c = *c;
  a.r = *r;
  a.row8 = c->head_dim / 8;
  a.rows = (uint32_t)(r->tokens * c->num_kv_heads);
  a.row8_shift = shift_of(a.row8);
  a.ps_shift = shift_of(c->page_size);
  a.head_shift = shift_of(c->num_kv_heads);
  a.same = 1;
  for (int i = 0; i < 3; ++i)
    if (c->k_stride[i] != c->v_stride[i] || (row_kind(c->kv_format) == kRowsMx4 && c->ks_stride[i] != c->vs_stride[i]))
      a.same = 0;
  return a;
}

// Slots of one sequence: the selection counts them, in steps of a workgroup, in
// 32 bits.
constexpr int64_t kMostSlots = INT32_MAX - 2 * 1024;

// Workspace of an eviction: 256 bytes of slack, a count per unit, the move lists.  A unit of
// capacity C moves at most C / 2 rows (sources at or above the new length,
// targets below it).
static int64_t most_moves(int64_t max_pages, int64_t page_size) { return max_pages * page_size / 2; }
static size_t evict_counts_bytes(int64_t units) { return ((size_t)units * sizeof(int) + 255) & ~(size_t)255; }
static size_t evict_bytes(int64_t units, int64_t max_pages, int64_t page_size) {
  return 256 + evict_counts_bytes(units) + (size_t)(units * most_moves(max_pages, page_size)) * sizeof(int2);
}

static void launch_select(const EvictArgs& a, hipStream_t st) {
  const dim3 grid(a.c.num_kv_heads, a.e.batch);
  const int64_t cap = (int64_t)a.e.max_pages * a.c.page_size;
  if (cap <= 2 * 1024)
    hipLaunchKernelGGL((pad_evict_select_kernel<2, 1024>), grid, dim3(1024), 0, st, a);
  else if (cap <= 4 * 1024)
    hipLaunchKernelGGL((pad_evict_select_kernel<4, 1024>), grid, dim3(1024), 0, st, a);
  else if (cap <= 8 * 1024)
    hipLaunchKernelGGL((pad_evict_select_kernel<8, 1024>), grid, dim3(1024), 0, st, a);
  else if (cap <= 16 * 1024)
    hipLaunchKernelGGL((pad_evict_select_kernel<16, 1024>), grid, dim3(1024), 0, st, a);
  else if (cap <= 32 * 1024)
    hipLaunchKernelGGL((pad_evict_select_kernel<32, 1024>), grid, dim3(1024), 0, st, a);
  else
    hipLaunchKernelGGL((pad_evict_select_kernel<0, 1024>), grid, dim3(1024), 0, st, a);
}

}  // namespace pad

using namespace pad;

extern "C" {

int pad_kv_append(const pad_kv_cache* cache, const pad_kv_rows* rows, const float* token_weights,
                  const int32_t* token_positions, void* stream) {
  const int st = check_rows(cache, rows);
  if (st != PAD_OK || rows->tokens == 0) return st;
  if ((cache->positions && !token_positions) || (token_weights && !cache->weights)) return PAD_ERR_NULL_POINTER;
  RowArgs a = row_args(cache, rows);
  a.token_weights = token_weights;
  a.token_positions = token_positions;
  launch_rows<Append>(a, reinterpret_cast<hipStream_t>(stream));
  return hipGetLastError() == hipSuccess ? PAD_OK : PAD_ERR_LAUNCH;
}

int pad_kv_read(const pad_kv_cache* cache, const pad_kv_rows* rows, void* stream) {
  const int st = check_rows(cache, rows);
  if (st != PAD_OK || rows->tokens == 0) return st;
  launch_rows<Read>(row_args(cache, rows), reinterpret_cast<hipStream_t>(stream));
  return hipGetLastError() == hipSuccess ? PAD_OK : PAD_ERR_LAUNCH;
}

int pad_kv_evict_workspace_bytes(int64_t batch, int64_t num_kv_heads, int64_t max_pages, int64_t page_size,
                                 size_t* bytes) {
  if (!bytes) return PAD_ERR_NULL_POINTER;
  if (batch < 0 || num_kv_heads <= 0 || max_pages < 0 || page_size <= 0 || max_pages > kMostSlots / page_size)
    return PAD_ERR_INVALID_SHAPE;
  *bytes = evict_bytes(batch * num_kv_heads, max_pages, page_size);
  return PAD_OK;
}

int pad_kv_evict(const pad_kv_cache* cache, const pad_kv_evict_call* call, void* stream) {
  int st = check_cache(cache);
  if (st != PAD_OK) return st;
  if (!call || !cache->weights || !cache->positions) return PAD_ERR_NULL_POINTER;
  if (call->batch < 0 || call->batch > 65535 || call->max_pages < 0 || call->recent < 0 ||
      (!call->keeps && call->keep < 0) || call->max_pages > kMostSlots / cache->page_size)
    return PAD_ERR_INVALID_SHAPE;
  if (call->batch == 0) return PAD_OK;
  if (!call->seq_lens || !call->new_lens || (!call->block_table && call->max_pages > 0)) return PAD_ERR_NULL_POINTER;
  const int64_t units = (int64_t)call->batch * cache->num_kv_heads;
  if (!call->workspace || call->workspace_bytes < evict_bytes(units, call->max_pages, cache->page_size))
    return PAD_ERR_WORKSPACE;
  EvictArgs a = {};
  a.c = *cache;
  a.e = *call;
  char* base = reinterpret_cast<char*>(((uintptr_t)call->workspace + 255u) & ~(uintptr_t)255u);
  a.num_moves = reinterpret_cast<int*>(base);
  a.moves = reinterpret_cast<int2*>(base + evict_counts_bytes(units));
  a.most = most_moves(call->max_pages, cache->page_size);
  a.ps_shift = shift_of(cache->page_size);
  a.elem_bytes = stride_bytes(cache);
  a.scale_bytes = row_kind(cache->kv_format) == kRowsMx4 ? cache->head_dim / 32 : 0;
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  a.wide = row_alignment(cache) == 16 ? 1 : 0;
  a.row_units = row_bytes(cache) / (a.wide ? 16 : 8);
  launch_select(a, hs);
  if (hipGetLastError() != hipSuccess) return PAD_ERR_LAUNCH;
  // No unit moves more rows than it loses, or than it keeps.
  const int64_t cap = (int64_t)call->max_pages * cache->page_size;
  const int64_t bound = call->keeps || call->keep >= cap ? a.most
                        : cap - call->keep < call->keep  ? cap - call->keep
                                                         : call->keep;
  if (bound <= kOwnMoves) return PAD_OK;
  const int per = 256 / (2 * a.row_units);
  const int64_t chunks = (bound + 4 * per - 1) / (4 * per);
  const int64_t limit = 8192 / units > 1 ? 8192 / units : 1;
  const dim3 grid((unsigned)(chunks < limit ? chunks : limit), cache->num_kv_heads, call->batch);
  if (a.wide)
    hipLaunchKernelGGL((pad_evict_move_kernel<u4_t>), grid, dim3(256), 0, hs, a);
  else
    hipLaunchKernelGGL((pad_evict_move_kernel<u2_t>), grid, dim3(256), 0, hs, a);
  return hipGetLastError() == hipSuccess ? PAD_OK : PAD_ERR_LAUNCH;
}

}  // extern "C"
