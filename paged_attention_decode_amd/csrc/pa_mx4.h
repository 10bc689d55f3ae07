// pa_mx4.h - wave loop of the decode over MX4 caches (OCP Microscaling MXFP4:
// e2m1 codes, two a byte with the even element in the low nibble, and one
// power-of-two scale byte per 32 elements of head_dim).
//
// A row is D/2 bytes of codes and D/32 scale bytes, a quarter of fp16's, so a
// wave works on 32 tokens at a time (two tiles of 16).  Lane (g, r16) holds D/4
// elements of token 16u + r16 in both K and V:
//  * S^T = K . Q^T needs no staging: the lane's elements, widened eight at a
//    time, are the A operand of a 16x16x32 step as loaded.  The contraction
//    runs over head_dim in the order the lanes hold it, and Q^T is loaded in
//    the same order.
//  * O^T = V^T . P^T contracts over tokens, so V is transposed on the way: the
//    widened rows go through an LDS tile and come back with gfx950's
//    transposing LDS reads, four tokens of one dim a lane.  A step covers both
//    tiles: contraction slot 8g + 4u + i is token 16u + 4g + i, which is how
//    the lanes hold P^T.
// v_cvt_scalef32_pk_{f16,bf16}_fp4 multiplies by the block's scale while it
// widens, exactly for every scale byte that bfloat16 (or, with fp16 q, fp16)
// can hold the products of; byte 255 gives NaN.
#ifndef PA_MX4_H_
#define PA_MX4_H_

#include <type_traits>

#include "pa_device.h"

namespace pad {

// Waves per SIMD that the per-unit kernels are compiled for (registers per lane):
// head_dim 128 does not fit the 168 of three.
constexpr int mx4_waves_per_simd(int d) { return d <= 64 ? 3 : d <= 128 ? 2 : 1; }

// One 16x16x32 step on 16-bit operands (8 elements of the contraction a lane).
template <int KVF>
__device__ __forceinline__ f4_t mfma16x32(h8_t a, h8_t b, f4_t c) {
  if constexpr (q_is_bf16<KVF>()) {
    typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0,
                                                   0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
}

__device__ __forceinline__ float mx4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes (one dword, element i in nibble i) times a scale.
template <int KVF>
__device__ __forceinline__ h8_t mx4x8(uint32_t w, float scale) {
  u4_t r;
  if constexpr (q_is_bf16<KVF>()) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
  }
  return __builtin_bit_cast(h8_t, r);
}

// Two floats rounded to q's type, in a dword.
template <int KVF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (q_is_bf16<KVF>()) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2_t{x, y}, b2_t));
  } else {
    return __builtin_bit_cast(uint32_t, h2_t{(_Float16)x, (_Float16)y});
  }
}

// A row is NC chunks of up to 32 elements a lane (one scale each), at elements
// c * 128 + g * kMx4Lane: a load instruction covers whole rows.
template <int D>
constexpr int mx4_chunks() { return D > 128 ? D / 128 : 1; }
template <int D>
constexpr int mx4_lane_elems() { return D > 128 ? 32 : D / 4; }

// First element of the lane's dword s (eight elements), and its chunk.
template <int D>
__device__ __forceinline__ int mx4_elem(int g, int s) {
  constexpr int DW = mx4_lane_elems<D>() / 8;
  return (s / DW) * 128 + g * mx4_lane_elems<D>() + (s % DW) * 8;
}

template <int D>
struct Mx4Tile {
  static constexpr int DW = D / 32;
  static constexpr int NC = mx4_chunks<D>();
  HVec<DW> k[2], v[2];
  uint32_t ks[2][NC], vs[2][NC];
};

// Transposing LDS read: lane 4r + c of a 16-lane group names four consecutive
// 16-bit elements (row r of four, columns 4c .. 4c+3); lane l gets column l of
// the four rows.
__device__ __forceinline__ h4_t lds_read_transposed(const char* p) {
  typedef short s4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4_t lds_s4_t;
  return __builtin_bit_cast(h4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)p));
}

// One wave's part of an item: tokens [t_begin, t_end) (t_begin on a page border,
// nblk blocks of 16) of kv head kvh, of which the wave takes the pairs of blocks
// wave, wave + nw, ...; its state goes to place `slot` of sm_ml and sm_o.
// MODE: kModeUniform (a 16-token block lies in one page, its rows next to each
// other) or kModeGeneric (each lane finds its own tokens' pages).  Strides are
// below 2^32 bytes, the scales' slot strides below 2^26 in uniform mode (the
// launcher sees to both).
template <int D, int MODE, int KVF>
__device__ __forceinline__ void wave_loop_mx4(const Phase1Args& a, const int32_t* bt_row, int64_t ids_stride, int b,
                                              int kvh, int t_begin, int t_end, int nblk, int wave, int nw, int slot,
                                              int lane, float2* sm_ml, float* sm_o, char* stage) {
  using Tile = Mx4Tile<D>;
  constexpr int DW = Tile::DW;
  constexpr int NC = Tile::NC;
  constexpr int CW = DW / NC;  // dwords per chunk
  constexpr int DT = D / 16;
  constexpr int ROW = k_stage_row_bytes<D>();
  const int g = lane >> 4;
  const int r16 = lane & 15;
  const bool row_ok = r16 < a.gqa;

  h8_t qv[DW];
  auto load_q = [&]() {
    const _Float16* qrow = a.q + (int64_t)b * a.sqb + (int64_t)(kvh * a.gqa + (row_ok ? r16 : 0)) * a.sqh;
#pragma unroll
    for (int s = 0; s < DW; ++s) {
      const h8_t x = *reinterpret_cast<const h8_t*>(qrow + mx4_elem<D>(g, s));
      qv[s] = row_ok ? x : (h8_t)0;
    }
  };

  float m_run = kNegInf;
  f4_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = (f4_t)0.f;
  // Row sums of P from one more matrix step with an operand of ones; where the
  // caller gets the weights, which are unrounded, a lane's own sum.
  f4_t o_l = (f4_t)0.f;
  const std::conditional_t<kv_weights<KVF>(), Logits, NoLogits> logits(a, b, kvh, r16);

  const char* k_head = reinterpret_cast<const char*>(a.k) + (int64_t)kvh * a.skh;
  const char* v_head = reinterpret_cast<const char*>(a.v) + (int64_t)kvh * a.svh;
  const char* ks_head = reinterpret_cast<const char*>(a.ks) + (int64_t)kvh * a.sksh;
  const char* vs_head = reinterpret_cast<const char*>(a.vs) + (int64_t)kvh * a.svsh;
  const int elem0 = mx4_elem<D>(g, 0);
  const uint32_t page_limit = (uint32_t)min(a.num_pages, (int64_t)0x7fffffff);
  auto clamp_id = [&](int id) -> uint32_t { return (uint32_t)id < page_limit ? (uint32_t)id : 0u; };

  // Where the wave's next pair lies: page (from the item's first) and slot of its
  // blocks (uniform mode, scalars) or of the lane's tokens; pairs are nw apart.
  // Page ids are fetched a pair ahead, before its predecessor's rows, so that
  // waiting for them waits for no rows.  Past the item's end the last page's id
  // is read again and the tokens are masked.
  const int lane_row = MODE == kModeUniform ? 0 : r16;
  const int p_first = page_of(a, t_begin);
  const int p_last = t_end > t_begin ? page_of(a, t_end - 1) : p_first;
  const int step_pages = page_of(a, nw * 32);
  const int step_slots = nw * 32 - step_pages * a.ps;
  int cur_page[2], cur_slot[2], pid[2], pslot[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = wave * 32 + 16 * u + lane_row;
    cur_page[u] = page_of(a, t);
    cur_slot[u] = t - cur_page[u] * a.ps;
  }
  auto fetch_ids = [&]() {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t col = (int64_t)min(p_first + cur_page[u], p_last) * ids_stride;
      if constexpr (MODE == kModeUniform)
        pid[u] = load_uniform_i32(bt_row + col);
      else
        pid[u] = bt_row[col];
      pslot[u] = cur_slot[u];
      cur_page[u] += step_pages;
      cur_slot[u] += step_slots;
      if (cur_slot[u] >= a.ps) {
        cur_slot[u] -= a.ps;
        ++cur_page[u];
      }
    }
  };

  // Rows and scales of one block: from a scalar base with 32-bit lane offsets
  // (uniform mode), or from each lane's own address.
  uint32_t koff = (uint32_t)(elem0 / 2), voff = koff, ksoff = (uint32_t)(elem0 / 32), vsoff = ksoff;
  if constexpr (MODE == kModeUniform) {
    koff += (uint32_t)r16 * (uint32_t)a.sks;
    voff += (uint32_t)r16 * (uint32_t)a.svs;
    ksoff += (uint32_t)r16 * (uint32_t)a.skss;
    vsoff += (uint32_t)r16 * (uint32_t)a.svss;
  }
  constexpr int kStream = 2;  // NT
  auto load_codes = [&](HVec<DW>& x, const char* base, uint32_t off) {
    if constexpr (MODE == kModeUniform) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base, 0xffffffffu);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (CW == 4) {
          const u4_t w = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off + c * 64, 0, kStream));
#pragma unroll
          for (int j = 0; j < 4; ++j) x.w[c * 4 + j] = w[j];
        } else {
          const u2_t w = __builtin_bit_cast(u2_t, __builtin_amdgcn_raw_buffer_load_b64(r, off + c * 64, 0, kStream));
#pragma unroll
          for (int j = 0; j < 2; ++j) x.w[c * 2 + j] = w[j];
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const HVec<CW> w = load_hvec<CW>(reinterpret_cast<const _Float16*>(base + off + c * 64));
#pragma unroll
        for (int j = 0; j < CW; ++j) x.w[c * CW + j] = w.w[j];
      }
    }
  };
  auto load_scales = [&](uint32_t (&x)[NC], const char* base, uint32_t off) {
    if constexpr (MODE == kModeUniform) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base, 0xffffffffu);
#pragma unroll
      for (int c = 0; c < NC; ++c) x[c] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, off + c * 4, 0, 0);
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) x[c] = (uint8_t)base[off + c * 4];
    }
  };
  auto at = [](const char* head, uint32_t page, int64_t page_bytes, uint32_t row, int64_t row_bytes) {
    return head + (uint64_t)page * (uint32_t)page_bytes + (uint64_t)row * (uint32_t)row_bytes;
  };
  auto load = [&](Tile& t) {
    uint32_t page[2], row[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      page[u] = clamp_id(pid[u]);
      row[u] = (uint32_t)pslot[u];
    }
    fetch_ids();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      load_codes(t.k[u], at(k_head, page[u], a.skp, row[u], a.sks), koff);
      load_scales(t.ks[u], at(ks_head, page[u], a.sksp, row[u], a.skss), ksoff);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      load_codes(t.v[u], at(v_head, page[u], a.svp, row[u], a.svs), voff);
      load_scales(t.vs[u], at(vs_head, page[u], a.svsp, row[u], a.svss), vsoff);
    }
  };

  auto compute = [&](Tile& t, int jp) {
    const int t0 = t_begin + jp * 32;
    float x[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f4_t sacc = (f4_t)0.f;
#pragma unroll
      for (int s = 0; s < DW; ++s)
        sacc = mfma16x32<KVF>(mx4x8<KVF>(t.k[u].w[s], mx4_scale(t.ks[u][s / CW])), qv[s], sacc);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] = sacc[i] * a.scale_log2;
    }
    if (t0 + 32 > t_end) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u][i] = t0 + 16 * u + 4 * g + i < t_end ? x[u][i] : kNegInf;
        if (t0 + 16 * u + r16 >= t_end) {  // stale slots may hold any scale
          t.v[u].zero();
#pragma unroll
          for (int c = 0; c < NC; ++c) t.vs[u][c] = 127;
        }
      }
    }
    if constexpr (kv_weights<KVF>()) {
#pragma unroll
      for (int u = 0; u < 2; ++u) logits.template store<logits_by4<MODE>()>(t0 + 16 * u + 4 * g, x[u], t_end);
    }
    float bm = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                     fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    // Lazy rescaling, as in the other loops: whether any score exceeds the
    // reference by the slack needs only each lane's own maximum.  A pair holds
    // at least one token, so the row's is finite.
    if (__builtin_amdgcn_ballot_w64(bm > m_run + kRescaleSlack) != 0) {
      bm = fmaxf(bm, shfl_xor_f(bm, 16));
      bm = fmaxf(bm, shfl_xor_f(bm, 32));
      const float m_new = fmaxf(m_run, bm);
      const float alpha = exp2_fast(m_run - m_new);
      o_l[0] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      m_run = m_new;
    }
    // P rounded to q's type; l sums the rounded weights that P.V uses (the
    // unrounded ones where the caller gets the weights).
    u4_t pw;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p0 = exp2_fast(x[j >> 1][2 * (j & 1)] - m_run), p1 = exp2_fast(x[j >> 1][2 * (j & 1) + 1] - m_run);
      pw[j] = pack2<KVF>(p0, p1);
      if constexpr (kv_weights<KVF>()) o_l[0] += p0 + p1;
    }
    const h8_t ph = __builtin_bit_cast(h8_t, pw);
    if constexpr (!kv_weights<KVF>()) {
      const uint32_t ones = pack2<KVF>(1.f, 1.f);
      o_l = mfma16x32<KVF>(__builtin_bit_cast(h8_t, u4_t{ones, ones, ones, ones}), ph, o_l);
    }
    // V through LDS, one block after the other in the same 16 rows (a wave's
    // LDS accesses complete in order).
    h4_t vt[2][DT];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int s = 0; s < DW; ++s)
        *reinterpret_cast<h8_t*>(stage + r16 * ROW + mx4_elem<D>(g, s) * 2) =
            mx4x8<KVF>(t.v[u].w[s], mx4_scale(t.vs[u][s / CW]));
      const char* src = stage + (4 * g + (r16 >> 2)) * ROW + (r16 & 3) * 8;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vt[u][dt] = lds_read_transposed(src + dt * 32);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      o[dt] = mfma16x32<KVF>(__builtin_shufflevector(vt[0][dt], vt[1][dt], 0, 1, 2, 3, 4, 5, 6, 7), ph, o[dt]);
  };

  // The next pair's rows are in flight while one is computed.
  const int npair = (nblk + 1) >> 1;
  const int n_mine = wave < npair ? (npair - wave + nw - 1) / nw : 0;
  Tile ta, tb;
  if (n_mine > 0) {
    int it = 0;
    fetch_ids();
    load(ta);
    load_q();
    for (; it + 2 < n_mine; it += 2) {
      load(tb);
      compute(ta, wave + it * nw);
      load(ta);
      compute(tb, wave + (it + 1) * nw);
    }
    if (it + 1 < n_mine) {
      load(tb);
      compute(ta, wave + it * nw);
      compute(tb, wave + (it + 1) * nw);
    } else {
      compute(ta, wave + it * nw);
    }
  }

  if constexpr (kv_weights<KVF>()) {
    o_l[0] += shfl_xor_f(o_l[0], 16);
    o_l[0] += shfl_xor_f(o_l[0], 32);
  }
  if (row_ok) {
    if (g == 0) sm_ml[slot * 16 + r16] = make_float2(m_run, o_l[0]);
    float* dst = sm_o + (slot * a.gqa + r16) * wave_row_floats<D>() + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4_t*>(dst + dt * 16) = o[dt];
  }
}

}  // namespace pad

#endif  // PA_MX4_H_
