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

#include "pa_device.h"

namespace pad {

// Waves per SIMD that the kernels are compiled for (registers per lane): the
// scores' row pointers did not fit 168 registers at head_dim 128.
constexpr int mx4_waves_per_simd(int d, bool weights) { return d <= 128 ? (d == 128 && weights ? 2 : 3) : 1; }

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

__device__ __forceinline__ float* logits_of(const Phase1Args& a, int b, int kvh, int row);
__device__ __forceinline__ void store_logits(float* p, const float (&x)[4], int n);

// MODE: kModeUniform (a 16-token tile lies in one page) or kModeGeneric (each
// lane finds its own tokens' pages).
template <int D, int MODE, int KVF>
__device__ __forceinline__ void wave_loop_mx4(const Phase1Args& a, const int32_t* bt_row, int64_t ids_stride, int b,
                                              int kvh, int t_begin, int t_end, int nblk, int wave, int nw, int lane,
                                              float2* sm_ml, float* sm_o, char* stage) {
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
  float l_run = 0.f;
  f4_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = (f4_t)0.f;

  const char* k_head = reinterpret_cast<const char*>(a.k) + (int64_t)kvh * a.skh;
  const char* v_head = reinterpret_cast<const char*>(a.v) + (int64_t)kvh * a.svh;
  const uint8_t* ks_head = a.ks + (int64_t)kvh * a.sksh;
  const uint8_t* vs_head = a.vs + (int64_t)kvh * a.svsh;
  const int elem0 = mx4_elem<D>(g, 0);
  float* logit_row = nullptr;
  if constexpr (kv_weights<KVF>()) logit_row = logits_of(a, b, kvh, row_ok ? r16 : 0);

  auto load_row = [&](Tile& t, int u, const char* kp, const char* vp, const uint8_t* ksp, const uint8_t* vsp) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const HVec<CW> x = load_hvec_stream<CW>(reinterpret_cast<const _Float16*>(kp + c * 64));
#pragma unroll
      for (int w = 0; w < CW; ++w) t.k[u].w[c * CW + w] = x.w[w];
      t.ks[u][c] = ksp[c * 4];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const HVec<CW> x = load_hvec_stream<CW>(reinterpret_cast<const _Float16*>(vp + c * 64));
#pragma unroll
      for (int w = 0; w < CW; ++w) t.v[u].w[c * CW + w] = x.w[w];
      t.vs[u][c] = vsp[c * 4];
    }
  };

  // Page ids of the pair the next load() reads: scalar reads (whole-page
  // tiles), or each lane's own.  They are fetched a pair ahead, before that
  // pair's predecessor's rows, so that waiting for them waits for no rows.
  const int p_first = page_of(a, t_begin);
  int pid[2], slot[2];
  auto fetch_ids = [&](int jp) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (MODE == kModeUniform) {
        const int jb = min(2 * jp + u, nblk - 1);
        const int page = block_page(a, jb);
        slot[u] = jb * kBlockTokens - page * a.ps;
        pid[u] = load_uniform_i32(bt_row + (int64_t)(p_first + page) * ids_stride);
      } else {
        const int tk = min(t_begin + jp * 32 + 16 * u + r16, t_end - 1);
        const int page = page_of(a, tk);
        slot[u] = tk - page * a.ps;
        pid[u] = bt_row[(int64_t)page * ids_stride];
      }
    }
  };
  // Lane offsets inside a tile (whole-page tiles: row r16 of it).
  const int lane_row = MODE == kModeUniform ? r16 : 0;
  const int64_t koff = (int64_t)lane_row * a.sks + elem0 / 2;
  const int64_t voff = (int64_t)lane_row * a.svs + elem0 / 2;
  const int64_t ksoff = (int64_t)lane_row * a.skss + elem0 / 32;
  const int64_t vsoff = (int64_t)lane_row * a.svss + elem0 / 32;
  const int npair = (nblk + 1) >> 1;
  auto load = [&](Tile& t, int jp) {
    int64_t page[2], at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      page[u] = clamp_page(pid[u], a.num_pages);
      at[u] = slot[u];
    }
    fetch_ids(min(jp + nw, npair - 1));
#pragma unroll
    for (int u = 0; u < 2; ++u)
      load_row(t, u, k_head + page[u] * a.skp + at[u] * a.sks + koff, v_head + page[u] * a.svp + at[u] * a.svs + voff,
               ks_head + page[u] * a.sksp + at[u] * a.skss + ksoff,
               vs_head + page[u] * a.svsp + at[u] * a.svss + vsoff);
  };

  auto compute = [&](Tile& t, int jp) {
    const int t0 = t_begin + jp * 32;
    const bool full = t0 + 32 <= t_end;
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
    if (!full) {
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
      for (int u = 0; u < 2; ++u) {
        const int tk = t0 + 16 * u + 4 * g;
        store_logits(logit_row + tk, x[u], row_ok ? t_end - tk : 0);
      }
    }
    float bm = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                     fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    bm = fmaxf(bm, shfl_xor_f(bm, 16));
    bm = fmaxf(bm, shfl_xor_f(bm, 32));
    // Lazy rescaling, as in wave_loop_mfma: a pair holds at least one token.
    if (__builtin_amdgcn_ballot_w64(bm > m_run + kRescaleSlack) != 0) {
      const float m_new = fmaxf(m_run, bm);
      const float alpha = exp2_fast(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      m_run = m_new;
    }
    // P rounded to q's type; l sums the rounded weights that P.V uses (the
    // unrounded ones where the caller gets the weights).
    h8_t ph;
    float psum = 0.f;
    if constexpr (q_is_bf16<KVF>()) {
      typedef float f2_t __attribute__((ext_vector_type(2)));
      typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
      u4_t w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f2_t pf = {exp2_fast(x[j >> 1][2 * (j & 1)] - m_run), exp2_fast(x[j >> 1][2 * (j & 1) + 1] - m_run)};
        const uint32_t pr = __builtin_bit_cast(uint32_t, __builtin_convertvector(pf, b2_t));
        w[j] = pr;
        if constexpr (kv_weights<KVF>())
          psum += pf.x + pf.y;
        else
          psum += __uint_as_float(pr << 16) + __uint_as_float(pr & 0xffff0000u);
      }
      ph = __builtin_bit_cast(h8_t, w);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float pf = exp2_fast(x[j >> 2][j & 3] - m_run);
        const _Float16 p = (_Float16)pf;
        ph[j] = p;
        psum += kv_weights<KVF>() ? pf : (float)p;
      }
    }
    l_run += psum;
    // V through LDS, one tile after the other in the same 16 rows (a wave's
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

  // This wave's pairs are wave, wave+nw, ...: the next pair's rows are in
  // flight while one is computed.
  const int n_mine = wave < npair ? (npair - wave + nw - 1) / nw : 0;
  Tile ta, tb;
  if (n_mine > 0) {
    int it = 0;
    fetch_ids(wave);
    load(ta, wave);
    load_q();
    for (; it + 2 < n_mine; it += 2) {
      load(tb, wave + (it + 1) * nw);
      compute(ta, wave + it * nw);
      load(ta, wave + (it + 2) * nw);
      compute(tb, wave + (it + 1) * nw);
    }
    if (it + 1 < n_mine) {
      load(tb, wave + (it + 1) * nw);
      compute(ta, wave + it * nw);
      compute(tb, wave + (it + 1) * nw);
    } else {
      compute(ta, wave + it * nw);
    }
  }

  float l_tot = l_run + shfl_xor_f(l_run, 16);
  l_tot += shfl_xor_f(l_tot, 32);
  if (row_ok) {
    if (g == 0) sm_ml[wave * 16 + r16] = make_float2(m_run, l_tot);
    float* dst = sm_o + (wave * a.gqa + r16) * wave_row_floats<D>() + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f4_t*>(dst + dt * 16) = o[dt];
  }
}

}  // namespace pad

#endif  // PA_MX4_H_
