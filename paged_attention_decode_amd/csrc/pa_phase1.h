// pa_phase1.h - the per-unit decode kernel (pad_phase1_kernel): its wave loops,
// work items and merge, instantiated by pa_decode.hip (fp16, bfloat16 and fp8
// caches), pa_mx4.hip (MX4 caches) and pa_weights*.hip (decodes that also write
// their logits).  pa_decode.hip describes the design.
#ifndef PA_PHASE1_H_
#define PA_PHASE1_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "pa_device.h"
#include "pa_decode_timeline.h"  // PAD_TL_* constants
#include "pa_mx4.h"

// Phase stamps of the measurement library (pa_decode.hip defines them there).
#ifndef PAD_TL
#define PAD_TL_AT(lin, slot, value) \
  do {                              \
  } while (0)
#define PAD_TL(lin, slot) \
  do {                    \
  } while (0)
#endif

namespace pad {

// One 16-token block of K and V in registers as loaded: lane (g, r16) holds
// its D/16 elements of token 4g+i (fp16: D/32 dwords; fp8 caches: D/64
// dwords of codes, widened to fp16 only where compute() uses them, so that
// the loads of the next block stay in flight across the current one).
template <int D, int ES = 2>
struct KVTile {
  HVec<D * ES / 64> k[4];
  HVec<D * ES / 64> v[4];
};

// Engine 0: MFMA 16x16x16 f16 tiles, two blocks in flight per wave (the
// loads of block j+nw are issued before block j is computed).
template <int D, int MODE, int KVF = kKvF16>
__device__ __forceinline__ void wave_loop_mfma(const Phase1Args& a, int phys_first, const int32_t* bt_row,
                                               int64_t ids_stride, int b, int kvh, int t_begin, int t_end,
                                               int nblk, int wave, int nw, int lane, float2* sm_ml, float* sm_o,
                                               char* k_stage, char* q_stage) {
  constexpr int DK = D / 32;  // 16-byte K chunks per lane per token
  constexpr int DT = D / 16;  // PV output tiles; V halves per lane per token
  constexpr int NDW = DT / 2;
  constexpr int ES = kv_elem_bytes<KVF>();  // bytes per cache element
  static_assert(!kv_is_fp8<KVF>() || NDW % 2 == 0, "fp8 caches: head_dim a multiple of 64");
  // A lane's DT halves of a token row are NSEG segments of SEG dwords, so
  // that the 16 lanes of a group read 16*SEG*4 contiguous bytes per load
  // instruction: half dt is head_dim slot dim(r16, dt) =
  // (dt / (2*SEG)) * (D / NSEG) + r16 * 2*SEG + dt % (2*SEG).  One segment
  // (the slice r16*DT .. +DT) up to head_dim 128; head_dim 256 reads two
  // 256-byte row halves rather than 16 strided 32-byte slices.
  constexpr int SEG = NDW > 4 ? 4 : NDW;
  constexpr int NSEG = NDW / SEG;
  constexpr int SEG_HALVES = D / NSEG;  // head_dim distance between segments
  // Dwords per lane per token row as loaded (fp8: half of NDW).
  constexpr int NDWR = NDW * ES / 2;
  using Tile = KVTile<D, ES>;
  auto load_slice = [](const char* p) -> HVec<NDWR> {
    if constexpr (kv_is_fp8<KVF>()) {
      // fp8: the same segments at one byte per element, kept as codes.
      HVec<NDWR> r;
#pragma unroll
      for (int sg = 0; sg < NSEG; ++sg) {
        const HVec<SEG / 2> x = load_hvec_stream<SEG / 2>(reinterpret_cast<const _Float16*>(p + sg * SEG_HALVES));
#pragma unroll
        for (int w = 0; w < SEG / 2; ++w) r.w[sg * (SEG / 2) + w] = x.w[w];
      }
      return r;
    } else if constexpr (NSEG == 1) {
      return load_hvec_stream<NDW>(reinterpret_cast<const _Float16*>(p));
    } else {
      HVec<NDW> r;
#pragma unroll
      for (int sg = 0; sg < NSEG; ++sg) {
        const HVec<SEG> x = load_hvec_stream<SEG>(reinterpret_cast<const _Float16*>(p) + sg * SEG_HALVES);
#pragma unroll
        for (int w = 0; w < SEG; ++w) r.w[sg * SEG + w] = x.w[w];
      }
      return r;
    }
  };
  // A loaded row in the fp16 layout (fp8 codes: four per dword, widened).
  auto widen = [](const HVec<NDWR>& x) -> HVec<NDW> {
    if constexpr (!kv_is_fp8<KVF>()) {
      return x;
    } else {
      HVec<NDW> r;
#pragma unroll
      for (int w = 0; w < NDWR; ++w) fp8x4_to_16x4<KVF>(x.w[w], r.w[2 * w], r.w[2 * w + 1]);
      return r;
    }
  };
  const int g = lane >> 4;
  const int r16 = lane & 15;
  const bool row_ok = r16 < a.gqa;
  // The wave's Q^T operand (B of S^T = K.Q^T: row r16, head_dim slots
  // kp*32 + g*8 + [0,8)), loaded after the first K/V block is in flight.
  h8_t qv[q_in_lds<D>() ? 1 : DK];
  auto q_slot = [&](int kp) -> h8_t* {
    return reinterpret_cast<h8_t*>(q_stage + r16 * k_stage_row_bytes<D>() + (kp * 32 + g * 8) * 2);
  };
  auto load_q = [&]() {
    const _Float16* qrow = a.q + (int64_t)b * a.sqb + (int64_t)(kvh * a.gqa + (row_ok ? r16 : 0)) * a.sqh;
#pragma unroll
    for (int kp = 0; kp < DK; ++kp) {
      const h8_t x = *reinterpret_cast<const h8_t*>(qrow + kp * 32 + g * 8);
      if constexpr (q_in_lds<D>())
        *q_slot(kp) = row_ok ? x : (h8_t)0;
      else
        qv[kp] = row_ok ? x : (h8_t)0;
    }
  };

  float m_run = kNegInf;
  float l_run = 0.f;
  f4_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = (f4_t)0.f;

  const char* k_head = reinterpret_cast<const char*>(a.k) + (int64_t)kvh * a.skh * ES;
  const char* v_head = reinterpret_cast<const char*>(a.v) + (int64_t)kvh * a.svh * ES;
  const std::conditional_t<kv_weights<KVF>(), Logits, NoLogits> logits(a, b, kvh, r16);
  // Lane byte offsets inside a 16-token slab of one page (loop invariant).
  // K and V are both read as whole token rows: lane (g, r16) reads row
  // 4g+i, segments at head_dim r16*2*SEG (+ D/NSEG), so one load
  // instruction covers four rows (contiguous 256 B each at head_dim 128).  K then goes through LDS
  // into the MFMA operand layout (token per lane%16).
  // Sub-page blocks: token 4g+i sits in slot (4g+i) mod page_size of its
  // page (blocks start on page boundaries), again loop invariant.
  constexpr int SUB_SHIFT = MODE >= kModeSubpage ? MODE - kModeSubpage : 0;
  constexpr int SUB_PAGES = 16 >> SUB_SHIFT;  // pages per 16-token block
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = MODE >= kModeSubpage ? (4 * g + i) & ((1 << SUB_SHIFT) - 1) : 4 * g + i;
    koff[i] = (uint32_t)(((int64_t)row * a.sks + r16 * 2 * SEG) * ES);
    voff[i] = (uint32_t)(((int64_t)row * a.svs + r16 * 2 * SEG) * ES);
  }
  constexpr int KROW = k_stage_row_bytes<D>();
  const int p_first = page_of(a, t_begin);
  // Sub-page and generic blocks: the raw page ids of the block the next
  // load() reads, read with scalar loads one block ahead like pid_next;
  // columns past the item's last page are clamped to it (its tokens are
  // masked).  Generic mode (page sizes >= 3 that neither divide nor are a
  // multiple of 16; the MFMA engine sends 1 and 2 to the sub-page mode):
  // 16 tokens starting anywhere in a page span at most
  // floor((ps + 14) / ps) + 1 <= 6 pages, the block's first page and its
  // first token's slot (gen_r0) are found by an exact float-reciprocal
  // division, and each token's page index and slot follow from
  // pos = gen_r0 + token: (pos + 0.5) / ps is never within 0.5 / ps of an
  // integer, so truncating its float value is exact for the small pos here.
  constexpr int GEN_PAGES = 6;
  int ids_next[MODE >= kModeSubpage ? SUB_PAGES : (MODE == kModeGeneric ? GEN_PAGES : 1)];
  const int p_last = t_end > t_begin ? page_of(a, t_end - 1) : p_first;
  const float inv_ps = 1.0f / (float)a.ps;
  int gen_r0 = 0;
  auto fetch_ids = [&](int jb) {
    if constexpr (MODE >= kModeSubpage) {
      const int p0 = p_first + jb * SUB_PAGES;
#pragma unroll
      for (int k = 0; k < SUB_PAGES; ++k)
        ids_next[k] = load_uniform_i32(bt_row + (int64_t)min(p0 + k, p_last) * ids_stride);
    } else if constexpr (MODE == kModeGeneric) {
      const int t0 = t_begin + jb * kBlockTokens;
      int p0 = __builtin_amdgcn_readfirstlane((int)(((float)t0 + 0.5f) * inv_ps));
      p0 -= p0 * a.ps > t0 ? 1 : 0;  // exact for t0 < 2^23
      p0 += (p0 + 1) * a.ps <= t0 ? 1 : 0;
      gen_r0 = t0 - p0 * a.ps;
#pragma unroll
      for (int k = 0; k < GEN_PAGES; ++k)
        ids_next[k] = load_uniform_i32(bt_row + (int64_t)min(p0 + k, p_last) * ids_stride);
    }
  };

  // Uniform mode: raw page id of the block the next load() reads.  Each load()
  // consumes it and issues the scalar read of the following block's id, so
  // that read is in flight during a whole compute() (calls come in block
  // order wave, wave+nw, ...; past the split the last block's id is reread).
  int pid_next = phys_first;

  auto load = [&](Tile& t, int jb) {
    if constexpr (MODE == kModeUniform) {
      // page_size % 16 == 0 and splits start on page boundaries: the block
      // lives in one page, so its page id and base address are wave-uniform.
      const int jp = block_page(a, jb);
      const int slot0 = jb * kBlockTokens - jp * a.ps;
      const int phys = clamp_page(pid_next, a.num_pages);
      const int page_after = p_first + block_page(a, min(jb + nw, nblk - 1));
      pid_next = load_uniform_i32(bt_row + (int64_t)page_after * ids_stride);
      const char* kb = k_head + ((int64_t)phys * a.skp + (int64_t)slot0 * a.sks) * ES;
      const char* vb = v_head + ((int64_t)phys * a.svp + (int64_t)slot0 * a.svs) * ES;
#pragma unroll
      for (int i = 0; i < 4; ++i) t.k[i] = load_slice(kb + koff[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) t.v[i] = load_slice(vb + voff[i]);
    } else if constexpr (MODE >= kModeSubpage) {
      // page_size divides 16: the block covers SUB_PAGES whole pages whose
      // ids arrived during the previous compute(); lane group g picks the
      // page of its token 4g+i.  Past the item's end the clamped ids still
      // name valid pages (the tokens are masked in compute).
      // The ids are used up before the next block's are fetched into the
      // same registers.
#pragma unroll
      for (int k = 0; k < SUB_PAGES; ++k) ids_next[k] = clamp_page(ids_next[k], a.num_pages);
      const int64_t kpage = a.skp * ES, vpage = a.svp * ES;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c0 = ids_next[i >> SUB_SHIFT], c1 = ids_next[(4 + i) >> SUB_SHIFT];
        const int c2 = ids_next[(8 + i) >> SUB_SHIFT], c3 = ids_next[(12 + i) >> SUB_SHIFT];
        const int phys = g == 0 ? c0 : (g == 1 ? c1 : (g == 2 ? c2 : c3));
        t.k[i] = load_slice(k_head + (int64_t)phys * kpage + koff[i]);
        t.v[i] = load_slice(v_head + (int64_t)phys * vpage + voff[i]);
      }
      fetch_ids(min(jb + nw, nblk - 1));
    } else {
      // Generic page size (>= 3): token 4g+i is at pos = gen_r0 + 4g+i from
      // the start of the block's first page, i.e. in page pos / ps of the
      // block's (up to 6) prefetched ids, slot pos mod ps.  The ids are used
      // up before the next block's are fetched into the same registers.
#pragma unroll
      for (int k = 0; k < GEN_PAGES; ++k) ids_next[k] = clamp_page(ids_next[k], a.num_pages);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = gen_r0 + 4 * g + i;
        const int idx = (int)(((float)pos + 0.5f) * inv_ps);
        const int slot = pos - idx * a.ps;
        // idx in [0, 6): a binary mux over idx's bits.  (An equality select
        // chain was folded into an indexed read of the id array, which the
        // compiler placed in scratch memory: a vector memory round trip per
        // token that also drained the K/V loads in flight.)
        static_assert(GEN_PAGES == 6, "mux below covers 6 page ids");
        const bool b0 = (idx & 1) != 0;
        const int p01 = b0 ? ids_next[1] : ids_next[0];
        const int p23 = b0 ? ids_next[3] : ids_next[2];
        const int p45 = b0 ? ids_next[5] : ids_next[4];
        const int p03 = (idx & 2) ? p23 : p01;
        const int phys = (idx & 4) ? p45 : p03;
        const char* kr = k_head + ((int64_t)phys * a.skp + (int64_t)slot * a.sks + r16 * 2 * SEG) * ES;
        const char* vr = v_head + ((int64_t)phys * a.svp + (int64_t)slot * a.svs + r16 * 2 * SEG) * ES;
        t.k[i] = load_slice(kr);
        t.v[i] = load_slice(vr);
      }
      fetch_ids(min(jb + nw, nblk - 1));
    }
  };

  auto compute = [&](Tile& t, int jb) {
    const int t0 = t_begin + jb * kBlockTokens;
    const bool full = t0 + kBlockTokens <= t_end;
    // K rows -> LDS (row 4g+i, the lane's segments), then the MFMA A operand back
    // out: lane (g, r16) takes token r16, head_dim kp*32 + g*8 + [0, 8).
    // LDS accesses of one wave complete in order, so the reads see the
    // writes, and the next block's writes follow these reads.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(k_stage + (4 * g + i) * KROW + r16 * SEG * 4);
      const HVec<NDW> kr = widen(t.k[i]);
#pragma unroll
      for (int w = 0; w < NDW; ++w) dst[(w / SEG) * (SEG_HALVES / 2) + w % SEG] = kr.w[w];
    }
    h8_t kk[DK];
#pragma unroll
    for (int kp = 0; kp < DK; ++kp)
      kk[kp] = *reinterpret_cast<const h8_t*>(k_stage + r16 * KROW + (kp * 32 + g * 8) * 2);
    // S^T[token 4g+i][row r16] over head_dim.
    f4_t sacc = (f4_t)0.f;
#pragma unroll
    for (int kp = 0; kp < DK; ++kp) {
      const h4_t k_lo = __builtin_shufflevector(kk[kp], kk[kp], 0, 1, 2, 3);
      const h4_t k_hi = __builtin_shufflevector(kk[kp], kk[kp], 4, 5, 6, 7);
      h8_t qk;
      if constexpr (q_in_lds<D>())
        qk = *q_slot(kp);
      else
        qk = qv[kp];
      const h4_t q_lo = __builtin_shufflevector(qk, qk, 0, 1, 2, 3);
      const h4_t q_hi = __builtin_shufflevector(qk, qk, 4, 5, 6, 7);
      sacc = mfma16<KVF>(k_lo, q_lo, sacc);
      sacc = mfma16<KVF>(k_hi, q_hi, sacc);
    }
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = sacc[i] * a.scale_log2;
    if (!full) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool valid = t0 + 4 * g + i < t_end;
        x[i] = valid ? x[i] : kNegInf;
        if (!valid) t.v[i].zero();  // stale cache slots may hold NaN/Inf
      }
    }
    if constexpr (kv_weights<KVF>()) logits.template store<logits_by4<MODE>()>(t0 + 4 * g, x, t_end);
    float bm = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    bm = fmaxf(bm, shfl_xor_f(bm, 16));
    bm = fmaxf(bm, shfl_xor_f(bm, 32));
    // Lazy rescaling: the reference m_run only moves when a score exceeds it
    // by more than kRescaleSlack (base-2 units), so weights stay <= 2^slack
    // and the O/l rescale is skipped (wave-uniformly) on most blocks.  Any
    // reference value gives the same O/l; partials carry it as their m.
    // Every block holds at least one valid token, so bm is finite.
    if (__builtin_amdgcn_ballot_w64(bm > m_run + kRescaleSlack) != 0) {
      const float m_new = fmaxf(m_run, bm);
      const float alpha = exp2_fast(m_run - m_new);  // 0 on the first block
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      m_run = m_new;
    }
    h4_t ph;
    float psum = 0.f;  // l accumulates the same rounded weights P.V uses
    if constexpr (q_is_bf16<KVF>()) {
      // Pairs through the packed conversion; a rounded bf16 pair's floats
      // are its high and low halves shifted into place.
      typedef float f2_t __attribute__((ext_vector_type(2)));
      typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
      uint32_t u[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f2_t pf = {exp2_fast(x[2 * j] - m_run), exp2_fast(x[2 * j + 1] - m_run)};
        u[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pf, b2_t));
        if constexpr (kv_weights<KVF>())
          psum += pf.x + pf.y;  // the weights are unrounded: so is their sum
        else
          psum += __uint_as_float(u[j] << 16) + __uint_as_float(u[j] & 0xffff0000u);
      }
      typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
      ph = __builtin_bit_cast(h4_t, u2_t{u[0], u[1]});
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float pf = exp2_fast(x[i] - m_run);
        const _Float16 p = (_Float16)pf;
        ph[i] = p;
        psum += kv_weights<KVF>() ? pf : (float)p;
      }
    }
    l_run += psum;
    HVec<NDW> vr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vr[i] = widen(t.v[i]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      h4_t av;
#pragma unroll
      for (int i = 0; i < 4; ++i) av[i] = vr[i].h(dt);
      o[dt] = mfma16<KVF>(av, ph, o[dt]);
    }
  };

  // This wave's blocks are wave, wave+nw, ...  The steady-state loop issues
  // the next block's loads unconditionally before computing the current one
  // (no control-flow join on the in-flight registers); the last one or two
  // blocks are peeled.
  const int n_mine = wave < nblk ? (nblk - wave + nw - 1) / nw : 0;
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

  // Row totals: the four 16-lane groups hold disjoint token subsets.
  float l_tot = l_run + shfl_xor_f(l_run, 16);
  l_tot += shfl_xor_f(l_tot, 32);
  auto o_slot = [&](int i, int dt) {
    return (dt / (2 * SEG)) * SEG_HALVES + (4 * g + i) * 2 * SEG + dt % (2 * SEG);
  };
  if (row_ok) {
    if (g == 0) sm_ml[wave * 16 + r16] = make_float2(m_run, l_tot);
    // Lane owns O[row r16][dim(4g+i, dt)]: for each i, NSEG runs of 2*SEG
    // consecutive floats, written as 16- or 8-byte vectors.
    float* dst = sm_o + (wave * a.gqa + r16) * wave_row_floats<D>();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT % 4 == 0) {
#pragma unroll
        for (int dt = 0; dt < DT; dt += 4)
          *reinterpret_cast<f4_t*>(dst + o_slot(i, dt)) = f4_t{o[dt][i], o[dt + 1][i], o[dt + 2][i], o[dt + 3][i]};
      } else {
#pragma unroll
        for (int dt = 0; dt < DT; dt += 2)
          *reinterpret_cast<float2*>(dst + o_slot(i, dt)) = make_float2(o[dt][i], o[dt + 1][i]);
      }
    }
  }
}

// Engine 1: VALU dot products with DPP row reductions.
template <int D, bool UNIFORM, int GQA_T>
__device__ __forceinline__ void wave_loop_valu(const Phase1Args& a, const int32_t* bt_row, int64_t ids_stride,
                                               int b, int kvh, int t_begin, int t_end, int nblk, int wave,
                                               int nw, int lane, float2* sm_ml, float* sm_o) {
  constexpr int DT = D / 16;  // halves per lane per token
  constexpr int NDW = DT / 2;
  const int g = lane >> 4;    // token group: tokens 4g+i of each block
  const int r16 = lane & 15;  // head_dim slice r16*DT .. +DT
  const int gqa = a.gqa;

  HVec<NDW> qh[GQA_T];
#pragma unroll
  for (int r = 0; r < GQA_T; ++r) {
    if (r < gqa) {
      const _Float16* qrow = a.q + (int64_t)b * a.sqb + (int64_t)(kvh * gqa + r) * a.sqh;
      qh[r] = load_hvec<NDW>(qrow + r16 * DT);
    } else {
      qh[r].zero();
    }
  }
  float m_run[GQA_T], l_run[GQA_T], acc[GQA_T][DT];
#pragma unroll
  for (int r = 0; r < GQA_T; ++r) {
    m_run[r] = kNegInf;
    l_run[r] = 0.f;
#pragma unroll
    for (int e = 0; e < DT; ++e) acc[r][e] = 0.f;
  }

  const int64_t koff_h = (int64_t)kvh * a.skh;
  const int64_t voff_h = (int64_t)kvh * a.svh;

  for (int j = wave; j < nblk; j += nw) {
    const int t0 = t_begin + j * kBlockTokens;
    const _Float16* krow[4];
    const _Float16* vrow[4];
    if constexpr (UNIFORM) {
      const int page = page_of(a, t0);
      const int phys = clamp_page(load_uniform_i32(bt_row + (int64_t)page * ids_stride), a.num_pages);
      const int slot0 = t0 - page * a.ps;
      const _Float16* kbase = a.k + (int64_t)phys * a.skp + koff_h + (int64_t)slot0 * a.sks;
      const _Float16* vbase = a.v + (int64_t)phys * a.svp + voff_h + (int64_t)slot0 * a.svs;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        krow[i] = kbase + (int64_t)(4 * g + i) * a.sks;
        vrow[i] = vbase + (int64_t)(4 * g + i) * a.svs;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tv = min(t0 + 4 * g + i, t_end - 1);
        const int page = page_of(a, tv);
        const int phys = clamp_page(bt_row[(int64_t)page * ids_stride], a.num_pages);
        const int slot = tv - page * a.ps;
        krow[i] = a.k + (int64_t)phys * a.skp + koff_h + (int64_t)slot * a.sks;
        vrow[i] = a.v + (int64_t)phys * a.svp + voff_h + (int64_t)slot * a.svs;
      }
    }
    HVec<NDW> kk[4], vv[4];
    bool valid[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kk[i] = load_hvec<NDW>(krow[i] + r16 * DT);
      vv[i] = load_hvec<NDW>(vrow[i] + r16 * DT);
      valid[i] = t0 + 4 * g + i < t_end;
      if (!valid[i]) vv[i].zero();
    }
    float vf[4][DT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < DT; ++e) vf[i][e] = (float)vv[i].h(e);
    }

#pragma unroll
    for (int r = 0; r < GQA_T; ++r) {
      if (r >= gqa) break;
      float sc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float part = 0.f;
#pragma unroll
        for (int w = 0; w < NDW; ++w) part = __builtin_amdgcn_fdot2(qh[r].h2(w), kk[i].h2(w), part, false);
        part = row16_sum(part);
        sc[i] = valid[i] ? part * a.scale_log2 : kNegInf;
      }
      const float bm = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
      const float m_new = fmaxf(m_run[r], bm);
      if (m_new == kNegInf) continue;  // this group has seen no valid token yet
      const float alpha = exp2_fast(m_run[r] - m_new);
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = exp2_fast(sc[i] - m_new);
      l_run[r] = l_run[r] * alpha + ((p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
      for (int e = 0; e < DT; ++e) {
        float t = acc[r][e] * alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) t = fmaf(p[i], vf[i][e], t);
        acc[r][e] = t;
      }
      m_run[r] = m_new;
    }
  }

  // Merge the four token groups of this wave (lanes r16, r16+16, ...).
#pragma unroll
  for (int r = 0; r < GQA_T; ++r) {
    if (r >= gqa) break;
    float M = fmaxf(m_run[r], shfl_xor_f(m_run[r], 16));
    M = fmaxf(M, shfl_xor_f(M, 32));
    const float c = (m_run[r] == kNegInf) ? 0.f : exp2_fast(m_run[r] - M);
    float l = l_run[r] * c;
    l += shfl_xor_f(l, 16);
    l += shfl_xor_f(l, 32);
#pragma unroll
    for (int e = 0; e < DT; ++e) {
      float v = acc[r][e] * c;
      v += shfl_xor_f(v, 16);
      v += shfl_xor_f(v, 32);
      acc[r][e] = v;
    }
    if (g == 0) {
      if (r16 == 0) sm_ml[wave * 16 + r] = make_float2(M, l);
      float* dst = sm_o + (wave * gqa + r) * wave_row_floats<D>() + r16 * DT;
#pragma unroll
      for (int e = 0; e < DT; ++e) dst[e] = acc[r][e];
    }
  }
}

// ---------------------------------------------------------------------------
// Work items.  Workgroup (s, h, b) of the grid (grid_pos: the grid
// coordinates, or a bijection of them that pairs kv heads on an XCD) has
// index g = s + S*(h + Hkv*b) and processes one item: a page range of one
// (sequence, kv head) unit, writing its partial to slot g of the workspace.
// The items of a unit occupy the consecutive slots [slot0, slot0 + nsplit).
//  * Static items (an explicit split count, or every sequence at full
//    capacity): item g is split s of unit (b, h), pages [s*pps, (s+1)*pps).
//  * Planned items (heuristic split count, batch <= kPlanMaxBatch): every
//    workgroup reads all sequence lengths and computes the same plan - the
//    smallest chunk of c pages (c >= min_chunk) such that the units need at
//    most G items, each unit cut into ceil(pages/c) chunks (an empty unit
//    keeps one item, which writes its zero rows) - then takes item g in
//    (sequence, kv head, chunk) order.  Ragged batches thus spread their
//    pages evenly over the grid instead of leaving the splits of short
//    sequences empty.
// ---------------------------------------------------------------------------
struct WorkItem {
  int b, kvh;
  int p_begin, p_end;  // logical pages [p_begin, p_end) of sequence b
  int L;               // tokens of sequence b
  int nsplit;          // items of the unit; 0: the unit is empty (write zeros)
  int slot0;           // workspace slot of the unit's first item
  int col_max;         // last page-id column that may be read speculatively
  int valid;           // 0: no item for this workgroup
  const int32_t* ids_row;
  int64_t ids_stride;
};

// Value of lane (b % 64) of register k = b / 64 (b wave-uniform).
template <int NK>
__device__ __forceinline__ int seq_lane_value(const int (&v)[NK], int b) {
  const int l = b & 63;
  int x = __builtin_amdgcn_readlane(v[0], l);
#pragma unroll
  for (int k = 1; k < NK; ++k)
    if ((b >> 6) == k) x = __builtin_amdgcn_readlane(v[k], l);
  return x;
}

// ceil(p / c) for 0 <= p, c < 2^23: a float estimate corrected with exact
// 24-bit products (the estimate is within one of the quotient).
__device__ __forceinline__ int ceil_div_u23(int p, int c, float rc) {
  int n = (int)__builtin_ceilf((float)p * rc);
  n += (int)__umul24(n, c) < p ? 1 : 0;
  n -= (n > 0 && (int)__umul24(n - 1, c) >= p) ? 1 : 0;
  return n;
}

// Items per sequence with chunks of c pages (an empty sequence keeps one).
__device__ __forceinline__ int items_for(int pages, int c, float rc) { return max(ceil_div_u23(pages, c, rc), 1); }

// Items the units need for each of J chunk sizes (wave-uniform totals).  The
// J evaluations are independent, so their latencies overlap.
template <int NK, int J>
__device__ __forceinline__ void plan_counts(const Phase1Args& a, const SeqTable<NK>& t, const int (&c)[J],
                                            int (&n)[J], int lane) {
  float rc[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    rc[j] = 1.0f / (float)c[j];
    n[j] = 0;
  }
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const bool in = lane + 64 * k < a.batch;
#pragma unroll
    for (int j = 0; j < J; ++j) n[j] += in ? items_for(t.pages[k], c[j], rc[j]) : 0;
  }
#pragma unroll
  for (int j = 0; j < J; ++j) n[j] = row16_sum_i32(n[j]);
#pragma unroll
  for (int j = 0; j < J; ++j)
    n[j] = (__builtin_amdgcn_readlane(n[j], 0) + __builtin_amdgcn_readlane(n[j], 16) +
            __builtin_amdgcn_readlane(n[j], 32) + __builtin_amdgcn_readlane(n[j], 48)) *
           a.hkv;
}

template <int NK>
__device__ WorkItem plan_item(const Phase1Args& a, const SeqTable<NK>& t, int g, int G, int lane) {
  WorkItem w{};  // a slot without an item keeps defined (zero) fields
  w.ids_row = a.bt;
  int tot = 0, pmax = 0;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    tot += t.pages[k];
    pmax = max(pmax, t.pages[k]);
  }
  tot = wave_sum_i32(tot);
  pmax = max(wave_max_i32(pmax), 1);
  // Chunk size: the smallest c >= c_lo whose item count fits the grid would
  // be ideal, but every probe costs a pass over the table, so at most two
  // are made.  c_lo = ceil(unit pages / G) (fits when the lengths divide
  // evenly); then c_est, which assumes each non-empty unit rounds up by half
  // a chunk; failing that c_hi = ceil(unit pages / (G - units)), which
  // always fits since sum(ceil(p / c)) <= unit pages / c + units (and so
  // does pmax: one item per unit, G >= units).
  const int units = a.batch * a.hkv;
  const int64_t unit_pages = (int64_t)tot * a.hkv;
  int c = min(max(max(a.min_chunk, (int)((unit_pages + G - 1) / G)), 1), pmax);
  int n1[1], c1[1] = {c};
  plan_counts<NK, 1>(a, t, c1, n1, lane);
  if (n1[0] > G) {
    int c_hi = pmax;
    if (G > units) c_hi = min(c_hi, (int)((unit_pages + (G - units) - 1) / (G - units)));
    const int half = G - units / 2;
    int c_est = half > 0 ? (int)((unit_pages + half - 1) / half) : c_hi;
    c_est = max(c + 1, min(c_est, c_hi));
    c1[0] = c_est;
    plan_counts<NK, 1>(a, t, c1, n1, lane);
    c = n1[0] <= G ? c_est : max(c_hi, c_est);
  }
  // Locate item g: units in (sequence, kv head) order, n_b items each.
  w.valid = 0;
  int carry = 0;
  const float rc = 1.0f / (float)c;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    if (64 * k >= a.batch) break;
    const int b = lane + 64 * k;
    const int nb = b < a.batch ? items_for(t.pages[k], c, rc) : 0;
    const int x = nb * a.hkv;
    const int incl = wave_incl_scan_i32(x, lane) + carry;
    const int excl = incl - x;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(b < a.batch && excl <= g && g < incl);
    if (hit != 0) {
      const int l = (int)__builtin_ctzll(hit);
      const int first = __builtin_amdgcn_readlane(excl, l);
      const int n = __builtin_amdgcn_readlane(nb, l);
      const int pages = __builtin_amdgcn_readlane(t.pages[k], l);
      const int r = g - first;
      w.b = 64 * k + l;
      w.kvh = r / n;
      const int chunk = r - w.kvh * n;
      w.p_begin = chunk * c;
      w.p_end = min(w.p_begin + c, pages);
      w.L = __builtin_amdgcn_readlane(t.len[k], l);
      w.nsplit = pages > 0 ? n : 0;
      w.slot0 = first + w.kvh * n;
      w.col_max = pages - 1;
      w.ids_row = a.csr ? a.bt + __builtin_amdgcn_readlane(t.row[k], l) : a.bt + (int64_t)w.b * a.sbb;
      w.valid = 1;
      break;
    }
    carry = __builtin_amdgcn_readlane(incl, 63);
  }
  w.ids_stride = a.csr ? 1 : a.sbp;
  return w;
}

// The static item of workgroup (s, kvh, b) given the sequence's length and
// page count.  The dense table splits every row's max_pages columns into
// num_splits ranges of pps pages; a CSR index has no common row width, so
// each sequence's own pages are cut into num_splits ranges.
__device__ __forceinline__ WorkItem static_item(const Phase1Args& a, int s, int kvh, int b, int L, int pages,
                                                const int32_t* ids_row, int64_t ids_stride) {
  WorkItem w;
  const int pps = a.csr ? max((pages + a.num_splits - 1) / a.num_splits, 1) : a.pps;
  w.b = b;
  w.kvh = kvh;
  w.L = L;
  w.p_begin = s * pps;
  w.p_end = min(w.p_begin + pps, pages);
  w.nsplit = (pages + pps - 1) / pps;
  w.slot0 = (b * a.hkv + kvh) * a.num_splits;
  w.col_max = a.csr ? pages - 1 : a.max_pages - 1;
  // Splits past the sequence's last page do nothing, except split 0 of an
  // empty sequence, which writes its zero rows.
  w.valid = s < w.nsplit || s == 0;
  w.ids_row = ids_row;
  w.ids_stride = ids_stride;
  return w;
}

// Planned mode: read every sequence length; with every sequence at full
// capacity the static split is already even (balance == 1) or, on an
// oversubscribed grid (balance >= 2), the static splits run on the first
// workgroups (one item per unit, workgroup g = unit, when the static rule
// gives one split) and the other workgroups exit; otherwise plan the items.
template <int NK>
__device__ __forceinline__ WorkItem resolve_item(const Phase1Args& a, const SeqRaw& raw, int s, int h, int bz, int g,
                                                 int G, int lin, const int32_t* static_row, int lane) {
  const SeqTable<NK> t = seq_table<NK>(a, raw, lane);
  bool full = !a.csr;
#pragma unroll
  for (int k = 0; k < NK; ++k)
    if (lane + 64 * k < a.batch && t.pages[k] != a.max_pages) full = false;
  if (__builtin_amdgcn_ballot_w64(!full) == 0) {
    if (a.balance >= 2) {
      // The static splits, s0 per unit of pps pages, on the first units * s0
      // workgroups in order: unit g / s0, split g mod s0, whose partials
      // take the unit's s0 consecutive slots (the launch keeps head pairing
      // off when s0 > 1, so g is the linear index and the active workgroups
      // spread over the XCDs).  With s0 = 1 (pps = max_pages) each unit is
      // one item that writes the output rows and never a partial, so its
      // slot is the workgroup's own (g, which the work list's record check
      // expects); with pair_heads, units 2r and 2r+1 (kv heads 2m, 2m+1 of
      // one sequence) then go to workgroups 8 apart, as grid_pos does for
      // splits.
      WorkItem w;
      const int units = a.batch * a.hkv;
      const int s0 = a.balance - 1;  // 1, 2 or 3 (setup_launch)
      const bool paired = s0 == 1 && a.pair_heads && units % 16 == 0;
      const int gu = paired ? 2 * (((lin >> 4) << 3) | (lin & 7)) + ((lin >> 3) & 1) : g;
      // g / s0 by a shift or a multiply (exact for g < 2^16; G is far below)
      const int q = s0 == 2 ? g >> 1 : s0 == 3 ? (int)(((uint32_t)g * 43691u) >> 17) : (paired ? (lin < units ? gu : units) : g);
      const int u = min(q, units - 1);
      w.b = u / a.hkv;
      w.kvh = u - w.b * a.hkv;
      w.p_begin = s0 > 1 ? (g - q * s0) * a.pps : 0;
      w.p_end = min(w.p_begin + a.pps, a.max_pages);
      w.L = seq_lane_value<NK>(t.len, w.b);
      w.nsplit = a.max_pages > 0 ? s0 : 0;
      w.slot0 = s0 > 1 ? q * s0 : g;
      w.col_max = a.max_pages - 1;
      w.valid = q < units;
      w.ids_row = a.bt + (int64_t)w.b * a.sbb;
      w.ids_stride = a.sbp;
      return w;
    }
    return static_item(a, s, h, bz, seq_lane_value<NK>(t.len, bz), a.max_pages, static_row, a.sbp);
  }
  return plan_item<NK>(a, t, g, G, lane);
}

// The work item of workgroup (s, h, bz) = slot g: the in-kernel plan when
// a.balance is set, else the static split.  raw is issue_seq_table()'s
// loads; static_len is seq_lens[bz] (dense) or any word (CSR).  The decode
// kernel and the work-list planner both call this, so a planned launch runs
// exactly the items of an unplanned one.
__device__ __forceinline__ WorkItem resolve_workgroup(const Phase1Args& a, const SeqRaw& raw, int s, int h, int bz,
                                                      int g, int G, int lin, const int32_t* static_row,
                                                      int static_len, int lane) {
  if (a.balance) {
    if (a.batch <= 64) return resolve_item<1>(a, raw, s, h, bz, g, G, lin, static_row, lane);
    return resolve_item<4>(a, raw, s, h, bz, g, G, lin, static_row, lane);
  }
  if (a.csr) {
    int row, pages, L;
    csr_row(a, bz, &row, &pages, &L);
    return static_item(a, s, h, bz, L, pages, a.bt + row, 1);
  }
  const int L = max(static_len, 0);
  return static_item(a, s, h, bz, L, min(pages_for(a, L), a.max_pages), static_row, a.sbp);
}

// Work list (pad_decode_plan_worklist): a header of kWlHeaderInts int32
// {magic, plan key, G} and one record of kWlRecordInts int32 per workgroup
// slot g: {b, kvh, p_begin, p_end, L, nsplit, slot0, col_max, valid, row
// (CSR offset of the sequence's ids, else 0), 6 unused, then the raw page id
// of the first block of waves 0-7 (whole-page blocks; 0 otherwise), 8
// unused}.
constexpr int kWlHeaderInts = 32;
constexpr int kWlRecordInts = 32;
constexpr int kWlMagic = 0x574c4150;  // "PALW"

// Record g of a.worklist as a work item and the raw first page id of this
// wave's first block.  False (use the in-kernel plan) when the header does
// not carry this launch's plan key.  A record that does not describe an
// item of this launch's shapes is treated as no item, so a stale list can
// give wrong rows but never reads or writes out of bounds.
__device__ __forceinline__ bool worklist_item(const Phase1Args& a, int g, int G, int wave, WorkItem& w, int& pid) {
  const int32_t* r = a.worklist + kWlHeaderInts + (int64_t)kWlRecordInts * g;
  const int magic = load_uniform_i32(a.worklist);
  const int key = load_uniform_i32(a.worklist + 1);
  int f[10];
#pragma unroll
  for (int i = 0; i < 10; ++i) f[i] = load_uniform_i32(r + i);
  pid = load_uniform_i32(r + 16 + wave);
  // The record's values are only used past the header check, so the
  // compiler would sink their loads below it: a second round trip.  Pinning
  // them here keeps the header and the record in one.
#pragma unroll
  for (int i = 0; i < 10; ++i) asm volatile("" : "+s"(f[i]));
  asm volatile("" : "+s"(pid));
  if (magic != kWlMagic || key != a.wl_key) return false;
  w.b = f[0];
  w.kvh = f[1];
  w.p_begin = f[2];
  w.p_end = f[3];
  w.L = f[4];
  w.nsplit = f[5];
  w.slot0 = f[6];
  w.col_max = f[7];
  const int row = f[9];
  const bool ok = f[8] != 0 && w.b >= 0 && w.b < a.batch && w.kvh >= 0 && w.kvh < a.hkv && w.p_begin >= 0 &&
                  w.p_begin <= w.p_end && w.p_end <= w.col_max + 1 && w.L >= 0 && w.nsplit >= 0 &&
                  w.nsplit <= G && w.slot0 >= 0 && w.slot0 <= G - w.nsplit &&
                  (w.nsplit == 0 || (g >= w.slot0 && g < w.slot0 + w.nsplit)) && row >= 0 &&
                  (int64_t)row + w.col_max < a.max_pages;
  w.valid = ok ? 1 : 0;
  w.ids_row = a.csr ? a.bt + row : a.bt + (int64_t)(ok ? w.b : 0) * a.sbb;
  w.ids_stride = a.csr ? 1 : a.sbp;
  return true;
}

// Minimum waves per SIMD each phase-1 instantiation is compiled for (it
// caps the registers per lane at 512 / waves).  The generic page-size mode
// of head_dim 128 gets 2 (256 registers): its six prefetched page ids did
// not fit 168 registers without one VGPR spilled to scratch; so do the
// bfloat16 sub-page modes of head_dim 128 (2 VGPRs spilled at page size 4).
constexpr int phase1_waves_per_simd(int d, int engine, int mode, int kvf) {
  if ((kvf & 15) >= kKvMx4) return mx4_waves_per_simd(d);
  const bool wide = d == 128 && (mode == 0 || ((kvf == kKvBF16 || kvf == kKvE4M3B || kvf == kKvE5M2B) &&
                                                 mode >= kModeSubpage) || (kvf & kKvWeights));
  return engine == 0 ? (d <= 128 ? (wide ? 2 : 3) : 1) : 1;
}

// Most waves in one workgroup.  head_dim 256 takes at most 4, so that each
// SIMD runs one wave of the workgroup and that wave has the whole register
// file (256 VGPRs plus AGPRs for spills): with 5 or more waves two share a
// SIMD's 256 VGPRs, and the loop spilled 7-10 VGPRs to scratch memory.
constexpr int max_group_waves(int d) { return d >= 256 ? 4 : kMaxWaves; }

// The (split, kv head, sequence) of this workgroup.  Normally the grid
// coordinates.  With pair_heads (head_dim rows that are not a multiple of
// 128 bytes, so kv heads 2m and 2m+1 share a cache line in every token
// slot; an even head count; G a multiple of 16) linear workgroup L takes
// head parity (L / 8) mod 2 and the rest of its position from the other
// bits: the two workgroups of a head pair are 8 apart, which the dispatcher
// places on the same XCD one after the other, so the line they share is
// fetched into that XCD's L2 once.  Any bijection of the grid is correct;
// this one only changes what shares a cache.
__device__ __forceinline__ void grid_pos(const Phase1Args& a, int& s, int& h, int& bz, int& lin) {
  s = blockIdx.x;
  h = blockIdx.y;
  bz = blockIdx.z;
  lin = blockIdx.x + a.num_splits * (blockIdx.y + a.hkv * blockIdx.z);
  if (a.pair_heads) {
    const int rest = ((lin >> 4) << 3) | (lin & 7);
    const int q = rest / a.num_splits;
    const int half = a.hkv >> 1;
    s = rest - q * a.num_splits;
    bz = q / half;
    h = 2 * (q - bz * half) + ((lin >> 3) & 1);
  }
}

// Phase 1: one workgroup per (split, kv head, sequence).  KVF: the caches'
// element format (fp16, or fp8 on the MFMA engine).
template <int D, int MODE, int ENGINE, int GQA_T, int KVF = kKvF16>
__global__ __launch_bounds__(max_group_waves(D) * 64)
    __attribute__((amdgpu_waves_per_eu(phase1_waves_per_simd(D, ENGINE, MODE, KVF))))
void pad_phase1_kernel(const Phase1Args a) {
#ifdef PAD_TIMELINE
  const unsigned long long tl_entry = __builtin_amdgcn_s_memrealtime();
  const unsigned long long tl_xcc = (unsigned long long)(__builtin_amdgcn_s_getreg((3 << 11) | 20) & 15) << 32;
#define PAD_TL_NOTE(item_slot, flags) \
  PAD_TL_AT(lin, PAD_TL_INFO, (unsigned long long)(uint32_t)(item_slot) | tl_xcc | ((unsigned long long)(flags) << 40))
#else
#define PAD_TL_NOTE(item_slot, flags) \
  do {                                \
  } while (0)
#endif
  extern __shared__ float4 smem_f4[];
  float2* sm_ml = reinterpret_cast<float2*>(smem_f4);  // [nw][16]
  const int nw = a.nw;
  float* sm_o = reinterpret_cast<float*>(smem_f4) + nw * 32;  // [nw][gqa][D + 4]
  // [nw] K staging tiles (MFMA engine), after the wave states.
  char* k_stage_all = reinterpret_cast<char*>(sm_o + nw * a.gqa * wave_row_floats<D>());

  int s, h, bz, lin;
  grid_pos(a, s, h, bz, lin);
  PAD_TL_AT(blockIdx.x + a.num_splits * (blockIdx.y + a.hkv * blockIdx.z), PAD_TL_ENTRY, tl_entry);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = s + a.num_splits * (h + a.hkv * bz);
  const int G = a.num_splits * a.hkv * a.batch;

  // With a work list, the item and its first page ids arrive in one round
  // trip.  Otherwise, with the dense table, read the first page id of this
  // workgroup's static split before the sequence lengths arrive; it stays
  // valid whenever the item turns out to be the static one.
  WorkItem it;
  int phys_first = 0;
  bool first_known;
  if (a.worklist != nullptr && worklist_item(a, g, G, wave, it, phys_first)) {
    first_known = true;
  } else {
    // The sequence table's loads go first, then the page id and this
    // workgroup's sequence length: one round trip for all of them.  The
    // page-id read has no branch (a CSR index or an empty table reads a
    // valid word that is never used), as a value loaded under a branch
    // would be waited for where the branch joins, before the later loads.
    const SeqRaw raw = issue_seq_table(a, lane);
    const int32_t* static_row = a.bt + (int64_t)bz * a.sbb;
    if constexpr (ENGINE == 0 && MODE == kModeUniform && !kv_is_mx4<KVF>()) {
      const int col = min(s * a.pps + block_page(a, wave), a.max_pages - 1);
      const bool use = !a.csr && a.max_pages > 0;
      phys_first = load_uniform_i32(use ? static_row + (int64_t)col * a.sbp : (a.csr ? a.indptr : a.sl));
    }
    const int static_len = load_uniform_i32(a.csr ? a.indptr : a.sl + (int64_t)bz * a.ssl);
    it = resolve_workgroup(a, raw, s, h, bz, g, G, lin, static_row, static_len, lane);
    first_known = !a.csr && it.b == bz && it.p_begin == s * a.pps;
  }
  PAD_TL(lin, PAD_TL_ITEM);
  if (!it.valid) {
    PAD_TL_NOTE(-1, PAD_TL_F_NO_ITEM);
    PAD_TL(lin, PAD_TL_EXIT);
    return;
  }
  const int b = it.b;
  const int kvh = it.kvh;
  const int nsplit = it.nsplit;
  const int gqa = a.gqa;
  const int total4 = gqa * (D / 4);
  _Float16* out_bh = a.out + (int64_t)b * a.sob + (int64_t)(kvh * gqa) * a.soh;
  if (nsplit == 0) {  // seq_len == 0: the output rows are zeros
    for (int e = threadIdx.x; e < total4; e += nw * 64) {
      const int row = e / (D / 4);
      *reinterpret_cast<h4_t*>(out_bh + (int64_t)row * a.soh + (e - row * (D / 4)) * 4) = (h4_t)0;
    }
    PAD_TL_NOTE(g, PAD_TL_F_SINGLE);
    PAD_TL(lin, PAD_TL_EXIT);
    return;
  }
  if constexpr (ENGINE == 0 && MODE == kModeUniform && !kv_is_mx4<KVF>()) {
    if (!first_known) phys_first = first_page_id(a, it.ids_row, it.ids_stride, it.col_max, it.p_begin, wave);
  }
  const int t_begin = it.p_begin * a.ps;
  const int t_end = min(it.p_end * a.ps, it.L);
  const int nblk = (t_end - t_begin + kBlockTokens - 1) / kBlockTokens;

  if constexpr (kv_is_mx4<KVF>()) {
    wave_loop_mx4<D, MODE, KVF>(a, it.ids_row, it.ids_stride, b, kvh, t_begin, t_end, nblk, wave, nw, wave, lane,
                                sm_ml, sm_o, k_stage_all + wave * k_stage_bytes<D>());
  } else if constexpr (ENGINE == 0) {
    wave_loop_mfma<D, MODE, KVF>(a, phys_first, it.ids_row, it.ids_stride, b, kvh, t_begin, t_end, nblk, wave,
                                 nw, lane, sm_ml, sm_o, k_stage_all + wave * k_stage_bytes<D>(),
                                 k_stage_all + nw * k_stage_bytes<D>());
  } else {
    wave_loop_valu<D, MODE == kModeUniform, GQA_T>(a, it.ids_row, it.ids_stride, b, kvh, t_begin, t_end, nblk, wave, nw, lane,
                                      sm_ml, sm_o);
  }
  __syncthreads();
  PAD_TL(lin, PAD_TL_LOOP_END);

  // Merge the waves' states: threads over (row, 4 consecutive d).  With a
  // single split the result is final; otherwise it is this split's partial.
  // Partials are stored and later loaded with device-scope (SC1) buffer
  // accesses, which are coherent across the XCDs' L2 caches on their own, so
  // publishing a partial needs no cache writeback.  The items of a (sequence,
  // kv head) own consecutive slots, addressed with 32-bit byte offsets.
  const int64_t seq_row0 = (int64_t)it.slot0 * gqa;
  const uint32_t region_rows = (uint32_t)(nsplit * gqa);
  const __amdgpu_buffer_rsrc_t o_rsrc = make_rsrc(a.o_part + seq_row0 * D, region_rows * D * 4u);
  const __amdgpu_buffer_rsrc_t ml_rsrc = make_rsrc(a.ml_part + seq_row0, region_rows * 8u);
  const int my_split = g - it.slot0;
  for (int e = threadIdx.x; e < total4; e += nw * 64) {
    const int row = e / (D / 4);
    const int col = (e - row * (D / 4)) * 4;
    // Unrolled over the largest wave count, so all LDS reads issue together.
    float2 ml[kMaxWaves];
    f4_t ow[kMaxWaves];
#pragma unroll
    for (int w = 0; w < kMaxWaves; ++w) {
      if (w < nw) {
        ml[w] = sm_ml[w * 16 + row];
        ow[w] = *reinterpret_cast<const f4_t*>(sm_o + (w * gqa + row) * wave_row_floats<D>() + col);
      }
    }
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < kMaxWaves; ++w)
      if (w < nw) M = fmaxf(M, ml[w].x);
    f4_t acc = (f4_t)0.f;
    float Ls = 0.f;
#pragma unroll
    for (int w = 0; w < kMaxWaves; ++w) {
      if (w < nw) {
        const float c = (ml[w].x == kNegInf) ? 0.f : exp2_fast(ml[w].x - M);
        Ls += c * ml[w].y;
        acc += c * ow[w];
      }
    }
    if (nsplit == 1) {
      // Ls >= 1: the max token contributes 2^0.  fp8 caches: V's scale too.
      const float inv = (kv_is_fp8<KVF>() ? a.v_fix : 1.f) / Ls;
      h4_t hv;
#pragma unroll
      for (int i = 0; i < 4; ++i) hv[i] = round16<KVF>(acc[i] * inv);
      *reinterpret_cast<h4_t*>(out_bh + (int64_t)row * a.soh + col) = hv;
      if constexpr (kv_weights<KVF>())
        if (col == 0) store_lse(a, b, kvh * gqa + row, M, Ls);
    } else {
      const uint32_t r = (uint32_t)(my_split * gqa + row);
      store_device(o_rsrc, (r * D + col) * 4u, acc);
      if (col == 0) store_device(ml_rsrc, r * 8u, make_float2(M, Ls));
    }
  }
  if (nsplit == 1) {
    PAD_TL(lin, PAD_TL_PUBLISHED);
    PAD_TL_NOTE(g, PAD_TL_F_SINGLE);
    PAD_TL(lin, PAD_TL_EXIT);
    return;
  }

  // Split-K merge, fused: the last workgroup of this (sequence, kv head) to
  // arrive folds every split's partial into the output.  A workgroup counts
  // itself in only after its partial stores have completed at device scope
  // (vmcnt(0) covers stores on this architecture); the last one to arrive
  // reads the partials with device-scope loads and resets the counter to
  // zero for the next launch.
  //
  // Past kTwoLevelSplits splits one workgroup reading every partial is the
  // tail (256 splits of 8 rows: 1 MB, ~17 us), so the merge takes two
  // levels: the last arrival of each group of 16 consecutive splits folds
  // the group into the slot of its first split (nothing else reads those
  // slots any more), publishes it like a partial and counts the group in;
  // the last group folds the group results.
  __shared__ int s_last;
  int* unit_counter = a.counters + (int64_t)b * a.hkv + kvh;
  int stride = 1, count = nsplit;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  PAD_TL(lin, PAD_TL_PUBLISHED);
  int tl_flags = 0;
  (void)tl_flags;
  // GQA_T == 1 marks the MFMA kernels that hold the shared fold: its registers
  // would cost the others occupancy (a d64 grid of several workgroups per CU
  // 98.4 -> 106.9 us).
  if (ENGINE == 0 && GQA_T == 1 && nsplit * total4 >= kSharedFoldElements &&
      nsplit <= max(kTwoLevelSplits, total4 / 16)) {
    // Shared fold: every workgroup of the unit folds one slice of the output,
    // where the last arrival alone would read 256 KB or more with one
    // workgroup's loads in flight (8 x 8192 tokens, 16/1 heads of 256, 32
    // splits: 10.2 us from the last arrival to the output, 4.4 us shared; the
    // call 26.0 us at its 16 splits before, 21.0 us now; 8 x 16384 of 16/1 at
    // 128 22.9 -> 19.8 us).
    //
    // counter = arrivals + departures << 16, on a line of the unit's own (its
    // group counters, which it leaves unused: with all units' polls on one
    // line the arrivals alone took 11 us).  A workgroup arrives, waits until
    // all have, departs, and folds its slice; the last to depart resets the
    // counter.  Waiting is bounded, as nothing says that all workgroups of a
    // unit run at once: one out of polls departs early, and the departures
    // that the last arrival finds tell it to fold the whole unit itself
    // (workgroups that fold their own slice as well write the same bits).
    // Without a bound of the streaming time of a split, the short last split
    // of a sequence gives up and the whole fold falls to one workgroup.
    __shared__ int s_fold;
    int* fold_counter = a.counters + (int64_t)a.batch * a.hkv + it.slot0;
    int departed = 0;
    if (threadIdx.x == 0) {
      const int before = atomicAdd(fold_counter, 1);
      int fold = 0;  // 1: own slice, 2: the whole unit
      if ((before & 0xffff) == nsplit - 1) {
        fold = before >> 16 ? 2 : 1;
      } else {
        for (int i = a.fold_polls; i > 0 && !fold; --i) {
          __builtin_amdgcn_s_sleep(8);
          fold = (__hip_atomic_load(fold_counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & 0xffff) == nsplit;
        }
      }
      if (!fold) {
        departed = atomicAdd(fold_counter, 1 << 16);
        fold = (departed & 0xffff) == nsplit ? 3 : 0;  // 3: as 1 (the last one arrived in between)
      }
      s_fold = fold;
    }
    __syncthreads();
    PAD_TL(lin, PAD_TL_ARRIVED);
    const int fold = s_fold;
    if (fold == 0) {
      PAD_TL_NOTE(g, 0);
      PAD_TL(lin, PAD_TL_EXIT);
      return;
    }
    if (threadIdx.x == 0 && fold != 3) departed = atomicAdd(fold_counter, 1 << 16);
    // An element's splits fold in runs of `cnt`, a thread each, and the runs'
    // states through LDS in order; the whole-unit fold keeps that order.
    const int nt = nw * 64;
    const int per = (total4 + nsplit - 1) / nsplit;
    int runs = min((nsplit + 3) / 4, max(1, nt / per));
    const int cnt = (nsplit + runs - 1) / runs;
    runs = (nsplit + cnt - 1) / cnt;
    const int hi = min((my_split + 1) * per, total4);
    const int span = min(per, nt / runs);
    f4_t* run_o = reinterpret_cast<f4_t*>(sm_ml);  // [runs][span], then the (m, l) pairs
    float2* run_ml = reinterpret_cast<float2*>(run_o + nt);
    for (int e0 = fold == 2 ? threadIdx.x : my_split * per; e0 < (fold == 2 ? total4 : hi); e0 += fold == 2 ? nt : span) {
      float m = kNegInf, l = 0.f;
      f4_t acc = (f4_t)0.f;
      int e = e0;
      if (fold == 2) {
        const int row = e / (D / 4);
        const int col = (e - row * (D / 4)) * 4;
        for (int r0 = 0; r0 < runs; r0 += 2) {
          MergeBatch<4> p[2];  // the first 4 entries of two runs
#pragma unroll
          for (int i = 0; i < 2; ++i)
            p[i].load_below(o_rsrc, ml_rsrc, (r0 + i) * cnt, min((r0 + i + 1) * cnt, nsplit), gqa, row, col, D);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int first = (r0 + i) * cnt;
            const int end = min(first + cnt, nsplit);
            if (first < end) {
              float mr = kNegInf, lr = 0.f;
              f4_t ar = (f4_t)0.f;
              p[i].fold_states(first, end, mr, lr, ar);
              for (int sp0 = first + 4; sp0 < end; sp0 += 4) {
                MergeBatch<4> q;
                q.load_below(o_rsrc, ml_rsrc, sp0, end, gqa, row, col, D);
                q.fold_states(sp0, end, mr, lr, ar);
              }
              fold_state(mr, lr, ar, m, l, acc);
            }
          }
        }
      } else {
        const int run = threadIdx.x / span;
        e = e0 + threadIdx.x - run * span;
        if (run < runs && e < hi) {
          const int row = e / (D / 4);
          const int col = (e - row * (D / 4)) * 4;
          fold_run(o_rsrc, ml_rsrc, run * cnt, min((run + 1) * cnt, nsplit), gqa, row, col, D, m, l, acc);
          run_o[threadIdx.x] = acc;
          run_ml[threadIdx.x] = make_float2(m, l);
        }
        __syncthreads();
        if (run > 0 || e >= hi) e = total4;
        m = kNegInf;
        l = 0.f;
        acc = (f4_t)0.f;
        if (e < total4)
          for (int r = 0; r < runs; ++r) {
            const float2 ml = run_ml[r * span + threadIdx.x];
            fold_state(ml.x, ml.y, run_o[r * span + threadIdx.x], m, l, acc);
          }
        __syncthreads();
      }
      if (e < total4) {
        const int row = e / (D / 4);
        const int col = (e - row * (D / 4)) * 4;
        const float inv = (kv_is_fp8<KVF>() ? a.v_fix : 1.f) / l;
        h4_t hv;
#pragma unroll
        for (int i = 0; i < 4; ++i) hv[i] = round16<KVF>(acc[i] * inv);
        *reinterpret_cast<h4_t*>(out_bh + (int64_t)row * a.soh + col) = hv;
      }
    }
    if (threadIdx.x == 0 && (departed >> 16) == nsplit - 1) atomicExch(fold_counter, 0);
    PAD_TL(lin, PAD_TL_MERGED);
    PAD_TL_NOTE(g, PAD_TL_F_MERGER);
    PAD_TL(lin, PAD_TL_EXIT);
    return;
  }
  if (nsplit > kTwoLevelSplits) {
    const int grp0 = my_split & ~15;  // first split of this group
    const int gsize = min(16, nsplit - grp0);
    int* group_counter = a.counters + (int64_t)a.batch * a.hkv + it.slot0 + grp0;
    if (threadIdx.x == 0) s_last = (atomicAdd(group_counter, 1) == gsize - 1);
    __syncthreads();
    if (!s_last) {
      PAD_TL(lin, PAD_TL_ARRIVED);
      PAD_TL_NOTE(g, 0);
      PAD_TL(lin, PAD_TL_EXIT);
      return;
    }
    tl_flags = PAD_TL_F_GROUP;
    // Each element's O is read and then overwritten by its own thread, but
    // a row's (m, l) is read by every thread of the row, and a row can span
    // waves and loop passes (head_dim 96: 24 elements per row): the group's
    // (m, l) goes to LDS first and to the slot only after a barrier.
    for (int e = threadIdx.x; e < total4; e += nw * 64) {
      const int row = e / (D / 4);
      const int col = (e - row * (D / 4)) * 4;
      float m = kNegInf, l = 0.f;
      f4_t acc = (f4_t)0.f;
      merge_partials(o_rsrc, ml_rsrc, grp0, gsize, 1, gqa, row, col, D, m, l, acc);
      const uint32_t r = (uint32_t)(grp0 * gqa + row);
      store_device(o_rsrc, (r * D + col) * 4u, acc);
      if (col == 0) sm_ml[row] = make_float2(m, l);
    }
    __syncthreads();
    if (threadIdx.x < gqa) store_device(ml_rsrc, (uint32_t)(grp0 * gqa + threadIdx.x) * 8u, sm_ml[threadIdx.x]);
    if (threadIdx.x == 0) atomicExch(group_counter, 0);
    stride = 16;
    count = (nsplit + 15) >> 4;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  if (threadIdx.x == 0) s_last = (atomicAdd(unit_counter, 1) == count - 1);
  __syncthreads();
  PAD_TL(lin, PAD_TL_ARRIVED);
  if (!s_last) {
    PAD_TL_NOTE(g, tl_flags);
    PAD_TL(lin, PAD_TL_EXIT);
    return;
  }
  for (int e = threadIdx.x; e < total4; e += nw * 64) {
    const int row = e / (D / 4);
    const int col = (e - row * (D / 4)) * 4;
    float m = kNegInf, l = 0.f;
    f4_t acc = (f4_t)0.f;
    merge_partials(o_rsrc, ml_rsrc, 0, count, stride, gqa, row, col, D, m, l, acc);
    const float inv = (kv_is_fp8<KVF>() ? a.v_fix : 1.f) / l;
    h4_t hv;
#pragma unroll
    for (int i = 0; i < 4; ++i) hv[i] = round16<KVF>(acc[i] * inv);
    *reinterpret_cast<h4_t*>(out_bh + (int64_t)row * a.soh + col) = hv;
    if constexpr (kv_weights<KVF>())
      if (col == 0) store_lse(a, b, kvh * gqa + row, m, l);
  }
  if (threadIdx.x == 0) atomicExch(unit_counter, 0);
  PAD_TL(lin, PAD_TL_MERGED);
  PAD_TL_NOTE(g, tl_flags | PAD_TL_F_MERGER);
  PAD_TL(lin, PAD_TL_EXIT);
#undef PAD_TL_NOTE
}

template <int D, int MODE, int ENGINE, int GQA_T, int KVF = kKvF16>
static hipError_t launch_p1(const Phase1Args& a, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if constexpr (ENGINE == 0 && GQA_T == 0 && D >= 128 && !kv_weights<KVF>())  // smaller rows never reach kSharedFoldElements
    if (a.fold_polls > 0) return launch_p1<D, MODE, 0, 1, KVF>(a, grid, nw, lds, st);
  hipLaunchKernelGGL((pad_phase1_kernel<D, MODE, ENGINE, GQA_T, KVF>), grid, dim3(nw * 64), lds, st, a);
  return hipGetLastError();
}

// Block mode from the page size (MFMA engine).
template <int D, int KVF>
static hipError_t dispatch_kvf(const Phase1Args& a, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if (a.ps % kBlockTokens == 0) return launch_p1<D, kModeUniform, 0, 0, KVF>(a, grid, nw, lds, st);
  switch (a.ps) {
    case 1: return launch_p1<D, kModeSubpage + 0, 0, 0, KVF>(a, grid, nw, lds, st);
    case 2: return launch_p1<D, kModeSubpage + 1, 0, 0, KVF>(a, grid, nw, lds, st);
    case 4: return launch_p1<D, kModeSubpage + 2, 0, 0, KVF>(a, grid, nw, lds, st);
    case 8: return launch_p1<D, kModeSubpage + 3, 0, 0, KVF>(a, grid, nw, lds, st);
    default: break;
  }
  return launch_p1<D, kModeGeneric, 0, 0, KVF>(a, grid, nw, lds, st);
}

}  // namespace pad

#endif  // PA_PHASE1_H_
