// pa_range.hip - the decode over equal page ranges (pa_range_kernel.h) over
// 16-bit and fp8 caches, and its work-list planner.

#include "pa_range_kernel.h"

namespace pad {

template <int D, int MODE, int KVF>
__global__ __launch_bounds__((range_waves<D, KVF>() * 64))
    __attribute__((amdgpu_waves_per_eu((range_waves<D, KVF>() / 4)))) void pad_range_kernel(const RangeArgs) {
  range_kernel<D, MODE, KVF>();
}

// Work-list planner: one wave per workgroup of the decode grid; lane i < 32
// writes word i of its record.
template <int NK>
__device__ __forceinline__ void write_record(const RangeArgs& a, int32_t* wl) {
  const int g = blockIdx.x;
  const int lane = threadIdx.x;
  uint64_t zeros = 0;
  int own[2] = {-1, -1};  // owners of sequences 2g, 2g + 1
  const RangePlan p = plan_ranges<NK>(a, g, lane, [&](int b, int owner) {
    zeros |= __builtin_amdgcn_ballot_w64(owner == g);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint64_t at = __builtin_amdgcn_ballot_w64(b == 2 * g + j);
      if (at != 0) own[j] = __builtin_amdgcn_readlane(owner, (int)__builtin_ctzll(at));
    }
  });
  const Unit& u = p.first;
  const int lo = g * p.T, hi = min(lo + p.T, p.P);
  const bool valid = lo < hi;
  const int begin = max(lo - u.start - p.E, 0);  // first page of the first segment
  int v = 0;
  switch (lane) {
    case 0: v = u.b; break;
    case 1: v = u.kvh; break;
    case 4: v = u.len; break;
    case 7: v = u.pages - 1; break;
    case 8: v = valid ? 1 : 0; break;
    case 9: v = u.row; break;
    case 10: v = u.start; break;
    case 11: v = p.T; break;
    case 12: v = p.P; break;
    case 14: v = p.E; break;
    default: break;
  }
  if (!valid) v = 0;
  if (lane == 13) v = zeros != 0 ? 1 : 0;
  if (lane >= 16 && lane < 24 && valid && a.ps % kBlockTokens == 0) {
    const int col = min(begin + block_page(a, lane - 16), u.pages - 1);
    v = a.csr ? a.bt[u.row + col] : a.bt[(int64_t)u.b * a.sbb + (int64_t)col * a.sbp];
  }
  int32_t* r = wl + kRlHeaderInts + (int64_t)kRlRecordInts * g;
  if (lane < 24) r[lane] = v;
  // Sequences 2g and 2g + 1, from the lanes and registers that hold them.
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int b = 2 * g + j;
    int pages = 0, len = 0, row = 0;
    if (b < a.batch) sequence_info(a, b, &pages, &len, &row);
    const int w = lane - 24 - 4 * j;
    if (w >= 0 && w < 4) r[lane] = w == 0 ? pages : (w == 1 ? len : (w == 2 ? row : own[j]));
  }
  if (g == 0 && lane < kRlHeaderInts)
    wl[lane] = lane == 0 ? kRlMagic : (lane == 1 ? a.wl_key : (lane == 2 ? a.groups : 0));
}

__global__ __launch_bounds__(64) void pad_range_plan_kernel(const RangeArgs a, int32_t* wl) {
  if (a.batch <= 64)
    write_record<1>(a, wl);
  else
    write_record<4>(a, wl);
}

hipError_t launch_range_plan(const RangeArgs& a, int32_t* wl, hipStream_t st) {
  hipLaunchKernelGGL(pad_range_plan_kernel, dim3(a.groups), dim3(64), 0, st, a, wl);
  return hipGetLastError();
}

template <int D, int MODE, int KVF>
static hipError_t launch_one(const RangeArgs& a, int nw, size_t lds, hipStream_t st) {
  hipLaunchKernelGGL((pad_range_kernel<D, MODE, KVF>), dim3(a.groups), dim3(nw * 64), lds, st, a);
  return hipGetLastError();
}

template <int D, int KVF>
static hipError_t launch_mode(const RangeArgs& a, int nw, size_t lds, hipStream_t st) {
  if (a.ps % kBlockTokens == 0) return launch_one<D, kModeUniform, KVF>(a, nw, lds, st);
  switch (a.ps) {
    case 1: return launch_one<D, kModeSubpage + 0, KVF>(a, nw, lds, st);
    case 2: return launch_one<D, kModeSubpage + 1, KVF>(a, nw, lds, st);
    case 4: return launch_one<D, kModeSubpage + 2, KVF>(a, nw, lds, st);
    case 8: return launch_one<D, kModeSubpage + 3, KVF>(a, nw, lds, st);
    default: return launch_one<D, kModeGeneric, KVF>(a, nw, lds, st);
  }
}

template <int KVF>
static hipError_t launch_dim(const RangeArgs& a, int head_dim, int nw, size_t lds, hipStream_t st) {
  switch (head_dim) {
    case 64: return launch_mode<64, KVF>(a, nw, lds, st);
    case 128: return launch_mode<128, KVF>(a, nw, lds, st);
    case 256: return launch_mode<256, KVF>(a, nw, lds, st);
    default: break;
  }
  if constexpr (!kv_is_fp8<KVF>()) {
    if (head_dim == 32) return launch_mode<32, KVF>(a, nw, lds, st);
    if (head_dim == 96) return launch_mode<96, KVF>(a, nw, lds, st);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_range(const RangeArgs& a, int head_dim, int kvf, int nw, size_t lds, hipStream_t st) {
  switch (kvf) {
    case kKvF16: return launch_dim<kKvF16>(a, head_dim, nw, lds, st);
    case kKvE4M3: return launch_dim<kKvE4M3>(a, head_dim, nw, lds, st);
    case kKvE5M2: return launch_dim<kKvE5M2>(a, head_dim, nw, lds, st);
    case kKvBF16: return launch_dim<kKvBF16>(a, head_dim, nw, lds, st);
    case kKvE4M3B: return launch_dim<kKvE4M3B>(a, head_dim, nw, lds, st);
    case kKvE5M2B: return launch_dim<kKvE5M2B>(a, head_dim, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pad
