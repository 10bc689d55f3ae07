// pa_mx4.hip - the decode kernels over MX4 caches (pa_mx4.h).
#include "pa_ext.h"
#include "pa_phase1.h"
#include "pa_range_kernel.h"

namespace pad {

template <int D, int MODE, int KVF>
__global__ __launch_bounds__((range_waves<D, KVF>() * 64))
    __attribute__((amdgpu_waves_per_eu((range_waves<D, KVF>() / 4)))) void pad_mx4_range_kernel(const RangeArgs) {
  range_kernel<D, MODE, KVF>();
}

template <int D, int MODE, int KVF>
static hipError_t launch_one(const RangeArgs& a, bool range, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if (!range) return launch_p1<D, MODE, 0, 0, KVF>(a, grid, nw, lds, st);
  hipLaunchKernelGGL((pad_mx4_range_kernel<D, MODE, KVF>), dim3(a.groups), dim3(nw * 64), lds, st, a);
  return hipGetLastError();
}

// Uniform mode is for blocks whose rows lie next to each other: it streams them
// (non-temporal loads).  Rows of several kv heads in one cache line are loaded
// by each lane's own address and kept in the CU's cache, where the other heads'
// waves find the rest of the line.  us, streamed / kept: heads next to each other
// 64 x [1, 8192] of 32/8 89.4 / 85.3, 27 x [1, 4096] of 32/8 at head_dim 64, page
// 1, 34.1 / 24.6; rows next to each other 56.3 / 63.1, 1 x 131072 31.1 / 34.0.
template <int D, int KVF>
static hipError_t launch_dim(const RangeArgs& a, bool range, dim3 grid, int nw, size_t lds, hipStream_t st) {
  const bool rows = a.sks == D / 2 && a.svs == D / 2 && (a.skss | a.svss) < (1 << 26);
  if (a.ps % kBlockTokens == 0 && rows)
    return launch_one<D, kModeUniform, KVF>(a, range, grid, nw, lds, st);
  return launch_one<D, kModeGeneric, KVF>(a, range, grid, nw, lds, st);
}

template <int KVF>
static hipError_t launch_format(const RangeArgs& a, bool range, int head_dim, dim3 grid, int nw, size_t lds,
                                hipStream_t st) {
  switch (head_dim) {
    case 64: return launch_dim<64, KVF>(a, range, grid, nw, lds, st);
    case 128: return launch_dim<128, KVF>(a, range, grid, nw, lds, st);
    case 256: return launch_dim<256, KVF>(a, range, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_mx4(const RangeArgs& a, bool range, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                      hipStream_t st) {
  switch (kvf) {
    case kKvMx4: return launch_format<kKvMx4>(a, range, head_dim, grid, nw, lds, st);
    case kKvMx4B: return launch_format<kKvMx4B>(a, range, head_dim, grid, nw, lds, st);
    case kKvMx4 | kKvWeights: return launch_format<kKvMx4 | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
    case kKvMx4B | kKvWeights: return launch_format<kKvMx4B | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pad
