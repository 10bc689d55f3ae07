// pa_weights.h - the decode kernels with their scores and normalisers written
// out (kKvWeights), for pa_weights.hip and pa_weights_fp8.hip.
#ifndef PA_WEIGHTS_H_
#define PA_WEIGHTS_H_

#include "pa_ext.h"
#include "pa_phase1.h"
#include "pa_range_kernel.h"

namespace pad {

template <int D, int MODE, int KVF>
__global__ __launch_bounds__((range_waves<D, KVF>() * 64))
    __attribute__((amdgpu_waves_per_eu((range_waves<D, KVF>() / 4)))) void pad_weights_range_kernel(const RangeArgs) {
  range_kernel<D, MODE, KVF>();
}

template <int D, int MODE, int KVF>
static hipError_t launch_one(const RangeArgs& a, bool range, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if (!range) return launch_p1<D, MODE, 0, 0, KVF>(a, grid, nw, lds, st);
  hipLaunchKernelGGL((pad_weights_range_kernel<D, MODE, KVF>), dim3(a.groups), dim3(nw * 64), lds, st, a);
  return hipGetLastError();
}

template <int D, int KVF>
static hipError_t launch_dim(const RangeArgs& a, bool range, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if (a.ps % kBlockTokens == 0) return launch_one<D, kModeUniform, KVF>(a, range, grid, nw, lds, st);
  switch (a.ps) {
    case 1: return launch_one<D, kModeSubpage + 0, KVF>(a, range, grid, nw, lds, st);
    case 2: return launch_one<D, kModeSubpage + 1, KVF>(a, range, grid, nw, lds, st);
    case 4: return launch_one<D, kModeSubpage + 2, KVF>(a, range, grid, nw, lds, st);
    case 8: return launch_one<D, kModeSubpage + 3, KVF>(a, range, grid, nw, lds, st);
    default: return launch_one<D, kModeGeneric, KVF>(a, range, grid, nw, lds, st);
  }
}

}  // namespace pad

#endif  // PA_WEIGHTS_H_
