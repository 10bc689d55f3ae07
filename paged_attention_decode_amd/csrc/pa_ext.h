// pa_ext.h - launchers of the decode kernels' other instantiations, used by the
// launch path in pa_decode.hip.
#ifndef PA_EXT_H_
#define PA_EXT_H_

#include "pa_range.h"

namespace pad {

// Decode over MX4 caches (head_dim 64, 128 or 256); kvf: kKvMx4 or kKvMx4B,
// plus kKvWeights.  range: the range kernel (grid unused), else the per-unit one.
hipError_t launch_mx4(const RangeArgs& a, bool range, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                      hipStream_t st);

// Decode that also writes its scores and normalisers; kvf: a 16-bit
// (pa_weights.hip) or fp8 (pa_weights_fp8.hip) format, without kKvWeights.
hipError_t launch_weights(const RangeArgs& a, bool range, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                          hipStream_t st);
hipError_t launch_weights_fp8(const RangeArgs& a, bool range, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                              hipStream_t st);

// weights += the weights of p's launch (its logits and lse, dense page index).
hipError_t launch_accumulate(const Phase1Args& p, float* weights, const int64_t* w_stride, hipStream_t st);

}  // namespace pad

#endif  // PA_EXT_H_
