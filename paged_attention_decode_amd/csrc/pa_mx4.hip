// pa_mx4.hip - the per-unit decode kernel over MX4 caches (pa_mx4.h).
#include "pa_ext.h"
#include "pa_phase1.h"

namespace pad {

template <int D, int KVF>
static hipError_t launch_dim(const Phase1Args& a, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if (a.ps % kBlockTokens == 0) return launch_p1<D, kModeUniform, 0, 0, KVF>(a, grid, nw, lds, st);
  return launch_p1<D, kModeGeneric, 0, 0, KVF>(a, grid, nw, lds, st);
}

template <int KVF>
static hipError_t launch_format(const Phase1Args& a, int head_dim, dim3 grid, int nw, size_t lds, hipStream_t st) {
  switch (head_dim) {
    case 64: return launch_dim<64, KVF>(a, grid, nw, lds, st);
    case 128: return launch_dim<128, KVF>(a, grid, nw, lds, st);
    case 256: return launch_dim<256, KVF>(a, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_mx4(const Phase1Args& a, int head_dim, int kvf, dim3 grid, int nw, size_t lds, hipStream_t st) {
  switch (kvf) {
    case kKvMx4: return launch_format<kKvMx4>(a, head_dim, grid, nw, lds, st);
    case kKvMx4B: return launch_format<kKvMx4B>(a, head_dim, grid, nw, lds, st);
    case kKvMx4 | kKvWeights: return launch_format<kKvMx4 | kKvWeights>(a, head_dim, grid, nw, lds, st);
    case kKvMx4B | kKvWeights: return launch_format<kKvMx4B | kKvWeights>(a, head_dim, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pad
