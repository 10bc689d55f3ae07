// pa_weights.hip - the per-unit decode kernel with its scores and normalisers
// written out, over 16-bit caches.
#include "pa_ext.h"
#include "pa_phase1.h"

namespace pad {

template <int KVF>
static hipError_t launch_format(const Phase1Args& a, int head_dim, dim3 grid, int nw, size_t lds, hipStream_t st) {
  switch (head_dim) {
    case 32: return dispatch_kvf<32, KVF>(a, grid, nw, lds, st);
    case 64: return dispatch_kvf<64, KVF>(a, grid, nw, lds, st);
    case 96: return dispatch_kvf<96, KVF>(a, grid, nw, lds, st);
    case 128: return dispatch_kvf<128, KVF>(a, grid, nw, lds, st);
    case 256: return dispatch_kvf<256, KVF>(a, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_weights(const Phase1Args& a, int head_dim, int kvf, dim3 grid, int nw, size_t lds, hipStream_t st) {
  if (kvf == kKvBF16) return launch_format<kKvBF16 | kKvWeights>(a, head_dim, grid, nw, lds, st);
  if (kvf == kKvF16) return launch_format<kKvF16 | kKvWeights>(a, head_dim, grid, nw, lds, st);
  return hipErrorInvalidValue;
}

}  // namespace pad
