// pa_weights.hip - the per-unit decode kernel with its scores and normalisers
// written out, over 16-bit caches.
#include "pa_weights.h"

namespace pad {

template <int KVF>
static hipError_t launch_format(const RangeArgs& a, bool range, int head_dim, dim3 grid, int nw, size_t lds,
                                hipStream_t st) {
  switch (head_dim) {
    case 32: return launch_dim<32, KVF>(a, range, grid, nw, lds, st);
    case 64: return launch_dim<64, KVF>(a, range, grid, nw, lds, st);
    case 96: return launch_dim<96, KVF>(a, range, grid, nw, lds, st);
    case 128: return launch_dim<128, KVF>(a, range, grid, nw, lds, st);
    case 256: return launch_dim<256, KVF>(a, range, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_weights(const RangeArgs& a, bool range, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                          hipStream_t st) {
  if (kvf == kKvBF16) return launch_format<kKvBF16 | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
  if (kvf == kKvF16) return launch_format<kKvF16 | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
  return hipErrorInvalidValue;
}

}  // namespace pad
