// pa_weights_fp8.hip - the per-unit decode kernel with its scores and
// normalisers written out, over fp8 caches.
#include "pa_weights.h"

namespace pad {

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

hipError_t launch_weights_fp8(const RangeArgs& a, bool range, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                              hipStream_t st) {
  switch (kvf) {
    case kKvE4M3: return launch_format<kKvE4M3 | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
    case kKvE5M2: return launch_format<kKvE5M2 | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
    case kKvE4M3B: return launch_format<kKvE4M3B | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
    case kKvE5M2B: return launch_format<kKvE5M2B | kKvWeights>(a, range, head_dim, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pad
