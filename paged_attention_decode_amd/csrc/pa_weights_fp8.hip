// pa_weights_fp8.hip - the per-unit decode kernel with its scores and
// normalisers written out, over fp8 caches.
#include "pa_ext.h"
#include "pa_phase1.h"

namespace pad {

template <int KVF>
static hipError_t launch_format(const Phase1Args& a, int head_dim, dim3 grid, int nw, size_t lds, hipStream_t st) {
  switch (head_dim) {
    case 64: return dispatch_kvf<64, KVF>(a, grid, nw, lds, st);
    case 128: return dispatch_kvf<128, KVF>(a, grid, nw, lds, st);
    case 256: return dispatch_kvf<256, KVF>(a, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_weights_fp8(const Phase1Args& a, int head_dim, int kvf, dim3 grid, int nw, size_t lds,
                              hipStream_t st) {
  switch (kvf) {
    case kKvE4M3: return launch_format<kKvE4M3 | kKvWeights>(a, head_dim, grid, nw, lds, st);
    case kKvE5M2: return launch_format<kKvE5M2 | kKvWeights>(a, head_dim, grid, nw, lds, st);
    case kKvE4M3B: return launch_format<kKvE4M3B | kKvWeights>(a, head_dim, grid, nw, lds, st);
    case kKvE5M2B: return launch_format<kKvE5M2B | kKvWeights>(a, head_dim, grid, nw, lds, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pad
