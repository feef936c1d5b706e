// Tensor-core form of the multi-token decode: pages of an odd number of eights of tokens.
#include "tq_multi_mma_body.cuh"

namespace anna {

int launch_tq_multi_mma_halves(const TqMultiParams& p, int head_dim, int bits, int dtype, cudaStream_t stream) {
  return launch_pages_of<true>(p, head_dim, bits, dtype, stream);
}

int tq_multi_mma_halves_faults(int* count) { return multi_mma_faults(count); }

}  // namespace anna
