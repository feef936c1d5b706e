// Tensor-core form of the multi-token decode: pages of a multiple of 16 tokens, and the choice between the two objects (each takes a
// minute to compile).
#include "tq_multi_mma_body.cuh"

namespace anna {

int launch_tq_multi_mma_halves(const TqMultiParams& p, int head_dim, int bits, int dtype, cudaStream_t stream);
int tq_multi_mma_halves_faults(int* count);

bool tq_multi_mma_applicable(const TqMultiParams& p, int head_dim, int dtype) {
  if (dtype == ANNA_DTYPE_F32 || (head_dim != 64 && head_dim != 128 && head_dim != 256) || p.value_group != 32 || p.block_size % 8 != 0) return false;
  // the window product reads queries 16 bytes at a time
  return aligned_to(p.q, 16) && p.q_stride_b % 8 == 0 && p.q_stride_h % 8 == 0 && p.q_stride_t % 8 == 0 && p.max_len < (1ll << 30);
}

int launch_tq_multi_mma(const TqMultiParams& p, int head_dim, int bits, int dtype, cudaStream_t stream) {
  return p.block_size % kTile == 0 ? launch_pages_of<false>(p, head_dim, bits, dtype, stream)
                                   : launch_tq_multi_mma_halves(p, head_dim, bits, dtype, stream);
}

int tq_multi_mma_faults(int* count) {
  int halves = 0;
  const int rc = tq_multi_mma_halves_faults(&halves);
  if (rc != ANNA_OK) return rc;
  const int rc_whole = multi_mma_faults(count);
  *count += halves;
  return rc_whole;
}

}  // namespace anna
