// Attention over the 8-bit paged cache on tensor cores: fp32 caches.
#include "q8_attention_mma_body.cuh"

namespace anna {

template int launch_q8_mma_of<float>(const Q8Params& p, const Q8Plan& plan, int head_dim, int ctas, cudaStream_t stream);

}  // namespace anna
