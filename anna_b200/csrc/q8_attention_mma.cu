// Attention over the 8-bit paged cache on tensor cores: bf16 caches, and the shapes of all.
#include "q8_attention_mma_body.cuh"

namespace anna {

template int launch_q8_mma_of<__nv_bfloat16>(const Q8Params& p, const Q8Plan& plan, int head_dim, int ctas, cudaStream_t stream);

Q8Shape q8_mma_shape(int head_dim, int rows, bool few) {
  auto of = [](auto cfg) { return Q8Shape{decltype(cfg)::kRows, decltype(cfg)::kCtas, decltype(cfg)::kWarps}; };
  using T = __nv_bfloat16;
  if (head_dim == 64) return rows <= 8 ? few ? of(Q8Cfg<T, 64, 1, 8>{}) : of(Q8Cfg<T, 64, 1, 4>{}) : rows <= 16 ? of(Q8Cfg<T, 64, 2, 4>{}) : of(Q8Cfg<T, 64, 4, 4>{});
  if (head_dim == 128)
    return rows <= 8 ? few ? of(Q8Cfg<T, 128, 1, 8>{}) : of(Q8Cfg<T, 128, 1, 4>{}) : rows <= 16 ? of(Q8Cfg<T, 128, 2, 4>{}) : of(Q8Cfg<T, 128, 4, 4>{});
  return rows <= 8 ? few ? of(Q8Cfg<T, 256, 1, 8>{}) : of(Q8Cfg<T, 256, 1, 4>{}) : of(Q8Cfg<T, 256, 2, 4>{});
}

}  // namespace anna
