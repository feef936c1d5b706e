// Parameters and the merge of the multi-token decode over packed TurboQuant pages (tq_multi_decode.cu, tq_multi_mma.cu).
//
// The newest T tokens of a sequence are its queries; query t sees the keys at positions up to len - T + t.  The T * G queries that
// share a KV head are the rows of one product (row r = t * G + g), cut into row tiles; the keys [0, len) are cut into chunks.  A
// CTA takes one (chunk, KV head and row tile, sequence), leaves the rows' partial softmax, and the CTA of a (sequence, row tile)
// that arrives last merges them.
#pragma once

#include "fused_combine.cuh"
#include "tq_common.cuh"

namespace anna {

struct TqMultiParams {
  const void* q;
  int64_t q_stride_b, q_stride_h, q_stride_t;
  const uint8_t* pages;
  const int32_t* block_table;
  int64_t table_stride;
  const void* window;
  const int64_t* window_slots;
  const int64_t* lengths;
  const float* signs1;
  const float* signs2;
  const float* centroids;
  const void* gate;
  int64_t gate_stride_b, gate_stride_h, gate_stride_t;
  void* out;
  int64_t out_stride_b, out_stride_h, out_stride_t;
  float* stats;      // [B, Hkv, T * G, chunks, 2]: running maximum (natural units), denominator
  float* values;     // [B, Hkv, T * G, chunks, D]
  int32_t* counters;  // [B, Hkv, row tiles]
  int q_heads, kv_heads, groups, tokens, rows;  // rows = tokens * groups
  int block_size, block_shift, residual_len, value_group;
  int64_t num_pages, max_blocks, max_len;
  int chunk_tokens, num_chunks;
  float scaling;
  anna_tq_layout layout;
};

// One output row, from its dims d .. d + N - 1.
template <typename T, int N>
__device__ __forceinline__ void multi_store(const TqMultiParams& p, int64_t b, int kvh, int row, int d, const float (&o)[N]) {
  const int t = row / p.groups, h = kvh * p.groups + row % p.groups;
  T* out = reinterpret_cast<T*>(p.out) + b * p.out_stride_b + h * p.out_stride_h + t * p.out_stride_t + d;
  const T* gate = p.gate == nullptr
                      ? nullptr
                      : reinterpret_cast<const T*>(p.gate) + b * p.gate_stride_b + h * p.gate_stride_h + t * p.gate_stride_t + d;
#pragma unroll
  for (int i = 0; i < N; ++i)
    out[i] = ElemTraits<T>::from_float(gate != nullptr ? o[i] / (1.0f + __expf(-ElemTraits<T>::to_float(gate[i]))) : o[i]);
}

__device__ __forceinline__ int64_t multi_row_index(const TqMultiParams& p, int64_t b, int kvh, int row) {
  return (b * p.kv_heads + kvh) * p.rows + row;
}

// Merges the partials of rows [row0, row0 + count) when this CTA is the last of `chunks` to get here.  A warp per row, a lane holds
// D / 32 dims.
template <typename T, int D, int WARPS>
__device__ __forceinline__ void multi_merge(const TqMultiParams& p, int64_t b, int kvh, int tile, int tiles, int row0, int count, int chunks) {
  if (!merge_arrive(FusedCombine{p.counters}, (b * p.kv_heads + kvh) * tiles + tile, chunks)) return;
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < count; i += WARPS) {
    const int64_t at = multi_row_index(p, b, kvh, row0 + i) * p.num_chunks;
    const float2* stats = reinterpret_cast<const float2*>(p.stats) + at;
    const float* values = p.values + at * D + lane * N;
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 32) m = fmaxf(m, __ldcg(stats + c).x);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float m_ref = m == -INFINITY ? 0.0f : m;
    float den = 0.0f, acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.0f;
    for (int c0 = 0; c0 < chunks; c0 += 32) {
      float w = 0.0f;
      if (c0 + lane < chunks) {
        const float2 s = __ldcg(stats + c0 + lane);
        w = __expf(s.x - m_ref);
        den += w * s.y;
      }
      const int here = min(32, chunks - c0);
#pragma unroll 4
      for (int c = 0; c < here; ++c) {
        const float wc = __shfl_sync(0xffffffffu, w, c);
        const float* v = values + (int64_t)(c0 + c) * D;
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(v + j));
          acc[j] = fmaf(x.x, wc, acc[j]);
          acc[j + 1] = fmaf(x.y, wc, acc[j + 1]);
        }
      }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) den += __shfl_xor_sync(0xffffffffu, den, d);
    // a NaN among the scores has to stay one, so only an empty row is zero
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] *= inv;
    multi_store<T, N>(p, b, kvh, row0 + i, lane * N, acc);
  }
}

// Tensor-core form (tq_multi_mma.cu): 16-bit caches, head_dim 128 / 256, value groups of 32, pages of a multiple of 16 tokens.
bool tq_multi_mma_applicable(const TqMultiParams& p, int batch, int head_dim, int bits, int dtype);
int launch_tq_multi_mma(const TqMultiParams& p, int batch, int head_dim, int bits, int dtype, cudaStream_t stream);

}  // namespace anna
