// Attention of the newest T tokens of every sequence over [packed TurboQuant prefix | un-quantized window ring]: the CUDA-core
// form and the entry points.
//
// Keys are scored in the basis of their codes, as in the single-token decode (tq_decode.cu):
//   q . k_hat = norm / D * [ fwht(s1*q) . centroid[idx] + sqrt(pi/2)/sqrt(D) * rnorm * fwht(s2*fwht(s1*q)) . (2*sign-1) ]
// so a CTA rotates its rows once and no key is taken back to the original basis.
//
// This form serves fp32 caches, pages that are no multiple of 8 tokens and value groups other than 32; everything in it is 32 bits.  A
// CTA de-quantizes 32 tokens at a time into shared memory for its 8 rows; a warp scores two rows (256 dims: one) with a token a lane.
// Bound: issue, of which the reads of shared memory are as many as the FMAs.  A lane takes neighbouring dims, so that its codes are one
// load instead of one a dim: 8 fp32 rows of 20-3000 tokens, 20 queries to a KV head of 128 dims 181 -> 106 us, 256 dims (with 256 threads
// instead of 128, too) 727 -> 240, 64 dims 96 -> 72.
#include "tq_multi_params.cuh"

namespace anna {

template <int D>
constexpr int kMultiThreads = D == 256 ? 256 : 128;  // shared memory holds one CTA of 256 dims per SM
constexpr int kMultiRows = 8;    // of a CTA of this form
constexpr int kMultiTokens = 32;  // de-quantized at a time: a lane's token
constexpr int kMultiAhead = 4;    // tokens of a warp whose codes are on their way together

// This lane's NB bits of a run of codes.
template <int NB>
__device__ __forceinline__ uint32_t lane_bits(const uint8_t* codes, int lane) {
  if constexpr (NB == 32) return reinterpret_cast<const uint32_t*>(codes)[lane];
  else if constexpr (NB == 16) return reinterpret_cast<const uint16_t*>(codes)[lane];
  else if constexpr (NB == 8) return codes[lane];
  else return (uint32_t)codes[lane * NB / 8] >> (lane * NB % 8);
}

template <int D>
constexpr int kMultiSmemFloats = 3 * kMultiRows * D + 2 * kMultiTokens * (D + 1) + kMultiTokens * D + kMultiRows * kMultiTokens;

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(kMultiThreads<D>) tq_multi_kernel(const TqMultiParams p, int row_tiles) {
  constexpr int E = D / 32, kThreads = kMultiThreads<D>, kMultiWarps = kThreads / 32, kWarpRows = kMultiRows / kMultiWarps;
  constexpr int M = BITS - 1;
  constexpr int VS = BITS == 2 ? 2 : 4;
  extern __shared__ __align__(16) float smem[];
  // Rows of D are held in an order of their own, dim lane * E + j at j * 32 + lane: a lane takes neighbouring dims, whose codes are one
  // access, and neighbouring lanes write neighbouring floats.
  float* q_smem = smem;                                // [3][rows][D]: as it is, rotated, rotated twice; scaled
  float* ka = q_smem + 3 * kMultiRows * D;             // [tokens][D + 1]: centroids, or the key itself
  float* kb = ka + kMultiTokens * (D + 1);             // signs times the residual norm
  float* vt = kb + kMultiTokens * (D + 1);             // [tokens][D]
  float* weight = vt + kMultiTokens * D;               // [rows][tokens]
  __shared__ float sm_cent[1 << M], sm_norm[kMultiTokens], sm_rescale[kMultiRows];
  __shared__ bool sm_there[kMultiTokens];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < (1 << M)) sm_cent[threadIdx.x] = p.centroids[threadIdx.x];
  multi_for_each_segment<T, D, kThreads>(p, row_tiles, [&](int64_t b, int kvh, int tile, int64_t t0, int64_t t1, const MultiPartial& part) {
  const int row0 = tile * kMultiRows, count = min(kMultiRows, p.rows - row0);
  const int64_t len = max((int64_t)0, min(p.lengths[b], p.max_len));
  const int64_t lq = len > p.residual_len ? len - p.residual_len : 0;
  const int64_t first_seen = len - p.tokens;  // newest key that query 0 sees

  const float f1 = p.scaling / (float)D;
  const float f2 = f1 * 1.2533141373155001f * rsqrt_dim_const<D>();
  for (int i = warp; i < kMultiRows; i += kMultiWarps) {
    if (i >= count) break;  // rows that are not there: their scores are not looked at
    float w[E];
    const int row = row0 + i;
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_stride_b + (int64_t)(kvh * p.groups + row % p.groups) * p.q_stride_h +
                 (int64_t)(row / p.groups) * p.q_stride_t + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = ElemTraits<T>::to_float(q[j]);
      q_smem[i * D + j * 32 + lane] = w[j] * p.scaling;
      w[j] *= p.signs1[lane * E + j];
    }
    warp_fwht<E>(w, lane);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      q_smem[(kMultiRows + i) * D + j * 32 + lane] = w[j] * f1;
      w[j] *= p.signs2[lane * E + j];
    }
    warp_fwht<E>(w, lane);
#pragma unroll
    for (int j = 0; j < E; ++j) q_smem[(2 * kMultiRows + i) * D + j * 32 + lane] = w[j] * f2;
  }

  // every kMultiWarps-th row from `warp` on is of this warp's softmax; the thread's rows of one dim of the output
  float m_run[kWarpRows], l_run[kWarpRows];
#pragma unroll
  for (int k = 0; k < kWarpRows; ++k) {
    m_run[k] = -INFINITY;
    l_run[k] = 0.0f;
  }
  static_assert(D <= kThreads && kThreads % D == 0, "a thread has one dim");
  constexpr int kOutRows = kMultiRows * D / kThreads;
  const int out_row0 = (int)threadIdx.x / D * kOutRows, place = (int)threadIdx.x % D, out_dim = place % 32 * E + place / 32;
  float acc[kOutRows];
#pragma unroll
  for (int r = 0; r < kOutRows; ++r) acc[r] = 0.0f;
  int group[E];
#pragma unroll
  for (int j = 0; j < E; ++j) group[j] = (lane * E + j) / p.value_group;
  const bool one_group = p.value_group % E == 0;

  const int64_t slot = len > lq ? p.window_slots[b] : 0;
  const T* ring = reinterpret_cast<const T*>(p.window) + (slot * 2 * p.kv_heads + kvh) * p.residual_len * D;
  const int64_t ring_values = (int64_t)p.kv_heads * p.residual_len * D;
  for (int64_t base = t0; base < t1;) {
    const bool packed = base < lq;
    const int64_t stop = min(packed ? min(lq, t1) : t1, base + kMultiTokens);
    const int n = (int)(stop - base);
    __syncthreads();
    // ---- 32 tokens into shared memory -----------------------------------------------------------------------------------------
    // A lane finds the page of its token; then a warp takes a token at a time, whose codes are on their way for several at once.
    int64_t chunk = -1;  // of this lane's token, in bytes
    int in_page = 0;
    if (packed && lane < n) {
      const int64_t t = base + lane, blk = t / p.block_size;
      in_page = (int)(t - blk * p.block_size);
      const int32_t pid = blk < p.max_blocks ? p.block_table[b * p.table_stride + blk] : -1;
      if (pid >= 0 && pid < p.num_pages) chunk = ((int64_t)pid * p.kv_heads + kvh) * p.layout.chunk_bytes;
      if (warp == 0) {
        sm_there[lane] = chunk >= 0;
        sm_norm[lane] = chunk >= 0 ? reinterpret_cast<const float*>(p.pages + chunk + p.layout.off_knorm)[in_page] : 0.0f;
      }
    }
    if (!packed && warp == 0 && lane < n) {
      sm_there[lane] = true;
      sm_norm[lane] = 1.0f;
    }
    for (int i = warp; i < n; i += kMultiWarps * kMultiAhead) {
      if (!packed) {
        float k[kMultiAhead][E], v[kMultiAhead][E];
#pragma unroll
        for (int u = 0; u < kMultiAhead; ++u) {
          const T* key = ring + ((base + min(i + u * kMultiWarps, n - 1)) % p.residual_len) * D + lane * E;
          lane_load<T, E>(key, k[u]);
          lane_load<T, E>(key + ring_values, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kMultiAhead; ++u) {
          const int at = i + u * kMultiWarps;
          if (at >= n) break;
#pragma unroll
          for (int j = 0; j < E; ++j) {
            ka[at * (D + 1) + j * 32 + lane] = k[u][j];
            vt[at * D + j * 32 + lane] = v[u][j];
          }
        }
        continue;
      }
      constexpr int kIndexBits = BITS == 3 ? 2 * E : BITS * E;
      uint32_t code[kMultiAhead], sign[kMultiAhead], value[kMultiAhead];
      T scale[kMultiAhead][E], zero[kMultiAhead][E];
      float rnorm[kMultiAhead];
#pragma unroll
      for (int u = 0; u < kMultiAhead; ++u) {
        const int at = min(i + u * kMultiWarps, n - 1);
        const int64_t where = __shfl_sync(0xffffffffu, chunk, at);
        const int tok = __shfl_sync(0xffffffffu, in_page, at);
        const bool there = where >= 0;
        const uint8_t* page = p.pages + (there ? where : 0);
        const uint8_t* keys = page + p.layout.off_kcodes + tok * p.layout.key_bytes;
        const uint8_t* codes = page + p.layout.off_vdata + tok * p.layout.value_bytes;
        const T* scales = reinterpret_cast<const T*>(page + p.layout.off_vscale) + tok * p.layout.groups;
        const T* zeros = reinterpret_cast<const T*>(page + p.layout.off_vzero) + tok * p.layout.groups;
        rnorm[u] = there ? reinterpret_cast<const float*>(page + p.layout.off_krnorm)[tok] : 0.0f;
        code[u] = there ? lane_bits<kIndexBits>(keys, lane) : 0u;
        sign[u] = BITS == 3 && there ? lane_bits<E>(keys + D / 4, lane) : 0u;
        value[u] = there ? lane_bits<VS * E>(codes, lane) : 0u;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          if (j > 0 && one_group) {
            scale[u][j] = scale[u][0];
            zero[u][j] = zero[u][0];
          } else {
            scale[u][j] = there ? scales[group[j]] : T(0.0f);
            zero[u][j] = there ? zeros[group[j]] : T(0.0f);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kMultiAhead; ++u) {
        const int at = i + u * kMultiWarps;
        if (at >= n) break;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          uint32_t index, negative;
          if constexpr (BITS == 3) {
            index = (code[u] >> (2 * j)) & 3u;
            negative = ((sign[u] >> j) & 1u) ^ 1u;
          } else {
            const uint32_t field = (code[u] >> (BITS * j)) & ((1u << BITS) - 1u);
            index = field & ((1u << M) - 1u);
            negative = (field >> M) ^ 1u;
          }
          ka[at * (D + 1) + j * 32 + lane] = sm_cent[index];
          kb[at * (D + 1) + j * 32 + lane] = negative != 0 ? -rnorm[u] : rnorm[u];
          vt[at * D + j * 32 + lane] = fmaf((float)((value[u] >> (VS * j)) & ((1u << VS) - 1u)), ElemTraits<T>::to_float(scale[u][j]),
                                            ElemTraits<T>::to_float(zero[u][j]));
        }
      }
    }
    __syncthreads();
    // ---- scores: token `lane` --------------------------------------------------------------------------------------------------
    float s[kWarpRows];
#pragma unroll
    for (int k = 0; k < kWarpRows; ++k) s[k] = -INFINITY;
    if (lane < n) {
      float a[kWarpRows];
      auto product = [&](const float* q, const float* x) {
        float sum[kWarpRows];
#pragma unroll
        for (int k = 0; k < kWarpRows; ++k) sum[k] = 0.0f;
#pragma unroll 16
        for (int d = 0; d < D; ++d)
#pragma unroll
          for (int k = 0; k < kWarpRows; ++k) sum[k] = fmaf(q[k * kMultiWarps * D + d], x[d], sum[k]);
#pragma unroll
        for (int k = 0; k < kWarpRows; ++k) a[k] += sum[k];
      };
#pragma unroll
      for (int k = 0; k < kWarpRows; ++k) a[k] = 0.0f;
      product(q_smem + ((packed ? kMultiRows : 0) + warp) * D, ka + lane * (D + 1));
      if (packed) product(q_smem + (2 * kMultiRows + warp) * D, kb + lane * (D + 1));
#pragma unroll
      for (int k = 0; k < kWarpRows; ++k) {
        const int i = warp + k * kMultiWarps;
        if (i < count && sm_there[lane] && base + lane <= first_seen + (row0 + i) / p.groups) s[k] = a[k] * sm_norm[lane];
      }
    }
#pragma unroll
    for (int k = 0; k < kWarpRows; ++k) {
      float m_new = s[k];
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, d));
      m_new = fmaxf(m_run[k], m_new);
      const float m_safe = m_new == -INFINITY ? 0.0f : m_new;
      const float w = __expf(s[k] - m_safe), rescale = __expf(m_run[k] - m_safe);
      l_run[k] = l_run[k] * rescale + w;  // a lane's share of the sum
      m_run[k] = m_new;
      weight[(warp + k * kMultiWarps) * kMultiTokens + lane] = w;
      if (lane == 0) sm_rescale[warp + k * kMultiWarps] = rescale;
    }
    __syncthreads();
    // ---- values -----------------------------------------------------------------------------------------------------------
#pragma unroll
    for (int r = 0; r < kOutRows; ++r) acc[r] *= sm_rescale[out_row0 + r];
    int i = 0;
    if (base + n - 1 <= first_seen) {  // every row sees every token
      for (; i + 4 <= n; i += 4) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = vt[(i + u) * D + place];
#pragma unroll
        for (int r = 0; r < kOutRows; ++r) {
          const float4 w = *reinterpret_cast<const float4*>(weight + (out_row0 + r) * kMultiTokens + i);
          acc[r] = fmaf(w.w, v[3], fmaf(w.z, v[2], fmaf(w.y, v[1], fmaf(w.x, v[0], acc[r]))));
        }
      }
    }
    for (; i < n; ++i) {
      const float v = vt[i * D + place];
#pragma unroll
      for (int r = 0; r < kOutRows; ++r) {
        const float w = weight[(out_row0 + r) * kMultiTokens + i];
        if (w != 0.0f) acc[r] = fmaf(w, v, acc[r]);  // a value that the row does not see may be infinite or NaN
      }
    }
    base = stop;
  }

#pragma unroll
  for (int k = 0; k < kWarpRows; ++k) {
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) l_run[k] += __shfl_xor_sync(0xffffffffu, l_run[k], d);
  }
  __syncthreads();
  if (part.count == 1) {
    float* den = weight;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < kWarpRows; ++k) den[warp + k * kMultiWarps] = l_run[k];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kOutRows; ++r) {
      if (out_row0 + r >= count) break;
      const float l = den[out_row0 + r], inv = l == 0.0f ? 0.0f : 1.0f / l;
      const float o[1] = {acc[r] * inv};
      multi_store<T, 1>(p, b, kvh, row0 + out_row0 + r, out_dim, o);
    }
    __syncthreads();
    return;
  }
  const int64_t at = multi_partial_row(part, part.mine, kMultiRows);
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < kWarpRows; ++k) {
      const int i = warp + k * kMultiWarps;
      if (i < count)
        reinterpret_cast<float2*>(p.stats)[at + i] = make_float2(m_run[k], l_run[k]);
    }
  }
#pragma unroll
  for (int r = 0; r < kOutRows; ++r) {
    if (out_row0 + r >= count) break;
    p.values[(at + out_row0 + r) * D + out_dim] = acc[r];
  }
  multi_merge<T, D, kMultiWarps, kMultiRows>(p, b, kvh, tile, row_tiles, count, part, smem);
  __syncthreads();
  });
}

// CTAs per SM: what shared memory holds, and there is room for the partials of.  (8 fp32 rows of 20-3000 tokens, 20 queries to a KV head,
// 64 dims, with a load per dim: two per SM 135 us, four 96; 24 rows of 3-31 tokens, 160 queries, 128 dims: two 68, three 50.)
template <int D>
constexpr int kMultiCtas = D == 64 ? 4 : D == 128 ? 3 : 1;
static_assert(148 * kMultiCtas<64> * kMultiRows <= kMultiMaxCtas * kMultiScratchRows, "partials of more rows than there is room for");

}  // namespace anna

using namespace anna;

extern "C" int anna_tq_multi_decode_plan(int batch, int q_heads, int kv_heads, int tokens, int head_dim, int64_t* scratch_size,
                                         int* counters) {
  const char* what = "anna_tq_multi_decode_plan";
  ANNA_REQUIRE(scratch_size != nullptr && counters != nullptr, "%s: null pointer argument", what);
  ANNA_REQUIRE(batch > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && tokens > 0 && head_dim > 0, "%s: bad sizes", what);
  ANNA_REQUIRE((int64_t)tokens * q_heads < (1 << 20) && (int64_t)tokens * (q_heads / kv_heads) * (q_heads / kv_heads) < (1ll << 32),
               "%s: too many queries", what);
  const int64_t tiles = (int64_t)batch * kv_heads * ((tokens * (q_heads / kv_heads) + kMultiRows - 1) / kMultiRows);
  ANNA_REQUIRE(tiles < (1ll << 31), "%s: too many queries", what);
  *scratch_size = (int64_t)kMultiMaxCtas * 2 * kMultiScratchRows * (head_dim + 2);
  *counters = (int)tiles;
  return ANNA_OK;
}

extern "C" int anna_tq_paged_multi_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                                          const uint8_t* packed_pages, const int32_t* block_table, int64_t table_stride,
                                          const void* window, const int64_t* window_slots, const int64_t* lengths,
                                          const float* signs1, const float* signs2, const float* centroids, const void* gate,
                                          int64_t gate_stride_b, int64_t gate_stride_h, int64_t gate_stride_t, void* out,
                                          int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t, float* scratch,
                                          int64_t scratch_size, int32_t* counters, int batch, int q_heads, int kv_heads,
                                          int tokens, int head_dim, int block_size, int residual_len, int bits,
                                          int value_group, int64_t num_pages, int64_t max_blocks, float scaling, int dtype,
                                          anna_stream_t stream) {
  const char* what = "anna_tq_paged_multi_decode";
  ANNA_REQUIRE(q && window && window_slots && lengths && signs1 && signs2 && centroids && out && counters && scratch,
               "%s: null pointer argument", what);
  ANNA_REQUIRE(max_blocks >= 0 && block_size > 0 && residual_len > 0, "%s: bad sizes", what);
  ANNA_REQUIRE(max_blocks == 0 || (packed_pages && block_table && num_pages > 0), "%s: a block table needs pages", what);
  int64_t needed = 0;
  int tiles = 0;
  if (const int rc = anna_tq_multi_decode_plan(batch, q_heads, kv_heads, tokens, head_dim, &needed, &tiles)) return rc;
  if (scratch_size < needed)
    return set_error(ANNA_ERR_WORKSPACE, "%s: scratch holds %lld floats, %lld are needed", what, (long long)scratch_size, (long long)needed);
  ANNA_REQUIRE(max_blocks < ((1ll << 30) - residual_len) / block_size, "%s: too many keys", what);
  TqMultiParams p{};
  ANNA_REQUIRE(dtype == ANNA_DTYPE_F32 || dtype == ANNA_DTYPE_F16 || dtype == ANNA_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  if (!tq_make_layout(head_dim, bits, block_size, dtype_bytes_of(dtype), value_group, &p.layout))
    return set_error(ANNA_ERR_UNSUPPORTED, "%s: unsupported page geometry (head_dim %d, bits %d, value group %d)", what, head_dim, bits,
                     value_group);
  ANNA_REQUIRE(aligned_to(packed_pages, 16) && aligned_to(window, 16), "%s: pages and window must be 16-byte aligned", what);
  ANNA_REQUIRE(aligned_to(scratch, 16), "%s: scratch must be 16-byte aligned", what);
  // the stride of a dim of one entry may be anything
  p.q = q; p.q_stride_b = batch > 1 ? q_stride_b : 0; p.q_stride_h = q_heads > 1 ? q_stride_h : 0; p.q_stride_t = tokens > 1 ? q_stride_t : 0;
  p.pages = packed_pages; p.block_table = block_table; p.table_stride = table_stride;
  p.window = window; p.window_slots = window_slots; p.lengths = lengths;
  p.signs1 = signs1; p.signs2 = signs2; p.centroids = centroids;
  p.gate = gate; p.gate_stride_b = gate_stride_b; p.gate_stride_h = gate_stride_h; p.gate_stride_t = gate_stride_t;
  p.out = out; p.out_stride_b = out_stride_b; p.out_stride_h = out_stride_h; p.out_stride_t = out_stride_t;
  p.values = scratch; p.stats = scratch + (int64_t)kMultiMaxCtas * 2 * kMultiScratchRows * head_dim; p.counters = counters;
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.groups = q_heads / kv_heads; p.tokens = tokens; p.rows = tokens * p.groups;
  p.groups_inverse = (uint32_t)(((1ull << 32) + p.groups - 1) / p.groups);  // of one: not read
  p.block_size = block_size; p.residual_len = residual_len; p.value_group = value_group;
  p.block_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1 << s) == block_size) p.block_shift = s;
  p.num_pages = num_pages; p.max_blocks = max_blocks; p.max_len = max_blocks * block_size + residual_len;
  p.scaling = scaling;
  const int row_tiles = (p.rows + kMultiRows - 1) / kMultiRows;
  const bool tensor_cores = tq_multi_mma_applicable(p, head_dim, dtype);
  p.stream_tiles = !tensor_cores ? 4 : head_dim <= 128 && p.rows <= 16 ? 32 : 64;
  p.min_share = tensor_cores ? 32 : 4;
  p.whole_tiles = tensor_cores ? 48 : 0;
  // The line of a launch has room for so many rows and positions: larger batches go in several, one behind the other.
  const int64_t row_positions = (int64_t)kv_heads * row_tiles * ((p.max_len + kBalancedTileTokens - 1) / kBalancedTileTokens + p.stream_tiles);
  ANNA_REQUIRE(row_positions < (1ll << 30), "%s: too many queries and keys of one sequence", what);
  int most = (int)(((1ll << 30) - 1) / row_positions);
  if (most > kBalancedMaxRows) most = kBalancedMaxRows;
  for (int at = 0; at < batch; at += most) {
    p.batch = batch - at < most ? batch - at : most;
    const int rc = tensor_cores ? launch_tq_multi_mma(p, head_dim, bits, dtype, (cudaStream_t)stream)
                                : ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
        return ANNA_DISPATCH_TQ_BITS(bits, BITS, [&]() -> int {
          constexpr int smem = kMultiSmemFloats<D> * 4;
          auto kernel = tq_multi_kernel<T, D, BITS>;
          ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
          kernel<<<multi_ctas(p, row_tiles, kMultiCtas<D>), kMultiThreads<D>, smem, (cudaStream_t)stream>>>(p, row_tiles);
          return check_launch("tq_multi_kernel");
        });
      });
    });
    if (rc != ANNA_OK) return rc;
    const int64_t elem = dtype_bytes_of(dtype);
    p.q = static_cast<const uint8_t*>(p.q) + (int64_t)most * p.q_stride_b * elem;
    p.out = static_cast<uint8_t*>(p.out) + (int64_t)most * out_stride_b * elem;
    if (p.gate != nullptr) p.gate = static_cast<const uint8_t*>(p.gate) + (int64_t)most * gate_stride_b * elem;
    if (p.block_table != nullptr) p.block_table += (int64_t)most * table_stride;
    p.window_slots += most;
    p.lengths += most;
  }
  return ANNA_OK;
}
