// Attention of the newest T tokens of every sequence over the 8-bit paged cache: the CUDA-core form and the entry points.
//
// This form serves pages that are no multiple of 8 tokens; everything in it is 32 bits.  A CTA brings 32 tokens at a
// time into shared memory, as floats without their scale, for its 8 rows; a warp scores two rows (256 dims: one) with a token a lane.
// Bound: issue, of which the reads of shared memory are as many as the FMAs (16 rows of 32768 tokens in pages of 20, 4 queries a KV head, 3.2 ms; in pages of
// 24, which tensor cores read, 0.21).  A tile of 16 tokens of those lies in one page or half and half in two; pages of other sizes would take a page lookup, scales and
// a copy of their own for every token.
#include "q8_common.cuh"

namespace anna {

template <int D>
constexpr int kQ8Threads = D == 256 ? 256 : 128;
constexpr int kQ8Rows = 8;     // of a CTA of this form
constexpr int kQ8Tokens = 32;  // in shared memory at a time: a lane's token
template <int D>
constexpr int kQ8SmemFloats = kQ8Rows * D + kQ8Tokens * (D + 1) + kQ8Tokens * D + kQ8Rows * kQ8Tokens;

template <typename T, int D, bool kBlocks>
__global__ void __launch_bounds__(kQ8Threads<D>) q8_attention_kernel(const Q8Params p, int row_tiles) {
  constexpr int E = D / 32, kThreads = kQ8Threads<D>, kWarps = kThreads / 32, kWarpRows = kQ8Rows / kWarps;
  extern __shared__ __align__(16) float smem[];
  // rows of D are held in an order of their own, dim lane * E + j at j * 32 + lane: a lane takes neighbouring dims
  float* q_smem = smem;                          // [rows][D], scaled
  float* keys = q_smem + kQ8Rows * D;            // [tokens][D + 1]
  float* vals = keys + kQ8Tokens * (D + 1);      // [tokens][D]
  float* weight = vals + kQ8Tokens * D;          // [rows][tokens]
  __shared__ float sm_scale[kQ8Tokens], sm_rescale[kQ8Rows];
  __shared__ int sm_position[kQ8Tokens];         // in the sequence; past its end for what is not there

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  q8_wait_for_previous();
  q8_for_each_segment<T, D, kThreads, kBlocks>(p, row_tiles, [&](int64_t b, int kvh, int tile, int t0, int t1, int len, const MultiPartial& part) {
  const Q8Stream st = q8_stream<kQ8Rows>(p, b, kvh, tile, len);
  const int row0 = st.row0, count = st.count;
  const int first_seen = st.len - p.tokens;  // newest key that query 0 sees

  for (int i = warp; i < count; i += kWarps) {
    const int t = multi_token_of(p, row0 + i), h = kvh * p.groups + row0 + i - t * p.groups;
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_stride_b + h * p.q_stride_h + t * p.q_stride_t + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) q_smem[i * D + j * 32 + lane] = ElemTraits<T>::to_float(q[j]) * p.scaling;
  }
  float m_run[kWarpRows], l_run[kWarpRows];  // of every kWarps-th row from `warp` on
#pragma unroll
  for (int k = 0; k < kWarpRows; ++k) {
    m_run[k] = -INFINITY;
    l_run[k] = 0.0f;
  }
  static_assert(D <= kThreads && kThreads % D == 0, "a thread has one dim");
  constexpr int kOutRows = kQ8Rows * D / kThreads;
  const int out_row0 = (int)threadIdx.x / D * kOutRows, place = (int)threadIdx.x % D, out_dim = place % 32 * E + place / 32;
  float acc[kOutRows];
#pragma unroll
  for (int r = 0; r < kOutRows; ++r) acc[r] = 0.0f;

  const int64_t slot = st.len > st.full ? p.window_slots[b] : -1;
  const T* ring = slot >= 0 && slot < p.num_slots ? reinterpret_cast<const T*>(p.window) + (slot * 2 * p.kv_heads + kvh) * p.block_size * D : nullptr;
  const int64_t ring_values = (int64_t)p.kv_heads * p.block_size * D;
  for (int base = t0; base < t1;) {
    const bool packed = base < st.packed;
    const int stop = min(packed ? min(st.packed, t1) : t1, base + kQ8Tokens), n = stop - base;
    __syncthreads();
    // ---- 32 tokens into shared memory: a lane finds its token, then a warp takes a token at a time --------------------------------
    int64_t page = -1;
    int position = INT32_MAX;
    int in_page = 0;
    float value_scale = 0.0f;
    if (lane < n) {
      if (packed) {
        const int entry = (base + lane) / p.block_size;
        in_page = base + lane - entry * p.block_size;
        int block;
        page = q8_page_at(p, st, b, kvh, entry, &block);
        if (page >= 0) {
          position = block * p.block_size + in_page;
          const float2 scale = *reinterpret_cast<const float2*>(p.pages + page + q8_scale_offset(D, p.block_size));
          value_scale = scale.y;
          if (warp == 0) sm_scale[lane] = scale.x;
        }
      } else {
        in_page = base + lane - st.packed;
        page = ring != nullptr ? 0 : -1;
        if (page >= 0) position = st.full + in_page;
        value_scale = 1.0f;
        if (warp == 0) sm_scale[lane] = 1.0f;
      }
    }
    if (warp == 0) sm_position[lane] = position;
    for (int i = warp; i < n; i += kWarps) {
      const int64_t where = __shfl_sync(0xffffffffu, page, i);
      const int tok = __shfl_sync(0xffffffffu, in_page, i);
      const float scale = __shfl_sync(0xffffffffu, value_scale, i);
      float k[E], v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) k[j] = v[j] = 0.0f;
      if (where >= 0) {
        if (packed) {
          const int8_t* codes = reinterpret_cast<const int8_t*>(p.pages) + where + tok * D + lane * E;
#pragma unroll
          for (int j = 0; j < E; ++j) {
            k[j] = (float)codes[j];
            v[j] = scale * (float)codes[p.block_size * D + j];
          }
        } else {
          lane_load<T, E>(ring + tok * D + lane * E, k);
          lane_load<T, E>(ring + ring_values + tok * D + lane * E, v);
        }
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        keys[i * (D + 1) + j * 32 + lane] = k[j];
        vals[i * D + j * 32 + lane] = v[j];
      }
    }
    __syncthreads();
    // ---- scores: token `lane` -------------------------------------------------------------------------------------------------------
    float s[kWarpRows];
#pragma unroll
    for (int k = 0; k < kWarpRows; ++k) s[k] = -INFINITY;
    if (lane < n) {
      float sum[kWarpRows];
#pragma unroll
      for (int k = 0; k < kWarpRows; ++k) sum[k] = 0.0f;
#pragma unroll 16
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int k = 0; k < kWarpRows; ++k) sum[k] = fmaf(q_smem[(warp + k * kWarps) * D + d], keys[lane * (D + 1) + d], sum[k]);
#pragma unroll
      for (int k = 0; k < kWarpRows; ++k) {
        const int i = warp + k * kWarps;
        if (i < count && sm_position[lane] <= first_seen + multi_token_of(p, row0 + i)) s[k] = sum[k] * sm_scale[lane];
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
      weight[(warp + k * kWarps) * kQ8Tokens + lane] = w;
      if (lane == 0) sm_rescale[warp + k * kWarps] = rescale;
    }
    __syncthreads();
    // ---- values ------------------------------------------------------------------------------------------------------------------
#pragma unroll
    for (int r = 0; r < kOutRows; ++r) acc[r] *= sm_rescale[out_row0 + r];
    for (int i = 0; i < n; ++i) {
      const float v = vals[i * D + place];
      if (fabsf(v) < INFINITY) {
#pragma unroll
        for (int r = 0; r < kOutRows; ++r) acc[r] = fmaf(weight[(out_row0 + r) * kQ8Tokens + i], v, acc[r]);
      } else {  // infinite or NaN: for the rows that see it, however small its weight
#pragma unroll
        for (int r = 0; r < kOutRows; ++r)
          if (sm_position[i] <= first_seen + multi_token_of(p, row0 + out_row0 + r)) acc[r] += v;
      }
    }
    base = stop;
  }

#pragma unroll
  for (int k = 0; k < kWarpRows; ++k)
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) l_run[k] += __shfl_xor_sync(0xffffffffu, l_run[k], d);
  __syncthreads();
  if (part.count == 1) {
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < kWarpRows; ++k) weight[warp + k * kWarps] = l_run[k];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kOutRows; ++r) {
      if (out_row0 + r >= count) break;
      const float l = weight[out_row0 + r], inv = l == 0.0f ? 0.0f : 1.0f / l;  // a NaN among the scores has to stay one
      const float o[1] = {acc[r] * inv};
      multi_store<T, 1>(p, b, kvh, row0 + out_row0 + r, out_dim, o);
    }
    __syncthreads();
    return;
  }
  const int64_t at = multi_partial_row(part, part.mine, kQ8Rows);
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < kWarpRows; ++k) {
      const int i = warp + k * kWarps;
      if (i < count) reinterpret_cast<float2*>(p.stats)[at + i] = make_float2(m_run[k], l_run[k]);
    }
  }
#pragma unroll
  for (int r = 0; r < kOutRows; ++r) {
    if (out_row0 + r >= count) break;
    p.values[(at + out_row0 + r) * D + out_dim] = acc[r];
  }
  multi_merge_rows<T, D, kWarps, kQ8Rows>(p, b, kvh, tile, row_tiles, row0, count, part, smem);
  __syncthreads();
  });
}

template <int D>
constexpr int kQ8Ctas = D == 64 ? 4 : D == 128 ? 3 : 1;  // per SM

}  // namespace anna

using namespace anna;

namespace {

constexpr int kQ8MinTiles = 4;   // of a CTA with blocks, CUDA cores
// Tensor cores.  What a stream costs a CTA beside its tiles, in tiles; by this number (8, 16, 32, 64) 64 ragged rows of 0.5-16 K tokens 113, 107, 107,
// 112 us, 16 rows of 0.4-4 K tokens of 256 dims 70, 68, 63, 70.  Positions of the line that a CTA takes at least; by this number (8, 16, 32, 64) one row of
// 4000 tokens 11.5, 9.9, 11.2, 14.8; tiles of a list alike (one row's 256 pages: 4 to 12 tiles 9.8, 16 9.3, 24 10.9, 32 11.2).
constexpr int kQ8StreamTiles = 32, kQ8MinShare = 16;

// What a call takes; the sizes have been checked.
Q8Plan q8_plan(int batch, int q_heads, int kv_heads, int tokens, int head_dim, int block_size, int64_t max_blocks, int width, int dtype) {
  Q8Plan plan{};
  if (max_blocks == 0) width = 0;  // a table without columns has no page to choose: the kernels go by the ring alone
  const int groups = q_heads / kv_heads, rows = width > 0 ? groups : tokens * groups;
  plan.tensor_cores = block_size % 8 == 0;
  // key tiles of all streams, with what a stream costs beside its own; a stream has one row tile where `few` counts
  const int64_t axis = width > 0 ? (int64_t)(width + 1) * block_size : max_blocks * block_size + block_size - 1;
  const int64_t key_tiles = (axis + kBalancedTileTokens - 1) / kBalancedTileTokens;
  const bool few = (int64_t)batch * kv_heads * (width > 0 ? tokens * key_tiles : key_tiles + kQ8StreamTiles) <= 148 * kQ8MinShare;
  const Q8Shape shape = plan.tensor_cores ? q8_mma_shape(head_dim, rows, few)
                                          : Q8Shape{kQ8Rows, head_dim == 64 ? kQ8Ctas<64> : head_dim == 128 ? kQ8Ctas<128> : kQ8Ctas<256>, 4};
  plan.rows = shape.rows;
  plan.warps = shape.warps;
  const int per_sm = shape.ctas, min_tiles = plan.tensor_cores ? 16 : kQ8MinTiles;
  const int tiles = (rows + plan.rows - 1) / plan.rows;
  plan.tiles_per_token = tiles;
  plan.row_tiles = width > 0 ? tokens * tiles : tiles;
  const int64_t streams = (int64_t)batch * kv_heads * plan.row_tiles, wave = 148 * per_sm;
  plan.splits = 1;
  plan.ctas = wave;
  if (width > 0) {
    int64_t splits = wave / (streams < 1 ? 1 : streams);
    if (splits > key_tiles / min_tiles) splits = key_tiles / min_tiles;
    if (splits > kMultiMaxPartials) splits = kMultiMaxPartials;
    plan.splits = splits < 1 ? 1 : (int)splits;
    plan.ctas = streams * plan.splits;
  }
  const int64_t partials = width > 0 && plan.splits == 1 ? 0 : plan.ctas * 2 * plan.rows;
  plan.floats = partials * (head_dim + 2) + 4;
  plan.counters = (int)streams;
  return plan;
}

int q8_check_sizes(const char* what, int batch, int q_heads, int kv_heads, int tokens, int head_dim, int block_size, int64_t max_blocks, int width) {
  int64_t bytes = 0;
  if (const int rc = anna_q8_page_bytes(head_dim, block_size, &bytes)) return rc;
  ANNA_REQUIRE(batch > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && tokens > 0 && max_blocks >= 0 && width >= 0, "%s: bad sizes", what);
  ANNA_REQUIRE((int64_t)tokens * q_heads < (1 << 20) && (int64_t)tokens * (q_heads / kv_heads) * (q_heads / kv_heads) < (1ll << 32),
               "%s: too many queries", what);
  ANNA_REQUIRE(max_blocks < (1ll << 30) / block_size - 1 && width < (1ll << 30) / block_size - 1, "%s: too many keys", what);
  ANNA_REQUIRE((int64_t)batch * kv_heads * tokens * (q_heads / kv_heads) < (1ll << 31), "%s: too many queries", what);
  return ANNA_OK;
}

}  // namespace

extern "C" int anna_q8_attention_plan(int batch, int q_heads, int kv_heads, int tokens, int head_dim, int block_size, int64_t max_blocks,
                                      int width, int dtype, int64_t* scratch_size, int* counters) {
  const char* what = "anna_q8_attention_plan";
  ANNA_REQUIRE(scratch_size != nullptr && counters != nullptr, "%s: null pointer argument", what);
  if (const int rc = q8_check_sizes(what, batch, q_heads, kv_heads, tokens, head_dim, block_size, max_blocks, width)) return rc;
  const Q8Plan plan = q8_plan(batch, q_heads, kv_heads, tokens, head_dim, block_size, max_blocks, width, dtype);
  *scratch_size = plan.floats;
  *counters = plan.counters;
  return ANNA_OK;
}

extern "C" int anna_q8_attention(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, const uint8_t* pages,
                                 const int32_t* page_table, int64_t table_stride, const void* window, const int64_t* window_slots,
                                 const int64_t* lengths, const int32_t* blocks, int width, const void* gate, int64_t gate_stride_b,
                                 int64_t gate_stride_h, int64_t gate_stride_t, void* out, int64_t out_stride_b, int64_t out_stride_h,
                                 int64_t out_stride_t, float* scratch, int64_t scratch_size, int32_t* counters, int batch, int q_heads,
                                 int kv_heads, int tokens, int head_dim, int block_size, int64_t num_pages, int64_t max_blocks,
                                 int64_t num_slots, float scaling, int dtype, anna_stream_t stream) {
  const char* what = "anna_q8_attention";
  ANNA_REQUIRE(q && window && window_slots && lengths && out && counters && scratch, "%s: null pointer argument", what);
  ANNA_REQUIRE(dtype == ANNA_DTYPE_F32 || dtype == ANNA_DTYPE_F16 || dtype == ANNA_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  ANNA_REQUIRE((blocks != nullptr) == (width > 0), "%s: blocks go with their width", what);
  if (const int rc = q8_check_sizes(what, batch, q_heads, kv_heads, tokens, head_dim, block_size, max_blocks, width)) return rc;
  ANNA_REQUIRE(max_blocks == 0 || (pages && page_table && num_pages > 0), "%s: a block table needs pages", what);
  ANNA_REQUIRE(aligned_to(pages, 16) && aligned_to(window, 16), "%s: pages and window must be 16-byte aligned", what);
  ANNA_REQUIRE(aligned_to(scratch, 16), "%s: scratch must be 16-byte aligned", what);
  if (max_blocks == 0) {  // as q8_plan has it; there may be no pool either
    blocks = nullptr;
    width = 0;
  }
  const Q8Plan plan = q8_plan(batch, q_heads, kv_heads, tokens, head_dim, block_size, max_blocks, width, dtype);
  if (scratch_size < plan.floats)
    return set_error(ANNA_ERR_WORKSPACE, "%s: scratch holds %lld floats, %lld are needed", what, (long long)scratch_size, (long long)plan.floats);
  ANNA_REQUIRE(plan.ctas < (1ll << 31), "%s: too many queries", what);
  Q8Params p{};
  // the stride of a dim of one entry may be anything
  p.q = q; p.q_stride_b = batch > 1 ? q_stride_b : 0; p.q_stride_h = q_heads > 1 ? q_stride_h : 0; p.q_stride_t = tokens > 1 ? q_stride_t : 0;
  p.pages = pages; p.block_table = page_table; p.table_stride = table_stride;
  p.window = window; p.window_slots = window_slots; p.num_slots = num_slots; p.lengths = lengths;
  p.blocks = blocks; p.width = width; p.tiles_per_token = plan.tiles_per_token; p.splits = plan.splits;
  p.gate = gate; p.gate_stride_b = gate_stride_b; p.gate_stride_h = gate_stride_h; p.gate_stride_t = gate_stride_t;
  p.out = out; p.out_stride_b = out_stride_b; p.out_stride_h = out_stride_h; p.out_stride_t = out_stride_t;
  p.values = scratch;
  p.stats = scratch + (plan.floats - 4) / (head_dim + 2) * head_dim;
  p.counters = counters;
  p.batch = batch; p.q_heads = q_heads; p.kv_heads = kv_heads; p.groups = q_heads / kv_heads; p.tokens = tokens; p.rows = tokens * p.groups;
  p.groups_inverse = (uint32_t)(((1ull << 32) + p.groups - 1) / p.groups);  // of one: not read
  p.block_size = block_size; p.page_bytes = q8_page_bytes(head_dim, block_size);
  p.block_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1 << s) == block_size) p.block_shift = s;
  p.num_pages = num_pages; p.max_blocks = max_blocks; p.max_len = max_blocks * block_size + block_size - 1;
  p.scaling = scaling;
  p.stream_tiles = plan.tensor_cores ? kQ8StreamTiles : 4;
  p.min_share = plan.tensor_cores ? kQ8MinShare : 4;
  p.whole_tiles = 0;
  // The line of a launch without blocks has room for so many rows and positions: larger batches go in several, one behind the other.
  int most = batch;
  if (width == 0) {
    const int64_t row_positions = (int64_t)kv_heads * plan.row_tiles * ((p.max_len + kBalancedTileTokens - 1) / kBalancedTileTokens + p.stream_tiles);
    ANNA_REQUIRE(row_positions < (1ll << 30), "%s: too many queries and keys of one sequence", what);
    most = (int)(((1ll << 30) - 1) / row_positions);
    if (most > kBalancedMaxRows) most = kBalancedMaxRows;
  }
  for (int at = 0; at < batch; at += most) {
    p.batch = batch - at < most ? batch - at : most;
    const int ctas = width > 0 ? (int)plan.ctas : multi_ctas(p, plan.row_tiles, (int)(plan.ctas / 148));
    const int rc = ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      if (plan.tensor_cores) return launch_q8_mma_of<T>(p, plan, head_dim, ctas, (cudaStream_t)stream);
      return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
        constexpr int smem = kQ8SmemFloats<D> * 4;
        auto kernel = width > 0 ? q8_attention_kernel<T, D, true> : q8_attention_kernel<T, D, false>;
        ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return q8_launch("q8_attention_kernel", kernel, dim3((unsigned)ctas), kQ8Threads<D>, smem, (cudaStream_t)stream, p, plan.row_tiles);
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
