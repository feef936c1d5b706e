// Parameters and the merge of the multi-token decode over packed TurboQuant pages (tq_multi_decode.cu, tq_multi_mma.cu).
//
// The newest T tokens of a sequence are its queries; query t sees the keys at positions up to len - T + t.  The T * G queries that
// share a KV head are the rows of one product (row r = t * G + g), cut into row tiles.  A stream is one (sequence, KV head, row tile)
// with its keys [0, len).  One resident wave of CTAs takes even shares of the line on which all streams have their 16-token tiles
// (balanced_schedule.cuh): in fixed chunks, 32 ragged rows of 0.5-16 K tokens took 151 to 185 us by the length of the chunks, since
// the host does not know the lengths.  A share that ends inside a stream leaves the rows' partial softmax, and the CTA of a stream
// that arrives last merges them.
#pragma once

#include "balanced_schedule.cuh"
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
  float* stats;      // [CTAs, 2, rows of a tile, 2]: running maximum (natural units), denominator; see MultiPartial
  float* values;     // [CTAs, 2, rows of a tile, D]
  int32_t* counters;  // [B, Hkv, row tiles]
  int batch;
  int q_heads, kv_heads, groups, tokens, rows;  // rows = tokens * groups
  uint32_t groups_inverse;                       // ceil(2^32 / groups)
  int block_size, block_shift, residual_len, value_group;
  int64_t num_pages, max_blocks, max_len;
  float scaling;
  // What a stream costs a CTA beside its tiles (queries, first copies, merge), in tiles: 10 to 15 us.  By this number (16, 32, 64, 96),
  // tensor cores: 32 ragged rows of 0.5-16 K tokens, 20 queries to a KV head 181, 137, 127, 132 us; 16 rows of 0.4-4 K of 256 dims 109, 88, 83,
  // 90.  Of at most 16 queries and 128 dims, with shorter prologues, the same 32 rows 108, 88.4, 89.5, 92.4; 16 rows of 0.4-4 K 32.1, 28.4,
  // 29.3, 31.5; 64 rows of 0.1-2 K 50.8, 49.1, 48.0, 45.9; one row of 4000 24.4, 19.7, 20.1, 19.9.  So 32 there, 64 otherwise.
  int stream_tiles;
  // Positions of the line that a CTA takes at least, 32 with tensor cores: by this number (8, 16, 32, 64), one row of 16000 tokens, 4 new ones,
  // 32/8 heads 27.7, 27.4, 26.8, 28.1 us; of 4000 20.9, 18.2, 19.7, 27.3; of 1000 18.3, 17.4, 20.4, 31.2; batches of 16 rows and more the same.
  int min_share;
  int whole_tiles;  // streams of no more tiles, a CTA for each, are not cut: see multi_for_each_segment
  anna_tq_layout layout;
};

// Token of a row: row / groups, exact while row * groups < 2^32.
__device__ __forceinline__ int multi_token_of(const TqMultiParams& p, int row) {
  return p.groups == 1 ? row : (int)__umulhi((uint32_t)row, p.groups_inverse);
}

// One output row, from its dims d .. d + N - 1.
template <typename T, int N>
__device__ __forceinline__ void multi_store(const TqMultiParams& p, int64_t b, int kvh, int row, int d, const float (&o)[N]) {
  const int t = multi_token_of(p, row), h = kvh * p.groups + row - t * p.groups;
  T* out = reinterpret_cast<T*>(p.out) + b * p.out_stride_b + h * p.out_stride_h + t * p.out_stride_t + d;
  const T* gate = p.gate == nullptr
                      ? nullptr
                      : reinterpret_cast<const T*>(p.gate) + b * p.gate_stride_b + h * p.gate_stride_h + t * p.gate_stride_t + d;
#pragma unroll
  for (int i = 0; i < N; ++i)
    out[i] = ElemTraits<T>::from_float(gate != nullptr ? o[i] / (1.0f + __expf(-ElemTraits<T>::to_float(gate[i]))) : o[i]);
}

// The partials of a stream: one of each CTA from `first` on.  A CTA leaves two at most, of the stream that its share begins inside
// (slot 0) and of the one that it ends inside (slot 1): the first partial of a stream is in slot 1 of its CTA, the others in slot 0.
struct MultiPartial {
  int first, count, mine;
};
__device__ __forceinline__ int64_t multi_partial_row(const MultiPartial& part, int k, int rows_of_tile) {
  return ((int64_t)(part.first + k) * 2 + (k == 0 ? 1 : 0)) * rows_of_tile;
}

constexpr int kMultiMaxPartials = 256;  // of a stream
// Writes the zeros of this CTA's sequences without a key and calls segment(b, kvh, tile, t0, t1, partial) for each part of its share.
// All threads call it; `segment` ends with the CTA synchronised.
template <typename T, int D, int THREADS, typename Fn>
__device__ __forceinline__ void multi_for_each_segment(const TqMultiParams& p, int row_tiles, Fn&& segment) {
  __shared__ int s_prefix[kBalancedMaxRows + 1];
  const int streams_per_row = p.kv_heads * row_tiles;
  int tiles_of_rows[kBalancedRowsPerThread<THREADS>], streams;
  balanced_load_tiles<THREADS>(p.lengths, p.max_len, p.batch, 0, tiles_of_rows);
  const int max_tiles = balanced_scan<THREADS>(tiles_of_rows, p.batch, streams_per_row, s_prefix, p.stream_tiles, 0, &streams);
  const int total = s_prefix[p.batch];
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (s_prefix[b + 1] != s_prefix[b]) continue;
    for (int item = threadIdx.x; item < p.kv_heads * p.rows * (D / 4); item += THREADS) {
      const float zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const int row = item / (D / 4);
      multi_store<T, 4>(p, b, row / p.rows, row % p.rows, item % (D / 4) * 4, zeros);
    }
  }
  // Streams of few tiles with a CTA for each are not cut: what a CTA less has to do does not pay for the merge (16 rows of 300-500
  // tokens of 256 dims, 64 queries to a KV head: 41 us, 26 so).
  const bool whole = max_tiles <= p.whole_tiles && p.batch * streams_per_row <= (int)gridDim.x;
  const int share = whole ? 0 : max(max((total + (int)gridDim.x - 1) / (int)gridDim.x, p.min_share),
                                    (max_tiles + kMultiMaxPartials - 3) / (kMultiMaxPartials - 2));
  int pos = whole ? 0 : (int)min((int64_t)blockIdx.x * share, (int64_t)total);
  const int end = whole ? (int)blockIdx.x < p.batch * streams_per_row ? 1 : 0 : min(pos + share, total);
  if (pos >= end) return;
  int b = 0, hi = p.batch;  // s_prefix[b] <= pos < s_prefix[hi]
  if (whole) b = blockIdx.x / streams_per_row;
  while (!whole && hi - b > 1) {
    const int mid = (b + hi) >> 1;
    if (s_prefix[mid] <= pos) b = mid;
    else hi = mid;
  }
  while (pos < end) {
    while (share != 0 && s_prefix[b + 1] <= pos) ++b;
    const int len = (int)max((int64_t)0, min(p.lengths[b], p.max_len));
    const int n = (len + kBalancedTileTokens - 1) / kBalancedTileTokens + p.stream_tiles;
    const int stream = share == 0 ? (int)blockIdx.x - b * streams_per_row : (pos - s_prefix[b]) / n;
    const int at = share == 0 ? 0 : pos - s_prefix[b] - stream * n;
    const int stop = share == 0 ? n : min(n, at + end - pos);
    if (stop > p.stream_tiles) {
      const int begin = s_prefix[b] + stream * n;
      const int first = share == 0 ? 0 : (begin + p.stream_tiles) / share;
      segment(b, stream / row_tiles, stream % row_tiles, max(0, at - p.stream_tiles) * kBalancedTileTokens,
              min(len, (stop - p.stream_tiles) * kBalancedTileTokens),
              MultiPartial{first, share == 0 ? 1 : (begin + n - 1) / share - first + 1, (int)blockIdx.x - first});
    }
    pos += stop - at;
  }
}

// Merges the partials of rows [row0, row0 + count) when this CTA is the last of theirs to get here.  `weights`: shared memory for
// ROWS x kMultiMaxPartials floats, which nothing else uses any more.  What this takes is the latency of its reads from L2, so a thread
// has the same four dims of several rows and several partials on their way at a time (33 partials of 16 rows, a thread's rows one
// after the other: one row of 4000 tokens 46 us, 31 so).
template <typename T, int D, int WARPS, int ROWS>
__device__ __forceinline__ void multi_merge_rows(const TqMultiParams& p, int64_t b, int kvh, int tile, int tiles, int row0, int count,
                                                 const MultiPartial& part, float* weights) {
  if (!merge_arrive(FusedCombine{p.counters}, (b * p.kv_heads + kvh) * tiles + tile, part.count)) return;
  const int chunks = part.count;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float2* all_stats = reinterpret_cast<const float2*>(p.stats);
  for (int i = warp; i < count; i += WARPS) {
    constexpr int kHeld = kMultiMaxPartials / 32;
    float2 s[kHeld];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int c = lane + 32 * k;
      s[k] = c < chunks ? __ldcg(all_stats + multi_partial_row(part, c, ROWS) + i) : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, s[k].x);
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float m_ref = m == -INFINITY ? 0.0f : m;
    float den = 0.0f;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      s[k].x = __expf(s[k].x - m_ref);
      den += s[k].x * s[k].y;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) den += __shfl_xor_sync(0xffffffffu, den, d);
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;  // a NaN among the scores has to stay one, so only an empty row is zero
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (lane + 32 * k < chunks) weights[i * chunks + lane + 32 * k] = s[k].x * inv;
  }
  __syncthreads();
  constexpr int kCols = D / 4, kRowsAtOnce = WARPS * 32 / kCols > 0 ? WARPS * 32 / kCols : 1;  // rows that the threads cover
  constexpr int kMine = ROWS / kRowsAtOnce > 0 ? ROWS / kRowsAtOnce : 1;                          // rows of a thread
  constexpr int kAhead = kMine >= 8 ? 2 : kMine >= 4 ? 4 : 8;                                     // chunks on their way
  const int col = threadIdx.x % kCols, mine = threadIdx.x / kCols;
  if (mine >= kRowsAtOnce) return;
  float4 acc[kMine];
#pragma unroll
  for (int r = 0; r < kMine; ++r) acc[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const float* values = p.values + 4 * col;
  for (int c0 = 0; c0 < chunks; c0 += kAhead) {
    float4 v[kAhead][kMine];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int r = 0; r < kMine; ++r)
        v[k][r] = __ldcg(reinterpret_cast<const float4*>(
            values + (multi_partial_row(part, min(c0 + k, chunks - 1), ROWS) + min(mine + r * kRowsAtOnce, count - 1)) * D));
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (c0 + k < chunks) {
#pragma unroll
        for (int r = 0; r < kMine; ++r) merge_add(acc[r], v[k][r], weights[min(mine + r * kRowsAtOnce, count - 1) * chunks + c0 + k]);
      }
  }
#pragma unroll
  for (int r = 0; r < kMine; ++r) {
    const int i = mine + r * kRowsAtOnce;
    const float out[4] = {acc[r].x, acc[r].y, acc[r].z, acc[r].w};
    if (i < count) multi_store<T, 4>(p, b, kvh, row0 + i, 4 * col, out);
  }
}

// The same, the tiles of a (sequence, KV head) all of ROWS rows but the last.
template <typename T, int D, int WARPS, int ROWS>
__device__ __forceinline__ void multi_merge(const TqMultiParams& p, int64_t b, int kvh, int tile, int tiles, int count,
                                            const MultiPartial& part, float* weights) {
  multi_merge_rows<T, D, WARPS, ROWS>(p, b, kvh, tile, tiles, tile * ROWS, count, part, weights);
}

// Tensor-core form (tq_multi_mma.cu): 16-bit caches, head_dim 64, 128 and 256, value groups of 32, pages of a multiple of 8 tokens.
bool tq_multi_mma_applicable(const TqMultiParams& p, int head_dim, int dtype);
int launch_tq_multi_mma(const TqMultiParams& p, int head_dim, int bits, int dtype, cudaStream_t stream);
int tq_multi_mma_faults(int* count);  // bounded copy waits that expired on the current device

// CTAs of a call: one resident wave, or fewer where that would leave shares below the smallest.
constexpr int kMultiMaxCtas = 148 * 2, kMultiScratchRows = 16;  // or other numbers with the same product
inline int multi_ctas(const TqMultiParams& p, int row_tiles, int per_sm) {
  const int64_t line = (int64_t)p.batch * p.kv_heads * row_tiles * ((p.max_len + kBalancedTileTokens - 1) / kBalancedTileTokens + p.stream_tiles);
  const int64_t shares = (line + p.min_share - 1) / p.min_share;
  return (int)(shares < 148 * per_sm ? shares : 148 * per_sm);
}

}  // namespace anna
