// Selection of the pages that a query should look at, by a bound on its products with their keys.
//
// With high_d and low_d the largest and smallest code of dim d in a page, sum_d max(r_d high_d, r_d low_d) bounds r . code from above for
// every key of the page.  r is the query in whole numbers of 15 bits and a sign, so the sum is one, below 2^31: no order of summation
// changes it, and a score is the same wherever it is worked out.  With r+ = max(r, 0), r- = max(-r, 0) and the page's bounds
// [high, -low] the sum is one product of 2 D, [r+, r-] . [high, -low], of non-negative numbers of 15 bits, as two bytes (128 u + v,
// u < 256, v < 128), with signed bytes: integer mma, 16 pages to a tile, 8 query heads.
//
// Scores: a warp takes 16 pages at a time, for all heads and several tokens.  Bound: HBM (2 D + 4 bytes a page and head), or the launch.
// Choice: a CTA per query token and KV head finds the score of the last page that is taken, 8 bits at a time, counting how many scores
// share the bits so far; then the pages above it, and of those equal to it the first, are written in order.
#include "q8_common.cuh"

namespace anna {

struct Q8SelectParams {
  const void* q;
  int64_t q_stride_b, q_stride_h, q_stride_t;
  const uint8_t* pages;
  const int32_t* block_table;
  int64_t table_stride;
  const int64_t* lengths;
  int32_t* blocks;
  uint32_t* scores;  // [B, Hkv, T, max_blocks], larger is better, 0: no candidate
  int kv_heads, groups, tokens, block_size, page_bytes;
  int count, first, recent;
  int head_tiles, tokens_at_once;  // tiles of 8 query heads of a token; tokens of a CTA
  int64_t num_pages, max_blocks;
};

constexpr int kQ8SelectWarps = 8;
constexpr int kQ8SelectTile = 16;  // pages of a warp at a time
constexpr uint32_t kQ8Forced = 0xffffffffu;

// Full pages of which query t sees a token.
__device__ __forceinline__ int q8_candidates(const Q8SelectParams& p, int64_t b, int t) {
  const int64_t len = max((int64_t)0, min(p.lengths[b], p.max_blocks * p.block_size + p.block_size - 1));
  const int64_t seen = len - p.tokens + t + 1;
  return seen <= 0 ? 0 : (int)min(len / p.block_size, (seen + p.block_size - 1) / p.block_size);
}

__device__ __forceinline__ void mma_s8u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Order of floats as order of whole numbers, none of them 0.
__device__ __forceinline__ uint32_t q8_ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

template <typename T, int D>
__global__ void __launch_bounds__(kQ8SelectWarps * 32) q8_score_kernel(const Q8SelectParams p) {
  constexpr int kChunks = 2 * D / 64;  // of 64 bounds, 16 of them a lane's
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int64_t b = blockIdx.y / p.kv_heads;
  const int kvh = blockIdx.y % p.kv_heads;
  const int token0 = blockIdx.z * p.tokens_at_once, here = min(p.tokens_at_once, p.tokens - token0);
  const int head_tiles = p.head_tiles, tiles = here * head_tiles;
  uint4* parts = reinterpret_cast<uint4*>(smem);                                              // [2][tiles][kChunks][32 lanes]
  float* tops = reinterpret_cast<float*>(smem + p.tokens_at_once * head_tiles * 2 * kChunks * 512);  // [tiles][8]

  // ---- queries in whole numbers --------------------------------------------------------------------------------------------------
  for (int row = warp; row < tiles * 8; row += kQ8SelectWarps) {
    const int t = row / (8 * head_tiles), g = row % (8 * head_tiles);
    float x[D / 32], top = 0.0f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      x[j] = 0.0f;
      if (g < p.groups)
        x[j] = ElemTraits<T>::to_float(reinterpret_cast<const T*>(p.q)[b * p.q_stride_b + (int64_t)(kvh * p.groups + g) * p.q_stride_h +
                                                                      (int64_t)(token0 + t) * p.q_stride_t + lane + 32 * j]);
      top = fmaxf(top, fabsf(x[j]));
      fine = fine && fabsf(x[j]) < INFINITY;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    fine = __all_sync(0xffffffffu, fine);
    if (lane == 0) tops[row] = fine ? top : __int_as_float(0x7fc00000);
    // the whole number next to 32767 x / top, as q8_append.cu finds codes: a quotient that is no tie is at least 2^-40 of its power of
    // two away from one, the product is off by 2^-51 of it at most
    const double rate = fine && top > 0.0f ? 32767.0 / (double)top : 0.0;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const double r = fine ? __dmul_rn((double)x[j], rate) : 0.0, c = __dmul_rn(r, 257.0);
      const int whole = __double2int_rn(__dsub_rn(c, __dsub_rn(c, r)));
      const int d = lane + 32 * j;
#pragma unroll
      for (int negated = 0; negated < 2; ++negated) {
        const int n = max(negated ? -whole : whole, 0), at = d + negated * D;
        const int place = ((row / 8 * kChunks + at / 64) * 32 + row % 8 * 4 + at % 64 / 16) * 16 + at % 16;
        smem[place] = (uint8_t)(n >> 7);
        smem[tiles * kChunks * 512 + place] = (uint8_t)(n & 127);
      }
    }
  }
  __syncthreads();

  // ---- 16 pages at a time -----------------------------------------------------------------------------------------------------------
  const int most = q8_candidates(p, b, token0 + here - 1);
  for (int tile = blockIdx.x * kQ8SelectWarps + warp; tile * kQ8SelectTile < most; tile += gridDim.x * kQ8SelectWarps) {
    uint4 w[2][kChunks];
    float scale[2];
    bool there[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = tile * kQ8SelectTile + gid + 8 * i;
      int32_t pid = -1;
      if (j < most) pid = p.block_table[b * p.table_stride + j];
      there[i] = pid >= 0 && pid < p.num_pages;
      const uint8_t* page = p.pages + (there[i] ? ((int64_t)pid * p.kv_heads + kvh) * p.page_bytes : 0);
      scale[i] = *reinterpret_cast<const float*>(page + q8_scale_offset(D, p.block_size));
      const uint4* bounds = reinterpret_cast<const uint4*>(page + q8_bounds_offset(D, p.block_size));
#pragma unroll
      for (int c = 0; c < kChunks; ++c) w[i][c] = ldg_stream16(bounds + 4 * c + tig);
    }
    for (int t = 0; t < here; ++t) {
      float best[2] = {-INFINITY, -INFINITY};
      for (int h = 0; h < head_tiles; ++h) {
        int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
        const uint4* at = parts + (t * head_tiles + h) * kChunks * 32 + lane;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint4 u = at[c * 32], v = at[(tiles * kChunks + c) * 32];
          mma_s8u8(hi, w[0][c].x, w[1][c].x, w[0][c].y, w[1][c].y, u.x, u.y);
          mma_s8u8(lo, w[0][c].x, w[1][c].x, w[0][c].y, w[1][c].y, v.x, v.y);
          mma_s8u8(hi, w[0][c].z, w[1][c].z, w[0][c].w, w[1][c].w, u.z, u.w);
          mma_s8u8(lo, w[0][c].z, w[1][c].z, w[0][c].w, w[1][c].w, v.z, v.w);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int g = h * 8 + 2 * tig + (r & 1);
          if (g >= p.groups) continue;
          const float top = tops[(t * head_tiles + h) * 8 + 2 * tig + (r & 1)];
          const float x = __fmul_rn(__fmul_rn(top, scale[r / 2]), __int2float_rn(128 * hi[r] + lo[r]));
          best[r / 2] = isnan(x) ? INFINITY : fmaxf(best[r / 2], x);
        }
      }
      const int candidates = q8_candidates(p, b, token0 + t);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
        const int j = tile * kQ8SelectTile + gid + 8 * i;
        if (tig == 0 && j < candidates) {
          const bool forced = j < p.first || j >= candidates - p.recent;
          p.scores[((int64_t)blockIdx.y * p.tokens + token0 + t) * p.max_blocks + j] = !there[i] ? 0u : forced ? kQ8Forced : q8_ordered(best[i]);
        }
      }
    }
  }
}

constexpr int kQ8PickThreads = 256;
constexpr int kQ8PickHeld = 12288;  // scores that are kept in shared memory

// Exclusive sums of x and y over the CTA's threads.
__device__ __forceinline__ void q8_scan2(int& x, int& y, int* smem) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int a = x, b = y;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, a, d), v = __shfl_up_sync(0xffffffffu, b, d);
    if (lane >= d) {
      a += u;
      b += v;
    }
  }
  if (lane == 31) {
    smem[2 * warp] = a;
    smem[2 * warp + 1] = b;
  }
  __syncthreads();
  int before_a = 0, before_b = 0;
  for (int w = 0; w < warp; ++w) {
    before_a += smem[2 * w];
    before_b += smem[2 * w + 1];
  }
  x = before_a + a - x;
  y = before_b + b - y;
}

template <bool kHeld>
__global__ void __launch_bounds__(kQ8PickThreads) q8_pick_kernel(const Q8SelectParams p) {
  constexpr int kWarps = kQ8PickThreads / 32;
  extern __shared__ __align__(16) uint32_t held[];
  __shared__ int histogram[256], s_sums[2 * kWarps], s_digit, s_left;
  const int64_t stream = blockIdx.x;
  const int64_t b = stream / p.tokens / p.kv_heads;
  const int t = (int)(stream % p.tokens);
  const int n = q8_candidates(p, b, t);
  const uint32_t* scores = p.scores + stream * p.max_blocks;
  int32_t* out = p.blocks + stream * p.count;
  // place of score i in shared memory: a thread's run of scores and the next one's begin in different banks
  const int run = (n + kQ8PickThreads - 1) / kQ8PickThreads;
  auto score = [&](int i) { return kHeld ? held[i + i / 32] : __ldcg(scores + i); };
  if (kHeld)
    for (int i = threadIdx.x; i < n; i += kQ8PickThreads) held[i + i / 32] = __ldcg(scores + i);
  // ---- the score of the last page that is taken, and how many of that score --------------------------------------------------------
  uint32_t least = 1, known = 0;  // `known`: the bits of `least` that have been found
  int left = p.count;
  if (n > p.count) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      histogram[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kQ8PickThreads) {
        const uint32_t x = score(i);
        if (x != 0 && (x & known) == (least & known)) atomicAdd(&histogram[(x >> shift) & 255], 1);
      }
      __syncthreads();
      if (threadIdx.x < 32) {  // a lane has eight digits, the largest first
        const int lane = threadIdx.x;
        int mine[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += mine[i] = histogram[255 - 8 * lane - i];
        int up_to = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, up_to, d);
          if (lane >= d) up_to += v;
        }
        const bool crosses = up_to >= left && up_to - sum < left;
        if (lane == 0) s_digit = -1;
        __syncwarp();
        if (crosses) {
          int before = up_to - sum, i = 0;
          while (before + mine[i] < left) before += mine[i++];
          s_digit = 255 - 8 * lane - i;
          s_left = left - before;
        }
      }
      __syncthreads();
      if (s_digit < 0) break;  // fewer candidates than are asked for: only in the first round, as all are then taken
      least = (known == 0 ? 0u : least & known) | (uint32_t)s_digit << shift;
      known |= 255u << shift;
      left = s_left;
    }
    if (known == 0) left = p.count;
  }
  const bool all = known == 0;  // every candidate is taken
  __syncthreads();
  // ---- in order ------------------------------------------------------------------------------------------------------------------
  const int begin = min((int)threadIdx.x * run, n), end = min(begin + run, n);
  int above = 0, equal = 0;
  for (int i = begin; i < end; ++i) {
    const uint32_t x = score(i);
    above += all ? x != 0 : x > least;
    equal += !all && x == least;
  }
  const int mine_above = above, mine_equal = equal;
  q8_scan2(above, equal, s_sums);
  int at = above + min(equal, left), ties = equal;
  for (int i = begin; i < end; ++i) {
    const uint32_t x = score(i);
    if (all ? x != 0 : x > least) {
      out[at++] = i;
    } else if (!all && x == least) {
      if (ties++ < left) out[at++] = i;
    }
  }
  if (threadIdx.x == kQ8PickThreads - 1) s_digit = above + mine_above + min(equal + mine_equal, all ? 0 : left);
  __syncthreads();
  for (int i = s_digit + threadIdx.x; i < p.count; i += kQ8PickThreads) out[i] = -1;
}

}  // namespace anna

using namespace anna;

extern "C" int anna_q8_select_blocks(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, const uint8_t* pages,
                                     const int32_t* page_table, int64_t table_stride, const int64_t* lengths, int32_t* blocks, int count,
                                     int first, int recent, uint32_t* scores, int batch, int q_heads, int kv_heads, int tokens,
                                     int head_dim, int block_size, int64_t num_pages, int64_t max_blocks, int dtype,
                                     anna_stream_t stream) {
  const char* what = "anna_q8_select_blocks";
  int64_t bytes = 0;
  if (const int rc = anna_q8_page_bytes(head_dim, block_size, &bytes)) return rc;
  ANNA_REQUIRE(q && lengths && blocks, "%s: null pointer argument", what);
  ANNA_REQUIRE(batch > 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 && tokens > 0 && max_blocks >= 0, "%s: bad sizes", what);
  ANNA_REQUIRE(max_blocks == 0 || (pages && page_table && scores && num_pages > 0), "%s: a block table needs pages and scores", what);
  ANNA_REQUIRE(count > 0 && first >= 0 && recent >= 0 && first <= count && recent <= count - first,
               "%s: count must be positive and have room for the first and recent pages", what);
  ANNA_REQUIRE(aligned_to(pages, 16), "%s: pages must be 16-byte aligned", what);
  ANNA_REQUIRE(max_blocks < (1ll << 30) / block_size - 1, "%s: too many pages", what);
  const int64_t streams = (int64_t)batch * kv_heads * tokens;
  ANNA_REQUIRE(streams < (1ll << 31) && (int64_t)batch * kv_heads < 65536, "%s: too many queries", what);
  Q8SelectParams p{};
  p.q = q; p.q_stride_b = batch > 1 ? q_stride_b : 0; p.q_stride_h = q_heads > 1 ? q_stride_h : 0; p.q_stride_t = tokens > 1 ? q_stride_t : 0;
  p.pages = pages; p.block_table = page_table; p.table_stride = table_stride; p.lengths = lengths; p.blocks = blocks; p.scores = scores;
  p.kv_heads = kv_heads; p.groups = q_heads / kv_heads; p.tokens = tokens; p.block_size = block_size; p.page_bytes = (int)bytes;
  p.count = count; p.first = first; p.recent = recent; p.num_pages = num_pages; p.max_blocks = max_blocks;
  p.head_tiles = (p.groups + 7) / 8;
  p.tokens_at_once = p.head_tiles >= 8 ? 1 : 8 / p.head_tiles;
  if (p.tokens_at_once > tokens) p.tokens_at_once = tokens;
  const int row_tiles = p.tokens_at_once * p.head_tiles;
  const int smem = row_tiles * (2 * (2 * head_dim / 64) * 512 + 32);
  if (smem > 200 * 1024) return set_error(ANNA_ERR_UNSUPPORTED, "%s: too many query heads (%d) to a KV head", what, p.groups);
  const int chunks = (tokens + p.tokens_at_once - 1) / p.tokens_at_once;
  ANNA_REQUIRE(chunks < 65536, "%s: too many tokens", what);
  if (max_blocks > 0) {
    const int64_t tiles = (max_blocks + kQ8SelectTile - 1) / kQ8SelectTile, most = (tiles + kQ8SelectWarps - 1) / kQ8SelectWarps;
    int64_t splits = 148 * 2 / ((int64_t)batch * kv_heads * chunks);
    splits = splits < 1 ? 1 : splits > most ? most : splits;
    const int rc = ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
        auto kernel = q8_score_kernel<T, D>;
        ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        kernel<<<dim3((unsigned)splits, (unsigned)(batch * kv_heads), (unsigned)chunks), kQ8SelectWarps * 32, smem, (cudaStream_t)stream>>>(p);
        return check_launch("q8_score_kernel");
      });
    });
    if (rc != ANNA_OK) return rc;
  }
  if (max_blocks <= kQ8PickHeld) {
    const int held = (int)(max_blocks + max_blocks / 32 + 1) * 4;
    ANNA_CUDA_CHECK(cudaFuncSetAttribute(q8_pick_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kQ8PickHeld + kQ8PickHeld / 32 + 1) * 4));
    q8_pick_kernel<true><<<(unsigned)streams, kQ8PickThreads, held, (cudaStream_t)stream>>>(p);
  } else {
    q8_pick_kernel<false><<<(unsigned)streams, kQ8PickThreads, 0, (cudaStream_t)stream>>>(p);
  }
  return check_launch("q8_pick_kernel");
}
