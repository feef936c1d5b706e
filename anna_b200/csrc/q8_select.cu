// Selection of the pages that a query should look at, by a bound on its products with their keys.
//
// With high_d and low_d the largest and smallest code of dim d in a page, sum_d max(r_d high_d, r_d low_d) bounds r . code from above for
// every key of the page.  r is the query in whole numbers of 15 bits and a sign, so the sum is one, below 2^31: no order of summation
// changes it, and a score is the same wherever it is worked out.  With r+ = max(r, 0), r- = max(-r, 0) and the page's bounds
// [high, -low] the sum is one product of 2 D, [r+, r-] . [high, -low], of non-negative numbers of 15 bits, as two bytes (128 u + v,
// u < 256, v < 128), with signed bytes: integer mma, 16 pages to a tile, 8 query heads.
//
// Scores: a warp takes 16 pages at a time, for all heads and several tokens.  Bound: HBM (2 D + 4 bytes a page and head), or the launch.
// Choice: a CTA per query token and KV head finds the score of the last page that is taken, 8 bits at a time from the first bit in which
// scores differ, counting how many share the bits so far; then the pages above it, and of those equal to it the first, are written in order.
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
  int rounds;                      // tiles of a warp
  int64_t num_pages, max_blocks;
};

constexpr int kQ8SelectWarps = 8;
constexpr int kQ8SelectTile = 16;  // pages of a warp at a time
constexpr int kQ8SelectRounds = 8;   // tiles of a warp at most
constexpr uint32_t kQ8Forced = 0xffffffffu;

// Full pages of which query t sees a token.
__device__ __forceinline__ int q8_candidates(const Q8SelectParams& p, int64_t b, int t) {
  const int len = (int)max((int64_t)0, min(p.lengths[b], p.max_blocks * p.block_size + p.block_size - 1));  // below 2^30
  const int seen = len - p.tokens + t + 1;
  return seen <= 0 ? 0 : min(len / p.block_size, (seen + p.block_size - 1) / p.block_size);
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
__global__ void __launch_bounds__(kQ8SelectWarps * 32, D == 256 ? 1 : 2) q8_score_kernel(const Q8SelectParams p) {
  constexpr int kChunks = 2 * D / 64;  // of 64 bounds, 16 of them a lane's
  extern __shared__ __align__(16) uint8_t smem[];
  q8_let_next_start();
  q8_wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int b = blockIdx.y / p.kv_heads, kvh = blockIdx.y - b * p.kv_heads;
  const int token0 = blockIdx.z * p.tokens_at_once, here = min(p.tokens_at_once, p.tokens - token0);
  const int head_tiles = p.head_tiles, tiles = here * head_tiles;
  uint4* parts = reinterpret_cast<uint4*>(smem);                                              // [2][tiles][kChunks][32 lanes]
  float* tops = reinterpret_cast<float*>(smem + p.tokens_at_once * head_tiles * 2 * kChunks * 512);  // [tiles][8]

  // ---- this CTA's pages: `rounds` tiles of every warp -----------------------------------------------------------------------------------
  __shared__ int candidates_of[8];
  if (threadIdx.x < here) candidates_of[threadIdx.x] = q8_candidates(p, b, token0 + threadIdx.x);
  const int most = q8_candidates(p, b, token0 + here - 1);
  const int first_tile = blockIdx.x * p.rounds * kQ8SelectWarps + warp;
  if ((int)blockIdx.x * p.rounds * kQ8SelectWarps * kQ8SelectTile >= most) return;
  struct Tile {
    uint4 w[2][kChunks];
    float scale[2];
    bool there[2];
  };
  int32_t ids[2];  // pages of the tile after next
  auto find = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = tile * kQ8SelectTile + gid + 8 * i;
      ids[i] = j < most ? p.block_table[(int64_t)b * p.table_stride + j] : -1;
    }
  };
  auto load = [&](Tile& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x.there[i] = ids[i] >= 0 && ids[i] < p.num_pages;
      const uint8_t* page = p.pages + (x.there[i] ? ((int64_t)ids[i] * p.kv_heads + kvh) * p.page_bytes : 0);
      x.scale[i] = __ldg(reinterpret_cast<const float*>(page + q8_scale_offset(D, p.block_size)));
      const uint4* bounds = reinterpret_cast<const uint4*>(page + q8_bounds_offset(D, p.block_size));
#pragma unroll
      for (int c = 0; c < kChunks; ++c) x.w[i][c] = ldg_stream16(bounds + 4 * c + tig);
    }
  };
  Tile now, next;
  find(first_tile);
  load(now);
  find(first_tile + kQ8SelectWarps);

  // ---- queries in whole numbers --------------------------------------------------------------------------------------------------
  for (int row = warp; row < tiles * 8; row += kQ8SelectWarps) {
    const int t = row / (8 * head_tiles), g = row % (8 * head_tiles);
    float x[D / 32], top = 0.0f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      x[j] = 0.0f;
      if (g < p.groups)
        x[j] = ElemTraits<T>::to_float(reinterpret_cast<const T*>(p.q)[(int64_t)b * p.q_stride_b + (int64_t)(kvh * p.groups + g) * p.q_stride_h +
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
  for (int round = 0; round < p.rounds; ++round) {
    const int tile = first_tile + round * kQ8SelectWarps;
    if (tile * kQ8SelectTile >= most) break;
    if (round + 1 < p.rounds) {
      load(next);
      find(tile + 2 * kQ8SelectWarps);
    }
    for (int t = 0; t < here; ++t) {
      float best[2] = {-INFINITY, -INFINITY};
      for (int h = 0; h < head_tiles; ++h) {
        int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
        const uint4* at = parts + (t * head_tiles + h) * kChunks * 32 + lane;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint4 u = at[c * 32], v = at[(tiles * kChunks + c) * 32];
          mma_s8u8(hi, now.w[0][c].x, now.w[1][c].x, now.w[0][c].y, now.w[1][c].y, u.x, u.y);
          mma_s8u8(lo, now.w[0][c].x, now.w[1][c].x, now.w[0][c].y, now.w[1][c].y, v.x, v.y);
          mma_s8u8(hi, now.w[0][c].z, now.w[1][c].z, now.w[0][c].w, now.w[1][c].w, u.z, u.w);
          mma_s8u8(lo, now.w[0][c].z, now.w[1][c].z, now.w[0][c].w, now.w[1][c].w, v.z, v.w);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int g = h * 8 + 2 * tig + (r & 1);
          if (g >= p.groups) continue;
          const float top = tops[(t * head_tiles + h) * 8 + 2 * tig + (r & 1)];
          const float x = __fmul_rn(__fmul_rn(top, now.scale[r / 2]), __int2float_rn(128 * hi[r] + lo[r]));
          best[r / 2] = isnan(x) ? INFINITY : fmaxf(best[r / 2], x);
        }
      }
      const int candidates = candidates_of[t];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
        const int j = tile * kQ8SelectTile + gid + 8 * i;
        if (tig == 0 && j < candidates) {
          const bool forced = j < p.first || j >= candidates - p.recent;
          p.scores[((int64_t)blockIdx.y * p.tokens + token0 + t) * p.max_blocks + j] = !now.there[i] ? 0u : forced ? kQ8Forced : q8_ordered(best[i]);
        }
      }
    }
    now = next;
  }
}

// A CTA's choice of a query token and KV head.  kHeld scores a thread are kept in registers, thread i has the scores i, i + THREADS, ...; with
// kHeld = 0 they are read again wherever they are looked at.
template <int THREADS, int kHeld>
__global__ void __launch_bounds__(THREADS) q8_pick_kernel(const Q8SelectParams p) {
  constexpr int kWarps = THREADS / 32, kRounds = kHeld == 0 ? 1 : kHeld;
  __shared__ int histogram[256], s_before[kRounds * kWarps], s_digit, s_left, s_same, s_taken;
  __shared__ uint32_t s_high[kWarps], s_low[kWarps];
  __shared__ int s_some[kWarps];
  q8_let_next_start();
  q8_wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t stream = blockIdx.x;
  const int head = blockIdx.x / p.tokens, b = head / p.kv_heads;
  const int n = q8_candidates(p, b, blockIdx.x - head * p.tokens);
  const uint32_t* scores = p.scores + stream * p.max_blocks;
  int32_t* out = p.blocks + stream * p.count;
  const int rounds = (n + THREADS - 1) / THREADS;
  uint32_t held[kRounds] = {};
  auto score = [&](int k) {
    const int i = k * THREADS + (int)threadIdx.x;
    return i < n ? __ldcg(scores + i) : 0u;
  };
  auto each = [&](auto&& fn) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int k = 0; k < kRounds; ++k) fn(k, held[k]);
    } else {
      for (int k = 0; k < rounds; ++k) fn(k, score(k));
    }
  };
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int k = 0; k < kRounds; ++k) held[k] = score(k);
  }
  // ---- pages with a score above `least` are taken, and of those with that score the first `left` ----------------------------------------
  uint32_t least = 0;
  int left = 0;
  if (n > p.count) {
    uint32_t high = 0, low = 0xffffffffu;
    int some = 0;
    each([&](int, uint32_t x) {
      high = max(high, x);
      low = min(low, x - 1u);  // 0 is no candidate
      some += x != 0;
    });
    high = __reduce_max_sync(0xffffffffu, high);
    low = __reduce_min_sync(0xffffffffu, low);
    some = __reduce_add_sync(0xffffffffu, some);
    if (lane == 0) {
      s_high[warp] = high;
      s_low[warp] = low;
      s_some[warp] = some;
    }
    __syncthreads();
    some = 0;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      high = max(high, s_high[v]);
      low = min(low, s_low[v]);
      some += s_some[v];
    }
    low += 1u;
    if (some > p.count) {
      // `known`: the bits that all scores share, and further down those of the score that is looked for
      int bits = high == low ? 0 : 32 - __clz(high ^ low);  // still unknown
      uint32_t known = bits == 32 ? 0u : 0xffffffffu << bits;
      least = high & known;
      left = p.count;
      while (bits > 0) {
        const int width = min(bits, 8), shift = bits - width;
        for (int i = threadIdx.x; i < 256; i += THREADS) histogram[i] = 0;
        __syncthreads();
        each([&](int, uint32_t x) {
          if (x != 0 && (x & known) == least) atomicAdd(&histogram[(x >> shift) & ((1u << width) - 1u)], 1);
        });
        __syncthreads();
        if (threadIdx.x < 32) {  // a lane has eight digits, the largest first
          int mine[8], sum = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += mine[i] = histogram[255 - 8 * lane - i];
          int up_to = sum;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, up_to, d);
            if (lane >= d) up_to += v;
          }
          if (up_to >= left && up_to - sum < left) {
            int before = up_to - sum;
            bool found = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (!found && before + mine[i] >= left) {
                found = true;
                s_digit = 255 - 8 * lane - i;
                s_left = left - before;
                s_same = mine[i];
              }
              before += mine[i];
            }
          }
        }
        __syncthreads();
        least |= (uint32_t)s_digit << shift;
        known |= ((1u << width) - 1u) << shift;
        left = s_left;
        bits = shift;
        if (s_same == left && least != 0) {  // all that share these bits are taken
          least -= 1u;
          left = 0;
          break;
        }
      }
    }
  }
  // ---- in order: scores of a round of a warp, 32 neighbours, are counted by votes --------------------------------------------------------
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const unsigned above = __ballot_sync(0xffffffffu, held[k] > least), same = __ballot_sync(0xffffffffu, held[k] == least && held[k] != 0);
      if (lane == 0) s_before[k * kWarps + warp] = __popc(above) | __popc(same) << 16;
    }
    __syncthreads();
    if (warp == 0) {  // no more than 2^14 scores are held, so both counts fit into 16 bits
      constexpr int kEach = (kRounds * kWarps + 31) / 32;
      int mine[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int at = lane * kEach + i;
        mine[i] = at < kRounds * kWarps ? s_before[at] : 0;
        sum += mine[i];
      }
      int up_to = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up_to, d);
        if (lane >= d) up_to += v;
      }
      int before = up_to - sum;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int at = lane * kEach + i;
        if (at < kRounds * kWarps) s_before[at] = before;
        before += mine[i];
      }
      if (lane == 31) s_taken = (up_to & 0xffff) + min(up_to >> 16, left);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const bool is_above = held[k] > least, is_same = held[k] == least && held[k] != 0;
      const unsigned above = __ballot_sync(0xffffffffu, is_above), same = __ballot_sync(0xffffffffu, is_same);
      const unsigned before = (1u << lane) - 1u;
      const int base = s_before[k * kWarps + warp];
      const int rank = (base & 0xffff) + __popc(above & before), ties = (base >> 16) + __popc(same & before);
      if (is_above || (is_same && ties < left)) out[rank + min(ties, left)] = k * THREADS + (int)threadIdx.x;
    }
  } else {
    int taken = 0, ties = 0;  // in front of the round
    for (int k = 0; k < rounds; ++k) {
      const uint32_t x = score(k);
      const bool is_above = x > least, is_same = x == least && x != 0;
      const unsigned above = __ballot_sync(0xffffffffu, is_above), same = __ballot_sync(0xffffffffu, is_same);
      if (lane == 0) s_before[warp] = __popc(above) | __popc(same) << 16;
      __syncthreads();
      int rank = taken, tie = ties;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const int c = s_before[v];
        if (v < warp) {
          rank += c & 0xffff;
          tie += c >> 16;
        }
        taken += c & 0xffff;
        ties += c >> 16;
      }
      const unsigned before = (1u << lane) - 1u;
      rank += __popc(above & before);
      tie += __popc(same & before);
      if (is_above || (is_same && tie < left)) out[rank + min(tie, left)] = k * THREADS + (int)threadIdx.x;
      __syncthreads();
    }
    if (threadIdx.x == 0) s_taken = taken + min(ties, left);
  }
  __syncthreads();
  for (int i = s_taken + threadIdx.x; i < p.count; i += THREADS) out[i] = -1;
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
    // one wave where the pages are that few; a CTA whose pages lie behind its row's end leaves at once
    const int64_t tiles = (max_blocks + kQ8SelectTile - 1) / kQ8SelectTile, wave = 148 * (head_dim == 256 ? 1 : 2) * kQ8SelectWarps;
    const int64_t rounds = ((int64_t)batch * kv_heads * chunks * tiles + wave - 1) / wave;
    p.rounds = (int)(rounds > kQ8SelectRounds ? kQ8SelectRounds : rounds);
    const int64_t splits = (tiles + p.rounds * kQ8SelectWarps - 1) / (p.rounds * kQ8SelectWarps);
    const int rc = ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
        auto kernel = q8_score_kernel<T, D>;
        ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return q8_launch("q8_score_kernel", kernel, dim3((unsigned)splits, (unsigned)(batch * kv_heads), (unsigned)chunks), kQ8SelectWarps * 32,
                         smem, (cudaStream_t)stream, p);
      });
    });
    if (rc != ANNA_OK) return rc;
  }
  auto pick = [&](auto kernel, int threads) {
    return q8_launch("q8_pick_kernel", kernel, dim3((unsigned)streams), threads, 0, (cudaStream_t)stream, p);
  };
  if (max_blocks <= 1024) return pick(q8_pick_kernel<256, 4>, 256);
  if (max_blocks <= 2048) return pick(q8_pick_kernel<256, 8>, 256);
  if (max_blocks <= 4096) return pick(q8_pick_kernel<512, 8>, 512);
  if (max_blocks <= 8192) return pick(q8_pick_kernel<1024, 8>, 1024);
  if (max_blocks <= 16384) return pick(q8_pick_kernel<1024, 16>, 1024);
  return pick(q8_pick_kernel<1024, 0>, 1024);
}
