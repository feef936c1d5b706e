// Selection of the pages that a query should look at, by a bound on its products with their keys.
//
// With high_d and low_d the largest and smallest code of dim d in a page, sum_d max(r_d high_d, r_d low_d) bounds r . code from above for
// every key of the page.  r is the query in whole numbers of 15 bits and a sign, so the sum is one, below 2^31: no order of summation
// changes it, and a score is the same wherever it is worked out.  With r+ = max(r, 0), r- = max(-r, 0) and the page's bounds
// [high, -low] the sum is one product of 2 D, [r+, r-] . [high, -low], of non-negative numbers of 15 bits, as two bytes (128 u + v,
// u < 256, v < 128), with signed bytes: integer mma, 16 pages to a tile, 8 query heads.
//
// Scores: a warp takes 16 pages at a time, for all heads and several tokens.  Bound: HBM (2 D + 4 bytes a page and head), or the launch.
// Choice: a CTA per query token and KV head finds the score of the last page that is taken, in a 256th of the scores' range at a time, counting how many
// lie in each, until a warp holds all that are left; then the pages above it, and of those equal to it the first, are written in order.
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
  int row_group;       // rows of a token: its query heads, padded to 8 where they do not divide 8; see q8_score_kernel
  int group_shift, head_tiles;  // log2 of rows of a token in one tile; tiles of a token that has more
  int tokens_at_once;  // of a CTA
  int heads_at_once;   // KV heads of a CTA
  int batch, chunks, head_groups;  // chunks of tokens_at_once, groups of heads_at_once
  int part_tiles;      // of a CTA, where CTAs take parts
  int64_t num_pages, max_blocks;
};

constexpr int kQ8SelectWarps = 8;
constexpr int kQ8SelectTile = 16;  // pages of a warp at a time
constexpr int kQ8SelectCost = 4;     // tiles, of all KV heads of a CTA
constexpr int kQ8SelectRows = 64;    // rows of a CTA, where a token has no more
template <int D>
constexpr int kQ8SelectCtas = D == 256 ? 1 : 3;
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

// 16 bytes that are read once, coherently (see q8_wait_for_previous); half lines are fetched from memory, as bounds end a little way into a line (320 bytes a
// page of 128 dims instead of 384).  (Past L1, as ld.global.cg: 32 rows of 20000 to 32768 tokens and the attention behind it take 5.5 us more.)
__device__ __forceinline__ uint4 q8_load64(const uint4* ptr) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::64B.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(ptr));
  return v;
}
// Order of floats as order of whole numbers, none of them 0.
__device__ __forceinline__ uint32_t q8_ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// The whole number next to 32767 x / top, of two the even one; 0 where top is.  Of 16-bit values (11 bits) in 32 bits: the quotient is off by less than
// 0.01, and what 32767 x exceeds n top by is exact, a product in two parts less another (the first difference has no more than 24 bits, as n top and
// 32767 x lie that close).  (32-bit arithmetic, as the GPU has few units for 64 bits: the time of a
// call is the same within 0.3 us with what fp32 values take.)
template <typename T>
struct Q8Whole {
  float factor, top, rate;
  __device__ __forceinline__ explicit Q8Whole(float most) {
    const int up = most > 0.0f ? min(max(127 - (int)(__float_as_uint(most) >> 23), -126), 126) : 0;  // top is in [1, 4), or all is as good as 0
    factor = __uint_as_float((uint32_t)(up + 127) << 23);
    top = most * factor;
    rate = most > 0.0f ? __fdiv_rn(32767.0f, top) : 0.0f;
  }
  __device__ __forceinline__ int whole(float value) const {
    const float x = value * factor, n = rintf(x * rate);
    const float product = __fmul_rn(32767.0f, x), rest = __fmaf_rn(32767.0f, x, -product);
    const float over = __fadd_rn(__fmaf_rn(-n, top, product), rest), half = 0.5f * top;
    const int i = __float2int_rn(n);
    const bool odd = i & 1;
    return i + (over > half || (over == half && odd) ? 1 : 0) - (over < -half || (over == -half && odd) ? 1 : 0);
  }
};
// fp32 values: a quotient that is no tie is at least 2^-40 of its power of two away from one, the product is off by 2^-51 of it at most; rounded to 45 bits
// (as q8_append.cu does it) ties are ties again.
template <>
struct Q8Whole<float> {
  double rate;
  __device__ __forceinline__ explicit Q8Whole(float top) { rate = top > 0.0f ? 32767.0 / (double)top : 0.0; }
  __device__ __forceinline__ int whole(float value) const {
    const double r = __dmul_rn((double)value, rate), c = __dmul_rn(r, 257.0);
    return __double2int_rn(__dsub_rn(c, __dsub_rn(c, r)));
  }
};

// Rows are the query heads of several tokens, one behind the other: the heads of a token are in one tile of 8 rows where their number divides 8, else
// a token has tiles of its own.  The KV heads of a page lie next to one another, and a CTA's warps take them together: a page costs one translation of its
// address and one stretch of memory (32 rows of 20000 to 32768 tokens in scattered pages, 8 KV heads: 34.5 us, 45.6 with CTAs of one
// KV head).
//
// CTAs: a part of a stream (sequence, tokens, KV heads) each where the GPU holds them all at once; else one resident wave that takes even shares of the
// line of all streams' tiles, kQ8SelectCost tiles in front of each for its queries.
template <typename T, int D, bool kShares>
__global__ void __launch_bounds__(kQ8SelectWarps * 32, kQ8SelectCtas<D>) q8_score_kernel(const Q8SelectParams p) {
  constexpr int kChunks = 2 * D / 64;  // of 64 bounds, 16 of them a lane's
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int candidates_of[kQ8SelectRows];
  __shared__ int s_prefix[kShares ? kBalancedMaxRows + 1 : 1];
  q8_wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;

  // The pages of tiles [begin, end) of 16, for a chunk of tokens and a group of KV heads of row b.
  auto segment = [&](int b, int stream, int begin, int end) {
  const int heads0 = stream / p.chunks * p.heads_at_once, heads = min(p.heads_at_once, p.kv_heads - heads0);
  const int token0 = stream % p.chunks * p.tokens_at_once, here = min(p.tokens_at_once, p.tokens - token0);
  const int tiles = (here * p.row_group + 7) / 8;                                           // of a KV head
  uint4* parts = reinterpret_cast<uint4*>(smem);                                            // [2][heads][tiles][kChunks][32 lanes]
  float* tops = reinterpret_cast<float*>(smem + heads * tiles * 2 * kChunks * 512);         // [heads][tiles][8]
  const int plane = heads * tiles * kChunks * 32;
  const int most = q8_candidates(p, b, token0 + here - 1);
  if ((int)threadIdx.x < here) candidates_of[threadIdx.x] = q8_candidates(p, b, token0 + threadIdx.x);
  // this warp's items: tiles with their KV heads, these first
  int tile = begin + warp / heads, head = warp % heads;
  const int tile_step = kQ8SelectWarps / heads, head_step = kQ8SelectWarps - tile_step * heads;
  int32_t ids[2];  // pages of the next item
  auto find = [&](int of) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = of * kQ8SelectTile + gid + 8 * i;
      ids[i] = of < end && j < most ? p.block_table[(int64_t)b * p.table_stride + j] : -1;
    }
  };
  uint4 w[2][kChunks];
  float scale[2];
  bool there[2];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      there[i] = ids[i] >= 0 && ids[i] < p.num_pages;
      const uint8_t* page = p.pages + (there[i] ? ((int64_t)ids[i] * p.kv_heads + heads0 + h) * p.page_bytes : 0);
      scale[i] = *reinterpret_cast<const float*>(page + q8_scale_offset(D, p.block_size));
      const uint4* bounds = reinterpret_cast<const uint4*>(page + q8_bounds_offset(D, p.block_size));
#pragma unroll
      for (int c = 0; c < kChunks; ++c) w[i][c] = q8_load64(bounds + 4 * c + tig);
    }
  };
  auto next_tile = [&] { return tile + tile_step + (head + head_step >= heads ? 1 : 0); };
  // queries: the first of them are asked for ahead of the bounds, behind which they would wait
  const int of_head = here * p.groups, rows = heads * of_head;
  constexpr int kAhead = 4;  // rows on their way
  constexpr int E = D / 32;  // neighbouring dims of a lane
  T raw[kAhead][E];
  int place_of[kAhead];
  auto fetch = [&](int from) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int row = min(from + k, rows - 1), h = row / of_head, t = (row - h * of_head) / p.groups, g = row - h * of_head - t * p.groups;
      place_of[k] = 8 * h * tiles + t * p.row_group + g;
      const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_stride_b + (int64_t)((heads0 + h) * p.groups + g) * p.q_stride_h +
                   (int64_t)(token0 + t) * p.q_stride_t + lane * E;
#pragma unroll
      for (int j = 0; j < E; ++j) raw[k][j] = q[j];
    }
  };
  find(tile);
  fetch(warp * kAhead);
  load(head);
  find(next_tile());

  // ---- queries in whole numbers; rows that are not there stay as they are --------------------------------------------------------------
  for (int from = warp * kAhead; from < rows; from += kQ8SelectWarps * kAhead) {
    if (from > warp * kAhead) fetch(from);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (from + k >= rows) break;
      float x[E], top = 0.0f;
      bool fine = true;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        x[j] = ElemTraits<T>::to_float(raw[k][j]);
        top = fmaxf(top, fabsf(x[j]));
        fine = fine && fabsf(x[j]) < INFINITY;
      }
      top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
      fine = __all_sync(0xffffffffu, fine);
      if (lane == 0) tops[place_of[k]] = fine ? top : __int_as_float(0x7fc00000);
      const Q8Whole<T> rounder(fine ? top : 0.0f);
      uint32_t upper[2][(E + 3) / 4] = {}, lower[2][(E + 3) / 4] = {};  // bytes of positive and of negative numbers
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int whole = fine ? rounder.whole(x[j]) : 0;
#pragma unroll
        for (int negated = 0; negated < 2; ++negated) {
          const uint32_t n = (uint32_t)max(negated ? -whole : whole, 0);
          upper[negated][j / 4] |= (n >> 7) << (8 * (j % 4));
          lower[negated][j / 4] |= (n & 127u) << (8 * (j % 4));
        }
      }
      const int d = lane * E;
#pragma unroll
      for (int negated = 0; negated < 2; ++negated) {
        uint8_t* to = smem + ((place_of[k] / 8 * kChunks + d / 64 + negated * (D / 64)) * 32 + place_of[k] % 8 * 4 + d % 64 / 16) * 16 + d % 16;
        if constexpr (E == 2) {
          *reinterpret_cast<uint16_t*>(to) = (uint16_t)upper[negated][0];
          *reinterpret_cast<uint16_t*>(to + plane * 16) = (uint16_t)lower[negated][0];
        } else if constexpr (E == 4) {
          *reinterpret_cast<uint32_t*>(to) = upper[negated][0];
          *reinterpret_cast<uint32_t*>(to + plane * 16) = lower[negated][0];
        } else {
          *reinterpret_cast<uint2*>(to) = make_uint2(upper[negated][0], upper[negated][E / 4 - 1]);
          *reinterpret_cast<uint2*>(to + plane * 16) = make_uint2(lower[negated][0], lower[negated][E / 4 - 1]);
        }
      }
    }
  }
  __syncthreads();

  // ---- 16 pages of a KV head at a time ---------------------------------------------------------------------------------------------------
  for (bool first = true; tile < end && tile * kQ8SelectTile < most; first = false) {
    if (!first) {
      load(head);
      find(next_tile());
    }
    uint32_t* scores = p.scores + (((int64_t)b * p.kv_heads + heads0 + head) * p.tokens + token0) * p.max_blocks;
    float best[2] = {-INFINITY, -INFINITY};  // of one token
    for (int n = 0, t0 = 0, h = 0; n < tiles; ++n) {
      int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
      const uint4* at = parts + (head * tiles + n) * kChunks * 32 + lane;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint4 u = at[c * 32], v = at[plane + c * 32];
        mma_s8u8(hi, w[0][c].x, w[1][c].x, w[0][c].y, w[1][c].y, u.x, u.y);
        mma_s8u8(lo, w[0][c].x, w[1][c].x, w[0][c].y, w[1][c].y, v.x, v.y);
        mma_s8u8(hi, w[0][c].z, w[1][c].z, w[0][c].w, w[1][c].w, u.z, u.w);
        mma_s8u8(lo, w[0][c].z, w[1][c].z, w[0][c].w, w[1][c].w, v.z, v.w);
      }
      const float2 top = *reinterpret_cast<const float2*>(tops + 8 * (head * tiles + n) + 2 * tig);
      float x[4];  // rows 2 tig and 2 tig + 1 of pages gid and gid + 8
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = __fmul_rn(__fmul_rn(r & 1 ? top.y : top.x, scale[r / 2]), __int2float_rn(128 * hi[r] + lo[r]));
        if (isnan(x[r])) x[r] = INFINITY;
      }
      auto put = [&](int t, int i, float score) {  // of token t and page gid + 8 i
        const int j = tile * kQ8SelectTile + gid + 8 * i, candidates = candidates_of[t];
        if (j >= candidates) return;
        const bool forced = j < p.first || j >= candidates - p.recent;
        scores[(int64_t)t * p.max_blocks + j] = !there[i] ? 0u : forced ? kQ8Forced : q8_ordered(score);
      };
      if (p.group_shift == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (8 * n + 2 * tig + (r & 1) < here) put(8 * n + 2 * tig + (r & 1), r / 2, x[r]);
        continue;
      }
      if (p.group_shift == 3) {  // rows past a token's heads
        const int g = 8 * h + 2 * tig;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (g >= p.groups) x[2 * i] = -INFINITY;
          if (g + 1 >= p.groups) x[2 * i + 1] = -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float score = fmaxf(x[2 * i], x[2 * i + 1]);
        if (p.group_shift >= 2) score = fmaxf(score, __shfl_xor_sync(0xffffffffu, score, 1));
        if (p.group_shift == 3) score = fmaxf(score, __shfl_xor_sync(0xffffffffu, score, 2));
        best[i] = fmaxf(best[i], score);
      }
      if (++h < p.head_tiles) continue;  // more tiles of this token follow
      const int t = t0 + (2 * tig >> p.group_shift);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (t < here && (2 * tig & ((1 << p.group_shift) - 1)) == 0) put(t, i, best[i]);
        best[i] = -INFINITY;
      }
      t0 += 8 >> p.group_shift;
      h = 0;
    }
    tile = next_tile();
    head += head_step - (head + head_step >= heads ? heads : 0);
  }
  };

  if constexpr (!kShares) {
    const int begin = blockIdx.x * p.part_tiles;
    if (begin * kQ8SelectTile < q8_candidates(p, blockIdx.y, p.tokens - 1)) segment(blockIdx.y, blockIdx.z, begin, begin + p.part_tiles);
  } else {
    // at most 32 rows are lined up by every warp by itself
    constexpr int kThreads = kQ8SelectWarps * 32;
    const bool few = p.batch <= 32;
    const int per_row = p.chunks * p.head_groups;
    auto tiles_of = [&](int b) { return b < p.batch ? (q8_candidates(p, b, p.tokens - 1) + kQ8SelectTile - 1) / kQ8SelectTile : 0; };
    WarpLine line{};
    int total;
    if (few) {
      line.tiles = tiles_of(lane);
      total = line.scan(per_row, kQ8SelectCost, 0);
    } else {
      const int each = (p.batch + kThreads - 1) / kThreads;
      int tiles_of_rows[kBalancedRowsPerThread<kThreads>], streams;
#pragma unroll
      for (int i = 0; i < kBalancedRowsPerThread<kThreads>; ++i) tiles_of_rows[i] = i < each ? tiles_of(threadIdx.x * each + i) : 0;
      balanced_scan<kThreads>(tiles_of_rows, p.batch, per_row, s_prefix, kQ8SelectCost, 0, &streams);
      total = s_prefix[p.batch];
    }
    const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
    int pos = (int)min((int64_t)blockIdx.x * share, (int64_t)total), b = 0;
    const int stop = min(pos + share, total);
    if (!few && pos < stop) {
      int above = p.batch;  // s_prefix[b] <= pos < s_prefix[above]
      while (above - b > 1) {
        const int mid = (b + above) >> 1;
        if (s_prefix[mid] <= pos) b = mid;
        else above = mid;
      }
    }
    while (pos < stop) {
      int first, n;  // positions in front of the row; of a stream, its cost among them
      if (few) {
        b = __popc(__ballot_sync(0xffffffffu, line.next <= pos));
        first = __shfl_sync(0xffffffffu, line.first, b);
        n = __shfl_sync(0xffffffffu, line.tiles, b) + kQ8SelectCost;
      } else {
        while (s_prefix[b + 1] <= pos) ++b;
        first = s_prefix[b];
        n = (s_prefix[b + 1] - first) / per_row;
      }
      const int stream = (pos - first) / n, at = pos - first - stream * n, to = min(n, at + stop - pos);
      if (to > kQ8SelectCost) {
        segment(b, stream, max(0, at - kQ8SelectCost), to - kQ8SelectCost);
        __syncthreads();  // queries and candidates have been read
      }
      pos += to - at;
    }
  }
}

// A CTA's choice of a query token and KV head.  kHeld scores a thread are kept in registers, thread i has the scores i, i + THREADS, ...; with
// kHeld = 0 they are read again wherever they are looked at.
template <int THREADS, int kHeld>
__global__ void __launch_bounds__(THREADS) q8_pick_kernel(const Q8SelectParams p) {
  constexpr int kWarps = THREADS / 32, kRounds = kHeld == 0 ? 1 : kHeld;
  __shared__ int histogram[256], s_before[kRounds * kWarps], s_digit, s_left, s_same, s_taken, s_few;
  __shared__ uint32_t s_high[kWarps], s_low[kWarps], few[32];
  __shared__ int s_some[kWarps], s_forced[kWarps];
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
    // of those that are not taken in any case
    uint32_t high = 0, low = 0xffffffffu;
    int some = 0, forced = 0;
    each([&](int, uint32_t x) {
      high = max(high, x == kQ8Forced ? 0u : x);
      low = min(low, x - 1u);  // 0 is no candidate
      some += x != 0;
      forced += x == kQ8Forced;
    });
    high = __reduce_max_sync(0xffffffffu, high);
    low = __reduce_min_sync(0xffffffffu, low);
    some = __reduce_add_sync(0xffffffffu, some);
    forced = __reduce_add_sync(0xffffffffu, forced);
    if (lane == 0) {
      s_high[warp] = high;
      s_low[warp] = low;
      s_some[warp] = some;
      s_forced[warp] = forced;
    }
    if (threadIdx.x == 0) s_few = 0;
    __syncthreads();
    high = __reduce_max_sync(0xffffffffu, s_high[lane % kWarps]);
    low = __reduce_min_sync(0xffffffffu, s_low[lane % kWarps]) + 1u;
    some = __reduce_add_sync(0xffffffffu, lane < kWarps ? s_some[lane % kWarps] : 0);
    forced = __reduce_add_sync(0xffffffffu, lane < kWarps ? s_forced[lane % kWarps] : 0);
    left = p.count - forced;  // no more than the first and the recent ones: not negative
    if (some <= p.count) {
      left = 0;
    } else if (left == 0) {
      least = kQ8Forced - 1u;
    } else {
      // the score that is looked for is in low .. low + span, of those there the left-th largest; neither 0 nor kQ8Forced is
      uint32_t span = high - low;
      while (span > 0) {
        const int shift = max(24 - __clz(span), 0);
        for (int i = threadIdx.x; i < 256; i += THREADS) histogram[i] = 0;
        __syncthreads();
        each([&](int, uint32_t x) {
          if (x - low <= span) atomicAdd(&histogram[(x - low) >> shift], 1);
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
        low += (uint32_t)s_digit << shift;
        span = min(span - ((uint32_t)s_digit << shift), (1u << shift) - 1u);
        left = s_left;
        if (s_same == left) {  // all of them are taken
          low -= 1u;
          left = 0;
          break;
        }
        if (span > 0 && s_same <= 32) {  // the left-th largest of a warp's scores, without more counting
          each([&](int, uint32_t x) {
            if (x - low <= span) few[atomicAdd(&s_few, 1)] = x;
          });
          __syncthreads();
          const uint32_t mine = lane < s_few ? few[lane] : 0u;
          int larger = 0, same = 0;
#pragma unroll
          for (int v = 0; v < 32; ++v) {
            const uint32_t other = __shfl_sync(0xffffffffu, mine, v);
            larger += other > mine;
            same += other == mine;
          }
          const unsigned here = __ballot_sync(0xffffffffu, mine != 0 && larger < left && larger + same >= left);
          low = __shfl_sync(0xffffffffu, mine, __ffs(here) - 1);
          left -= __shfl_sync(0xffffffffu, larger, __ffs(here) - 1);
          break;
        }
      }
      least = low;
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
  ANNA_REQUIRE(streams < (1ll << 31), "%s: too many queries", what);
  Q8SelectParams p{};
  p.q = q; p.q_stride_b = batch > 1 ? q_stride_b : 0; p.q_stride_h = q_heads > 1 ? q_stride_h : 0; p.q_stride_t = tokens > 1 ? q_stride_t : 0;
  p.pages = pages; p.block_table = page_table; p.table_stride = table_stride; p.lengths = lengths; p.blocks = blocks; p.scores = scores;
  p.kv_heads = kv_heads; p.groups = q_heads / kv_heads; p.tokens = tokens; p.block_size = block_size; p.page_bytes = (int)bytes;
  p.count = count; p.first = first; p.recent = recent; p.num_pages = num_pages; p.max_blocks = max_blocks;
  p.row_group = p.groups <= 8 && 8 % p.groups == 0 ? p.groups : (p.groups + 7) / 8 * 8;
  p.group_shift = p.row_group == 1 ? 0 : p.row_group == 2 ? 1 : p.row_group == 4 ? 2 : 3;
  p.head_tiles = (p.row_group + 7) / 8;
  // As many KV heads as shared memory has room for with one token, then as many tokens.
  const int tile_bytes = 2 * (2 * head_dim / 64) * 512 + 32, room = 64 * 1024 / tile_bytes;
  // Where warps have few tiles each, one KV head: what counts is how soon a CTA's queries are ready (8 KV heads, one row of 8191 pages: all at once 17.4 us,
  // one 17.0; a row of 49160 tokens in pages of 16 12.7, 11.7).
  const int64_t page_tiles = (max_blocks + kQ8SelectTile - 1) / kQ8SelectTile, ctas = 148 * (head_dim == 256 ? kQ8SelectCtas<256> : kQ8SelectCtas<128>);
  const bool few = (int64_t)batch * kv_heads * page_tiles <= 2 * ctas * kQ8SelectWarps;
  p.heads_at_once = few || room / p.head_tiles < 1 ? 1 : room / p.head_tiles > kv_heads ? kv_heads : room / p.head_tiles;
  p.tokens_at_once = room / p.heads_at_once * 8 / p.row_group;
  if (p.tokens_at_once > kQ8SelectRows / p.row_group) p.tokens_at_once = kQ8SelectRows / p.row_group;
  if (p.tokens_at_once > tokens) p.tokens_at_once = tokens;
  if (p.tokens_at_once < 1) p.tokens_at_once = 1;
  const int smem = p.heads_at_once * ((p.tokens_at_once * p.row_group + 7) / 8) * tile_bytes;
  if (smem > 200 * 1024) return set_error(ANNA_ERR_UNSUPPORTED, "%s: too many query heads (%d) to a KV head", what, p.groups);
  p.chunks = (tokens + p.tokens_at_once - 1) / p.tokens_at_once;
  p.head_groups = (kv_heads + p.heads_at_once - 1) / p.heads_at_once;
  p.batch = batch;
  if (max_blocks > 0) {
    const int64_t tiles = page_tiles;
    const int64_t streams_of_all = (int64_t)batch * p.chunks * p.head_groups, line = streams_of_all * (tiles + kQ8SelectCost);
    // tiles of a CTA: at least one for every warp
    const int64_t least = (kQ8SelectWarps + p.heads_at_once - 1) / p.heads_at_once, even = (streams_of_all * tiles + ctas - 1) / ctas;
    p.part_tiles = (int)(even < least ? least : even > 64 ? 64 : even);
    const int64_t splits = (tiles + p.part_tiles - 1) / p.part_tiles;
    const bool shares = ((!few && batch > 1) || streams_of_all * splits > ctas) && batch <= kBalancedMaxRows && line < (1ll << 30);
    ANNA_REQUIRE(shares || (batch < 65536 && p.chunks * p.head_groups < 65536), "%s: too many queries", what);
    const dim3 grid = shares ? dim3((unsigned)ctas) : dim3((unsigned)splits, (unsigned)batch, (unsigned)(p.chunks * p.head_groups));
    const int rc = ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
      return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
        auto kernel = shares ? q8_score_kernel<T, D, true> : q8_score_kernel<T, D, false>;
        ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return q8_launch("q8_score_kernel", kernel, grid, kQ8SelectWarps * 32, smem, (cudaStream_t)stream, p);
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
