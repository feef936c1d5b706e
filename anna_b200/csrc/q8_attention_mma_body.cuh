// Attention over the 8-bit paged cache on tensor cores: pages of a multiple of 8 tokens.  Objects: q8_attention_mma.cu (bf16),
// q8_attention_mma_half.cu, q8_attention_mma_float.cu.
//
// Keys and values are the first operand of mma.sync (S^T = K Q^T with 16 tokens as rows, O^T = V^T P^T with 16 dims as rows), the queries that
// share a KV head its eight columns (NT times eight of a CTA).
//
// Scores: codes go into the integer product as they are.  A query is a whole number of 24 bits, -2^23 to 2^23 - 1, with 2^22 and more for its head's
// largest magnitude: three bytes, the first signed, three products, whose sums are exact.  What is not is a query: its entries are off by half a unit,
// 2^-23 of the head's largest magnitude at most.
// Sums: a code with its top bit flipped, as the low byte of an fp16 of exponent 1024, reads as 1152 + code, and taking 1152 off is exact.  Weights
// are 2^14 times exp2 of the score below the running maximum, as sums of two fp16.  The scale of a page's values goes into its weights where it is within
// 2^6 of the power of two above the largest so far, as a share of that power; where it is smaller, the tile's product is added to the sums in 32 bits,
// times the scale, so pages of any scales may meet.  A weight, times its share where it has one, is off by 2^-23 of itself (half a step of the second fp16),
// but where the largest weight is 2^14 by no less than half a step of subnormals, 2^-25: a weight whose share is 1 keeps 2^-23 down to 2^-16 of the
// largest and 2^-11 down to 2^-28, one whose share is 1/64 down to 2^-10 and 2^-22.
//
// The order of dims and tokens inside a product is free, so a lane's share of a tile is 16-byte pieces of rows.  A warp copies its own tiles,
// 16 bytes a lane and instruction, into a ring of its own; pieces are swizzled so that the reads of a tile are free of bank conflicts.
//
// A tile of 16 tokens lies in one page, or (kHalves: pages of an odd number of eights) its halves lie in two, with scales of their own.
//
// Tokens of the unfinished page take the same way as 16-token tiles of the ring: keys times queries in the cache's type, scaled by a power
// of two, and weights as a sum of two numbers of it.
//
// fp32 caches: all products are added in 32 bits, and tokens of the ring are scored and summed on CUDA cores.
#pragma once
#include "mma_utils.cuh"
#include "q8_common.cuh"

namespace anna {

// W warps: four, with several CTAs to an SM; eight, with one, where the tiles of a call are few (one row of 4000 tokens: 11.0 us with four, 9.9 with eight).
template <typename T, int D, int NT, int W>
struct Q8Cfg {
  static constexpr int kWarps = W;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtas = W == 8 ? 1 : D == 256 ? 2 : NT <= 2 ? 3 : 2;  // per SM
  static constexpr int kStages = D == 64 ? 4 : D == 256 && (NT == 2 || sizeof(T) == 4) ? 2 : 3;
  static constexpr int kRows = 8 * NT;
  static constexpr int kChunks = D / 64;         // 16-byte pieces of a lane's key
  static constexpr int kVWords = D / 32;         // 4-byte words of a lane's value
  static constexpr int kTileBytes = 32 * D;      // keys and values of 16 tokens
  static constexpr int kMergeStride = D + 4;     // floats
  static constexpr int kOffParts = 0;                                   // [NT][chunks][3][32 lanes] uint4: bytes of queries as second operands
  static constexpr int kOffRing = kOffParts + NT * kChunks * 3 * 512;   // [rows][D] queries in the cache's type
  static constexpr int kOffStats = kOffRing + kRows * D * (int)sizeof(T);  // [warps][rows] float2
  static constexpr int kOffRate = kOffStats + kWarps * kRows * 8;       // [rows] to units of log2 of a weight; in the end 1 / denominator
  static constexpr int kOffRingRate = kOffRate + kRows * 4;             // [rows] the same for keys of the ring
  static constexpr int kOffTiles = (kOffRingRate + kRows * 4 + 127) / 128 * 128;  // [warps][stages] tiles; in the end sums of the warps, weights of a merge
  static constexpr int kMergeBytes = kWarps * 8 * kMergeStride * 4;
  static constexpr int kWeightBytes = kRows * kMultiMaxPartials * 4;
  static constexpr int kRingBytes = kWarps * kStages * kTileBytes;
  static constexpr int kSmem = kOffTiles + (kRingBytes > kWeightBytes ? kRingBytes : kWeightBytes);
  static_assert(kMergeBytes <= kRingBytes && kCtas * (kSmem + 1024 + 5120) <= 228 * 1024, "shared memory");
};

// Place of the 16-byte piece `piece` of token `token` in a tile.  Reads of keys take pieces D / 64 t .. of tokens g and g + 8 (t = lane % 4, g = lane / 4),
// reads of values those of dims D / 8 g .. of tokens 2 t + const: eight lanes of either always in different banks.
template <int D>
__device__ __forceinline__ uint32_t q8_place(int token, int piece) {
  if constexpr (D == 64) {  // two tokens to a line of 128 bytes
    return token / 2 * 128 + ((((token & 1) << 2 | piece) ^ (token & 6)) << 4);
  } else if constexpr (D == 128) {
    return token * 128 + ((piece ^ (token & 7)) << 4);
  } else {  // a token has two lines
    const int turn = (token & 4) | (token & 1) << 1 | ((token >> 1 & 1) ^ piece >> 3);
    return token * 256 + (piece & 8) * 16 + (((piece & 7) ^ turn) << 4);
  }
}
// What one lane's places differ by, so that few of them have to be worked out: the copy of pieces 32 i + lane, value tokens 2 t and 2 t + 1.
// (All of them from q8_place in the loop: 39 instructions a tile more, 3 % of the time of 16 rows of 32768 tokens.)
template <int D>
__host__ __device__ constexpr uint32_t kQ8CopyTurn(int i) {
  return D == 64 ? 0u : D == 128 ? (uint32_t)(i & 1) << 6 : (uint32_t)((i >> 1 & 1) << 2 | (i & 1)) << 4;
}
template <int D>
constexpr uint32_t kQ8OddTurn = D == 64 ? 64u : D == 128 ? 16u : 32u;
template <int D>
constexpr uint32_t kQ8OddStep = D == 64 ? 0u : D;  // bytes from a token's line to the next one's

__device__ __forceinline__ uint4 q8_shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 q8_shared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}

// d += a . b of signed bytes with signed or unsigned ones; kFirst: d = a . b.
template <bool kSigned, bool kFirst>
__device__ __forceinline__ void q8_mma_bytes(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
#define ANNA_Q8_MMA(TYPE, C0, C1, C2, C3)                                                                                              \
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8." TYPE ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"      \
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                                        \
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(C0), "r"(C1), "r"(C2), "r"(C3))
  if constexpr (kSigned && kFirst) ANNA_Q8_MMA("s8", 0, 0, 0, 0);
  else if constexpr (kSigned) ANNA_Q8_MMA("s8", d[0], d[1], d[2], d[3]);
  else if constexpr (kFirst) ANNA_Q8_MMA("u8", 0, 0, 0, 0);
  else ANNA_Q8_MMA("u8", d[0], d[1], d[2], d[3]);
#undef ANNA_Q8_MMA
}
// d = a . b
__device__ __forceinline__ void q8_mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// The codes in bytes 0 and 2 of x as two fp16.
__device__ __forceinline__ uint32_t q8_halves(uint32_t x) {
  uint32_t r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"((x & 0x00ff00ffu) ^ 0x64806480u), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ float q8_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// All ones where the halves are finite.
template <typename T>
__device__ __forceinline__ uint32_t q8_finite_halves(uint32_t x) {
  constexpr uint32_t kExp = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
  return ((x & kExp) != kExp ? 0x0000ffffu : 0u) | ((x >> 16 & kExp) != kExp ? 0xffff0000u : 0u);
}

template <typename T, int D, int NT, int W, bool kBlocks, bool kHalves>
__global__ void __launch_bounds__(Q8Cfg<T, D, NT, W>::kThreads, Q8Cfg<T, D, NT, W>::kCtas) q8_mma_kernel(const Q8Params p, int row_tiles) {
  using Cfg = Q8Cfg<T, D, NT, W>;
  constexpr bool kFloat = std::is_same_v<T, float>;
  constexpr int kPages = kHalves ? 2 : 1, kPageTokens = 16 / kPages;  // of a tile
  constexpr int kTile = kBalancedTileTokens;
  constexpr int kFar = 0x7fff0000;  // position of a token that nobody sees
  // Queries of the ring are under 2^15 in fp16 and under 2 in bf16, whose keys may be as large as a product; for the same reason sums are 2^14
  // times what they stand for in fp16 alone.
  constexpr bool kHalf = std::is_same_v<T, __half>;
  constexpr float kWeight = 16384.0f;                        // of the largest
  constexpr float kRingWeight = kHalf ? kWeight : 1.0f;
  // One fp16 of 11 bits would show in an output, of fp16 (an error of 0.00029 of the whole instead of 0.00021) and of bf16 (0.00168 instead of 0.00166), so
  // weights are sums of two, the second kRest times what the first leaves (16 rows of 32768 tokens, 4 queries a KV head: 174 us with one, 186 so; of four tokens
  // 260 and 292).
  constexpr float kRest = kFloat ? 4096.0f : 1.0f;
  constexpr float kUnit = 1.0f / 4194304.0f;                 // of a query entry, its head's largest magnitude in [1, 2)
  extern __shared__ __align__(128) uint8_t smem[];
  float* rate = reinterpret_cast<float*>(smem + Cfg::kOffRate);
  float* ring_rate = reinterpret_cast<float*>(smem + Cfg::kOffRingRate);
  float2* stats = reinterpret_cast<float2*>(smem + Cfg::kOffStats);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const uint32_t tiles = smem_u32(smem + Cfg::kOffTiles) + warp * Cfg::kStages * Cfg::kTileBytes, tiles_end = tiles + Cfg::kStages * Cfg::kTileBytes;
  // this lane's places in a tile: what it copies, keys, values of tokens 2 t; see kQ8CopyTurn
  const uint32_t copy_place = q8_place<D>(lane / (D / 16), lane % (D / 16)), key_place = q8_place<D>(gid, Cfg::kChunks * tig);
  const uint32_t value_place = 16 * D + (D == 64 ? q8_place<D>(2 * tig, gid / 2) + gid % 2 * 8 : q8_place<D>(2 * tig, D / 128 * gid));
  const uint32_t parts = smem_u32(smem + Cfg::kOffParts) + lane * 16;
  q8_wait_for_previous();

  q8_for_each_segment<T, D, Cfg::kThreads, kBlocks>(p, row_tiles, [&](int64_t b, int kvh, int tile, int t0, int t1, int len, const MultiPartial& part) {
  const Q8Stream st = q8_stream<Cfg::kRows>(p, b, kvh, tile, len);
  const int first_seen = st.len - p.tokens;  // newest key that query 0 sees
  const int packed_tiles = max(0, min(t1, st.packed) - t0 + kTile - 1) / kTile;
  const int mine = packed_tiles > warp ? (packed_tiles - warp + Cfg::kWarps - 1) / Cfg::kWarps : 0;  // tiles of this warp: every kWarps-th

  // queries, on their way while the pages are found
  constexpr int E = D / 32, kMyRows = Cfg::kRows / Cfg::kWarps;
  T query[kMyRows][E];
#pragma unroll
  for (int k = 0; k < kMyRows; ++k) {
    const int row = st.row0 + min(warp + k * Cfg::kWarps, st.count - 1), t = multi_token_of(p, row), h = kvh * p.groups + row - t * p.groups;
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_stride_b + h * p.q_stride_h + t * p.q_stride_t + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) query[k][j] = q[j];
  }

  // ---- pages of 32 of the warp's tiles, one tile a lane -------------------------------------------------------------------------------
  struct Pages {
    const uint8_t* keys[kPages];
    int position[kPages];  // of the first token there in the sequence
    float2 scale[kPages];
  };
  auto find = [&](int from) {  // pages and positions; the scales are read by `scales`
    Pages x;
    const int i = from + lane;
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      x.keys[h] = p.pages;
      x.position[h] = kFar;
      x.scale[h] = make_float2(0.0f, 0.0f);
      const int at = t0 + (warp + i * Cfg::kWarps) * kTile + kPageTokens * h;
      if (i < mine && (!kHalves || at < st.packed)) {
        const int entry = p.block_shift >= 0 ? at >> p.block_shift : at / p.block_size, slot = at - entry * p.block_size;
        int block;
        const int64_t page = q8_page_at(p, st, b, kvh, entry, &block);
        if (page >= 0) {
          x.keys[h] = p.pages + page + slot * D;
          x.position[h] = block * p.block_size + slot;
        }
      }
    }
    return x;
  };
  auto scales = [&](Pages& x) {  // a tile's keys begin `slot` rows behind its page
#pragma unroll
    for (int h = 0; h < kPages; ++h)
      if (x.position[h] != kFar) {
        const int slot = p.block_shift >= 0 ? x.position[h] & (p.block_size - 1) : x.position[h] % p.block_size;
        x.scale[h] = *reinterpret_cast<const float2*>(x.keys[h] + (int64_t)(2 * p.block_size - slot) * D);
      }
  };
  const int values_at = p.block_size * D;
  auto copy_tile = [&](const uint8_t* const (&keys)[kPages], uint32_t to) {
#pragma unroll
    for (int value = 0; value < 2; ++value)
#pragma unroll
      for (int h = 0; h < kPages; ++h) {
        constexpr int kEach = D / 32 / kPages;
        const uint8_t* from = keys[h] + lane * 16 + value * values_at;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          cp_async16(to + (copy_place ^ kQ8CopyTurn<D>(h * kEach + i)) + 16 * D * value + (h * kEach + i) * 512, from + i * 512, 16);
      }
  };
  Pages now = find(0), next = now;
  uint32_t to = tiles;  // where the next copy goes
  auto start = [&](int i, int done) {  // copies of tile i, while `now` is of the 32 tiles that `done` is of
    if (i < mine) {
      const uint8_t* keys[kPages];
#pragma unroll
      for (int h = 0; h < kPages; ++h) {
        const unsigned long long x = (i >> 5) == (done >> 5) ? (unsigned long long)now.keys[h] : (unsigned long long)next.keys[h];
        keys[h] = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, x, i & 31));
      }
      copy_tile(keys, to);
    }
    to = to + Cfg::kTileBytes == tiles_end ? tiles : to + Cfg::kTileBytes;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < Cfg::kStages - 1; ++i) start(i, 0);
  scales(now);
  if (mine > 32) next = find(32);

  // ---- queries -----------------------------------------------------------------------------------------------------------------------
#pragma unroll
  for (int k = 0; k < kMyRows; ++k) {
    const int i = warp + k * Cfg::kWarps;
    // A row that is not there: its columns are not stored, but its scores count where the softmax asks whether any is above its maximum, so they must not
    // follow from what lies in shared memory.  Those of packed tiles are whole numbers times 0.
    if (i >= st.count) {
      if (lane == 0) rate[i] = ring_rate[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < E; ++j) reinterpret_cast<T*>(smem + Cfg::kOffRing)[i * D + lane * E + j] = ElemTraits<T>::from_float(0.0f);
      continue;
    }
    float x[E], top = 0.0f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      x[j] = ElemTraits<T>::to_float(query[k][j]);
      fine = fine && fabsf(x[j]) < INFINITY;
      top = fmaxf(top, fabsf(x[j]));
    }
    fine = __all_sync(0xffffffffu, fine);
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    // top * 2^up is in [1, 2)
    const int up = fine && top > 0.0f ? min(127 - (int)(__float_as_uint(top) >> 23), 126) : 0;
    const float factor = __uint_as_float((uint32_t)(max(up, -126) + 127) << 23) * (up < -126 ? 0.5f : 1.0f);
    const float back = p.scaling * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - up) << 23);
    constexpr float kRingFactor = kHalf ? 16384.0f : 1.0f;
    if (lane == 0) {
      rate[i] = fine ? back : __int_as_float(0x7fc00000);
      ring_rate[i] = back / kRingFactor;
    }
    // dims D / 4 t + 16 c .. are lane t's piece c; this lane's E dims lie in one piece, next to one another
    const int d0 = lane * E, place = (((i / 8 * Cfg::kChunks + d0 % (D / 4) / 16) * 3) * 32 + i % 8 * 4 + d0 / (D / 4)) * 16 + d0 % 16;
    uint32_t bytes[3][E >= 4 ? E / 4 : 1] = {};
    T scaled[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      // the top byte is signed, so what rounds up to 2^23 (fp32: 2^k less its last bit) stays half a unit below, as far off as any tie
      const int whole = fine ? min(__float2int_rn(x[j] * factor / kUnit), 8388607) : 0;
#pragma unroll
      for (int n = 0; n < 3; ++n) bytes[n][j / 4] |= ((uint32_t)whole >> (16 - 8 * n) & 255u) << (8 * (j % 4));
      scaled[j] = ElemTraits<T>::from_float(x[j] * factor * kRingFactor);
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      uint8_t* to = smem + Cfg::kOffParts + place + 512 * n;
      if constexpr (E == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)bytes[n][0];
      else if constexpr (E == 4) *reinterpret_cast<uint32_t*>(to) = bytes[n][0];
      else *reinterpret_cast<uint2*>(to) = make_uint2(bytes[n][0], bytes[n][E / 4 - 1]);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) reinterpret_cast<T*>(smem + Cfg::kOffRing)[i * D + d0 + j] = scaled[j];
  }
  __syncthreads();
  float to_log2[NT][2], m_run[NT][2], l_run[NT][2], o[NT][D / 16][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      to_log2[j][k] = rate[8 * j + 2 * tig + k];
      m_run[j][k] = -INFINITY;
      l_run[j][k] = 0.0f;
    }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[j][d][r] = 0.0f;
  auto limit = [&](int j, int k) { return first_seen + multi_token_of(p, st.row0 + 8 * j + 2 * tig + k); };  // newest key that a row sees

  // Scores of 16 tokens (rows gid and gid + 8 of every column pair) become weights, at 2^14 times their size.  A score may be up to 1 above the
  // running maximum (a weight of 2^15) before that is raised: the sums are scaled anew less often.
  auto softmax = [&](float (&s)[NT][4]) {
    bool more = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) more = more || fmaxf(s[j][k], s[j][k + 2]) > m_run[j][k] + 1.0f;
    if (__any_sync(0xffffffffu, more)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float top = fmaxf(s[j][k], s[j][k + 2]);
#pragma unroll
          for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(top, m_run[j][k]);
          const float by = top == -INFINITY ? 1.0f : q8_exp2(m_run[j][k] - top);
          m_run[j][k] = top;
          l_run[j][k] *= by;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[j][d][k] *= by;
            o[j][d][k + 2] *= by;
          }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // log2 of kWeight; a difference near 14 is off by 2^-21, so fp32 caches multiply
        const float base = m_run[j][k] == -INFINITY ? 0.0f : m_run[j][k] - (kFloat ? 0.0f : 14.0f);
        s[j][k] = q8_exp2(s[j][k] - base) * (kFloat ? kWeight : 1.0f);
        s[j][k + 2] = q8_exp2(s[j][k + 2] - base) * (kFloat ? kWeight : 1.0f);
        l_run[j][k] += s[j][k] + s[j][k + 2];
      }
  };

  // ---- packed tiles -------------------------------------------------------------------------------------------------------------------
  uint32_t at = tiles;  // of the tile that is read
  int unit = -120;         // of the sums, as a power of two
  for (int i = 0; i < mine; ++i) {
    int position[kPages];
    float2 scale[kPages];
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      position[h] = __shfl_sync(0xffffffffu, now.position[h], i & 31);
      scale[h] = make_float2(__shfl_sync(0xffffffffu, now.scale[h].x, i & 31), __shfl_sync(0xffffffffu, now.scale[h].y, i & 31));
    }
    cp_async_wait<Cfg::kStages - 2>();
    __syncwarp();  // the tile is there, and the one in front of it has been read
    start(i + Cfg::kStages - 1, i);
    int whole[NT][3][4];
#pragma unroll
    for (int c = 0; c < Cfg::kChunks; ++c) {
      const uint4 u = q8_shared16(at + (key_place ^ c << 4)), v = q8_shared16(at + (key_place ^ c << 4) + 8 * D);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t q = parts + (j * Cfg::kChunks + c) * 1536;
        const uint4 q0 = q8_shared16(q), q1 = q8_shared16(q + 512), q2 = q8_shared16(q + 1024);
        auto both = [&](auto first) {
          constexpr bool kFirst = decltype(first)::value;
          q8_mma_bytes<true, kFirst>(whole[j][0], u.x, v.x, u.y, v.y, q0.x, q0.y);
          q8_mma_bytes<false, kFirst>(whole[j][1], u.x, v.x, u.y, v.y, q1.x, q1.y);
          q8_mma_bytes<false, kFirst>(whole[j][2], u.x, v.x, u.y, v.y, q2.x, q2.y);
        };
        if (c == 0) both(std::true_type{});
        else both(std::false_type{});
        q8_mma_bytes<true, false>(whole[j][0], u.z, v.z, u.w, v.w, q0.z, q0.w);
        q8_mma_bytes<false, false>(whole[j][1], u.z, v.z, u.w, v.w, q1.z, q1.w);
        q8_mma_bytes<false, false>(whole[j][2], u.z, v.z, u.w, v.w, q2.z, q2.w);
      }
    }
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      // The lower two bytes' sums are below 2^23 each: together below 2^31.  The unit goes into the numbers and not into the rates, which for tiny queries
      // (of huge keys) are small as it is.
      for (int r = 0; r < 4; ++r)
        s[j][r] = fmaf(__int2float_rn(whole[j][0][r]), 65536.0f * kUnit, __int2float_rn(whole[j][1][r] * 256 + whole[j][2][r]) * kUnit) *
                  (scale[r / 2 * (kPages - 1)].x * to_log2[j][r & 1]);
    bool cut = false;  // tokens that some rows do not see, or a page that is none
#pragma unroll
    for (int h = 0; h < kPages; ++h) cut = cut || position[h] + kPageTokens - 1 > first_seen;
    if (cut) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int last = limit(j, k);
          if (position[0] + gid > last) s[j][k] = -INFINITY;
          if (position[kPages - 1] + gid + (kHalves ? 0 : 8) > last) s[j][k + 2] = -INFINITY;
        }
    }
    softmax(s);
    // The sums count in units of a power of two above the largest scale so far.
    float share[kPages];
    bool near = !kFloat;  // the weights may take the scales
    int exponent = -126;
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      const int e = (int)(__float_as_uint(scale[h].y) >> 23) - 126;
      exponent = e < 129 ? max(exponent, e) : exponent;  // else NaN
    }
    if (exponent > unit) {
      const float by = unit + 126 < exponent ? 0.0f : __uint_as_float((uint32_t)(127 + unit - exponent) << 23);
      unit = exponent;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[j][d][r] *= by;
    }
#pragma unroll
    for (int h = 0; h < kPages; ++h) {
      share[h] = scale[h].y * __uint_as_float((uint32_t)(127 - unit) << 23);
      near = near && share[h] <= 1.0f && (share[h] >= 1.0f / 64.0f || share[h] == 0.0f);
    }
    uint32_t w[NT][2], rest[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float f = near ? share[k * (kPages - 1)] : 1.0f;
        const uint32_t most = pack2<__half>(s[j][2 * k] * f, s[j][2 * k + 1] * f);
        w[j][k] = movmatrix_trans(most);
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&most));
        rest[j][k] = movmatrix_trans(pack2<__half>(fmaf(s[j][2 * k], f, -x.x) * kRest, fmaf(s[j][2 * k + 1], f, -x.y) * kRest));
      }
    uint32_t val[4][Cfg::kVWords];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t from = (value_place ^ ((k & 1) ? kQ8OddTurn<D> : 0u)) + (k & 1) * kQ8OddStep<D> + k / 2 * 8 * D;
      if constexpr (D == 64) {
        const uint2 v = q8_shared8(at + from);
        val[k][0] = v.x; val[k][1] = v.y;
      } else {
#pragma unroll
        for (int c = 0; c < D / 128; ++c) {
          const uint4 v = q8_shared16(at + (from ^ c << 4));
          val[k][4 * c] = v.x; val[k][4 * c + 1] = v.y; val[k][4 * c + 2] = v.z; val[k][4 * c + 3] = v.w;
        }
      }
    }
    auto sums = [&](auto&& add) {
#pragma unroll
      for (int v = 0; v < Cfg::kVWords; ++v) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x = __byte_perm(val[0][v], val[1][v], half == 0 ? 0x5410 : 0x7632), z = __byte_perm(val[2][v], val[3][v], half == 0 ? 0x5410 : 0x7632);
          const uint32_t a[4] = {q8_halves(x), q8_halves(x >> 8), q8_halves(z), q8_halves(z >> 8)};
#pragma unroll
          for (int j = 0; j < NT; ++j) add(j, o[j][2 * v + half], a);
        }
      }
    };
    if (near) {
      sums([&](int j, float (&sum)[4], const uint32_t (&a)[4]) {
        mma_m16n8k16<__half>(sum, a, w[j][0], w[j][1]);
        mma_m16n8k16<__half>(sum, a, rest[j][0], rest[j][1]);
      });
    } else {  // a scale far below the largest, or NaN, or an fp32 cache
      float by[kPages][NT][2];
#pragma unroll
      for (int h = 0; h < kPages; ++h)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) by[h][j][k] = cut && position[h] > limit(j, k) ? 0.0f : share[h];  // rows that see nothing there
      sums([&](int j, float (&sum)[4], const uint32_t (&a)[4]) {
#pragma unroll
        for (int h = 0; h < kPages; ++h) {
          float part[4];
          q8_mma_first(part, a, kHalves && h == 1 ? 0u : w[j][0], kHalves && h == 0 ? 0u : w[j][1]);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[r] = fmaf(part[r], by[h][j][r & 1], sum[r]);
          q8_mma_first(part, a, kHalves && h == 1 ? 0u : rest[j][0], kHalves && h == 0 ? 0u : rest[j][1]);
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[r] = fmaf(part[r], by[h][j][r & 1] * (1.0f / kRest), sum[r]);
        }
      });
    }
    if ((i & 31) == 16 && i + 16 < mine) scales(next);
    at = at + Cfg::kTileBytes == tiles_end ? tiles : at + Cfg::kTileBytes;
    if ((i & 31) == 31 && i + 1 < mine) {
      now = next;
      if (i + 33 < mine) next = find(i + 33);
    }
  }
  // to the units of the ring
  const float units = __uint_as_float((uint32_t)(127 + unit) << 23);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[j][d][r] = o[j][d][r] * (kRingWeight / kWeight) * units;

  // ---- tiles of the ring ----------------------------------------------------------------------------------------------------------------
  const int ring_from = max(t0, st.packed);
  const int64_t slot = ring_from < t1 ? p.window_slots[b] : -1;
  if (slot >= 0 && slot < p.num_slots) {
    const T* keys = reinterpret_cast<const T*>(p.window) + (slot * 2 * p.kv_heads + kvh) * p.block_size * D;
    const T* values = keys + (int64_t)p.kv_heads * p.block_size * D;
    const int begin = ring_from - st.packed, end = t1 - st.packed, full = st.full;  // ring slots; position of slot 0
    for (int from = begin + (warp + Cfg::kWarps - packed_tiles % Cfg::kWarps) % Cfg::kWarps * kTile; from < end; from += Cfg::kWarps * kTile) {
      const int valid = min(kTile, end - from), position = full + from;
      auto row_of = [&](int token) { return (int64_t)(from + min(token, valid - 1)) * D; };
      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[j][r] = 0.0f;
      if constexpr (kFloat) {
        const float4* k0 = reinterpret_cast<const float4*>(keys + row_of(gid));
        const float4* k1 = reinterpret_cast<const float4*>(keys + row_of(gid + 8));
        const float4* raw = reinterpret_cast<const float4*>(smem + Cfg::kOffRing) + 2 * tig * (D / 4);
#pragma unroll 4
        for (int d = 0; d < D / 4; ++d) {
          const float4 k[2] = {k0[d], k1[d]};
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float4 q = raw[(8 * j + (r & 1)) * (D / 4) + d];
              s[j][r] += fmaf(k[r / 2].w, q.w, fmaf(k[r / 2].z, q.z, fmaf(k[r / 2].y, q.y, k[r / 2].x * q.x)));  // a quarter of the roundings of one chain
            }
        }
      } else {
        const T* k0 = keys + row_of(gid) + 8 * tig;
        const T* k1 = keys + row_of(gid + 8) + 8 * tig;
        const uint8_t* raw = smem + Cfg::kOffRing + (gid * D + 8 * tig) * 2;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {  // 32 dims, 8 of them a lane's, are two products
          const uint4 ka = *reinterpret_cast<const uint4*>(k0 + 32 * c), kb = *reinterpret_cast<const uint4*>(k1 + 32 * c);
          const uint32_t lo[4] = {ka.x, kb.x, ka.y, kb.y}, hi[4] = {ka.z, kb.z, ka.w, kb.w};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 q = *reinterpret_cast<const uint4*>(raw + (8 * j * D + 32 * c) * 2);
            mma_m16n8k16<T>(s[j], lo, q.x, q.y);
            mma_m16n8k16<T>(s[j], hi, q.z, q.w);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = gid + 8 * (r / 2);
          s[j][r] = token >= valid || position + token > limit(j, r & 1) ? -INFINITY : s[j][r] * ring_rate[8 * j + 2 * tig + (r & 1)];
        }
      softmax(s);
      // Infinite and NaN values are left out of the sums, as they must not meet a weight of 0: of a row that does not see them, of a rest.
      bool strange = false;
      if constexpr (kFloat) {
        for (int token = 0; token < valid; ++token) {
          float weight[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              weight[j][k] = __shfl_sync(0xffffffffu, token < 8 ? s[j][k] : s[j][k + 2], (token & 7) * 4 + tig) * (kRingWeight / kWeight);
          const float4* value = reinterpret_cast<const float4*>(values + row_of(token) + gid * (D / 8));
#pragma unroll
          for (int d = 0; d < D / 32; ++d) {
            const float4 got = value[d];
            float v[4] = {got.x, got.y, got.z, got.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool fine = fabsf(v[i]) < INFINITY;
              strange = strange || !fine;
              v[i] = fine ? v[i] : 0.0f;
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k) o[j][2 * d + i / 2][2 * (i & 1) + k] = fmaf(weight[j][k], v[i], o[j][2 * d + i / 2][2 * (i & 1) + k]);
            }
          }
        }
      } else {
      // weights as a sum of two of the type, so that they keep 16 bits and more
      uint32_t w[NT][2], rest[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float x = s[j][2 * k] * (kRingWeight / kWeight), y = s[j][2 * k + 1] * (kRingWeight / kWeight);
          const uint32_t most = pack2<T>(x, y);
          const T* parts = reinterpret_cast<const T*>(&most);
          w[j][k] = movmatrix_trans(most);
          rest[j][k] = movmatrix_trans(pack2<T>(x - ElemTraits<T>::to_float(parts[0]), y - ElemTraits<T>::to_float(parts[1])));
        }
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {  // 8 of a lane's dims
        uint32_t x[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int token = 2 * tig + (k & 1) + 8 * (k / 2);
          const uint4 got = token < valid ? *reinterpret_cast<const uint4*>(values + row_of(token) + gid * (D / 8) + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
          x[k][0] = got.x; x[k][1] = got.y; x[k][2] = got.z; x[k][3] = got.w;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const uint32_t fine = q8_finite_halves<T>(x[k][v]);
            strange = strange || fine != 0xffffffffu;
            x[k][v] &= fine;
          }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const uint32_t a[4] = {__byte_perm(x[0][v], x[1][v], 0x5410), __byte_perm(x[0][v], x[1][v], 0x7632),
                                 __byte_perm(x[2][v], x[3][v], 0x5410), __byte_perm(x[2][v], x[3][v], 0x7632)};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma_m16n8k16<T>(o[j][4 * c + v], a, w[j][0], w[j][1]);
            mma_m16n8k16<T>(o[j][4 * c + v], a, rest[j][0], rest[j][1]);
          }
        }
      }
      }
      if (__any_sync(0xffffffffu, strange)) {  // what was left out, for the rows that see it, however small its weight
        for (int token = 0; token < valid; ++token) {
          const T* value = values + row_of(token) + gid * (D / 8);
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            const float x = ElemTraits<T>::to_float(value[d]);
            if (fabsf(x) < INFINITY) continue;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int k = 0; k < 2; ++k)
                if (position + token <= limit(j, k)) o[j][d / 2][2 * (d & 1) + k] += x;
          }
        }
      }
    }
  }

  // ---- the warps' rows together ----------------------------------------------------------------------------------------------------------
  cp_async_wait<0>();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int d = 4; d <= 16; d <<= 1) l_run[j][k] += __shfl_xor_sync(0xffffffffu, l_run[j][k], d);
      if (gid == 0) stats[warp * Cfg::kRows + 8 * j + 2 * tig + k] = make_float2(m_run[j][k], l_run[j][k]);
    }
  __syncthreads();
  // a thread per row: what each warp's sums count, in place of its maximum; and 1 / denominator, or 1 where partials are merged
  if (threadIdx.x < Cfg::kRows) {
    const int i = threadIdx.x;
    float top = -INFINITY, den = 0.0f;
#pragma unroll
    for (int v = 0; v < Cfg::kWarps; ++v) top = fmaxf(top, stats[v * Cfg::kRows + i].x);
#pragma unroll
    for (int v = 0; v < Cfg::kWarps; ++v) {
      const float2 x = stats[v * Cfg::kRows + i];
      // a warp without a key for the row has no sums; where none has, a NaN may be in them
      const float by = top == -INFINITY ? 1.0f : x.x == -INFINITY && x.y == 0.0f ? 0.0f : q8_exp2(x.x - top);
      stats[v * Cfg::kRows + i].x = by;
      den = fmaf(x.y, by, den);
    }
    den *= kRingWeight / kWeight;  // in the sums' units
    // a NaN among the scores has to stay one, so only a row without a key is zero
    rate[i] = part.count > 1 ? 1.0f : den == 0.0f ? 0.0f : 1.0f / den;
    if (part.count > 1 && i < st.count)
      reinterpret_cast<float2*>(p.stats)[multi_partial_row(part, part.mine, Cfg::kRows) + i] = make_float2(top * 0.6931471805599453f, den);
  }
  __syncthreads();
  float* merged = reinterpret_cast<float*>(smem + Cfg::kOffTiles);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float by = stats[warp * Cfg::kRows + 8 * j + 2 * tig + k].x;
      float* to = merged + (warp * 8 + 2 * tig + k) * Cfg::kMergeStride + gid * (D / 8);
#pragma unroll
      for (int d = 0; d < D / 16; d += 2)
        *reinterpret_cast<float4*>(to + 2 * d) = make_float4(o[j][d][k] * by, o[j][d][k + 2] * by, o[j][d + 1][k] * by, o[j][d + 1][k + 2] * by);
    }
    __syncthreads();
    const int rows = min(8, st.count - 8 * j);
    for (int item = threadIdx.x; item < rows * (D / 4); item += Cfg::kThreads) {
      const int i = item / (D / 4), d = 4 * (item % (D / 4));
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int v = 0; v < Cfg::kWarps; ++v) {
        const float4 x = *reinterpret_cast<const float4*>(merged + (v * 8 + i) * Cfg::kMergeStride + d);
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
      if (part.count == 1) {
        const float inv = rate[8 * j + i];
        const float out[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
        multi_store<T, 4>(p, b, kvh, st.row0 + 8 * j + i, d, out);
      } else {
        *reinterpret_cast<float4*>(p.values + (multi_partial_row(part, part.mine, Cfg::kRows) + 8 * j + i) * D + d) = sum;
      }
    }
    __syncthreads();
  }
  if (part.count > 1) {
    multi_merge_rows<T, D, Cfg::kWarps, Cfg::kRows>(p, b, kvh, tile, row_tiles, st.row0, st.count, part, merged);
    __syncthreads();
  }
  });
}

template <typename T, int D, int NT, int W = 4>
static int launch(const Q8Params& p, int row_tiles, int ctas, cudaStream_t stream) {
  using Cfg = Q8Cfg<T, D, NT, W>;
  const bool halves = p.block_size % kBalancedTileTokens != 0;
  auto kernel = p.blocks != nullptr ? (halves ? q8_mma_kernel<T, D, NT, W, true, true> : q8_mma_kernel<T, D, NT, W, true, false>)
                                    : (halves ? q8_mma_kernel<T, D, NT, W, false, true> : q8_mma_kernel<T, D, NT, W, false, false>);
  ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
  return q8_launch("q8_mma_kernel", kernel, dim3((unsigned)ctas), Cfg::kThreads, Cfg::kSmem, stream, p, row_tiles);
}

template <typename T>
int launch_q8_mma_of(const Q8Params& p, const Q8Plan& plan, int head_dim, int ctas, cudaStream_t stream) {
  return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
    if (plan.rows == 8) return plan.warps == 8 ? launch<T, D, 1, 8>(p, plan.row_tiles, ctas, stream) : launch<T, D, 1>(p, plan.row_tiles, ctas, stream);
    if (D == 256 || plan.rows == 16) return launch<T, D, 2>(p, plan.row_tiles, ctas, stream);
    if constexpr (D != 256) return launch<T, D, 4>(p, plan.row_tiles, ctas, stream);
    return ANNA_OK;
  });
}

}  // namespace anna
