// Attention over the 8-bit paged cache on tensor cores: 16-bit caches, pages of a multiple of 16 tokens.
//
// Keys and values are the first operand of mma.sync m16n8k16 (S^T = K Q^T with tokens as rows, O^T = V^T P^T with dims as rows), the
// queries that share a KV head its eight columns (NT times eight of a CTA).  Codes are whole numbers up to 127, which fp16 holds exactly:
// a byte with its top bit flipped under the exponent of 1024 reads as 1152 + code, and taking 1152 off is exact, too; a permute and half a
// subtraction per code.  The order of dims and tokens inside a product is free, so a lane's share of a tile is whole 16-byte pieces of
// rows, and tiles go from global memory to registers without a stop in shared memory.
//
// Queries are scaled by a power of two that brings their largest magnitude under 2^15, so bf16 ones fit into fp16 and lose no bit that is
// worth 2^-29 of the largest.  Scores take the keys' scale of the page in 32 bits.  Weights are 2^14 times exp2 of the score below the
// running maximum, rounded to fp16: all down to 2^-28 of the largest have 11 bits.  A tile's products are added to the sums in 32 bits, times
// the values' scale of its page, so pages of any scales may meet.
//
// Tokens of the unfinished page take the same way as 16-token tiles of the ring: keys times queries in the cache's type, scaled by a power
// of two as well, and weights as a sum of two numbers of it.
#include "mma_utils.cuh"
#include "q8_common.cuh"

namespace anna {

template <int D, int NT>
struct Q8Cfg {
  static constexpr int kWarps = NT == 1 && D <= 128 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  // per SM, by registers: 128, 168 or 255 a thread
  static constexpr int kCtas = NT == 1 ? (D <= 128 ? 2 : 3) : NT == 2 && D <= 128 ? 3 : 2;
  static constexpr int kRows = 8 * NT;
  static constexpr int kSteps = D / 16;          // products over the dims of a key
  static constexpr int kChunks = D / 64;         // 16-byte pieces of a lane's key
  static constexpr int kVWords = D / 32;         // 4-byte words of a lane's value
  static constexpr int kMergeStride = D + 4;     // floats
  static constexpr int kOffFrags = 0;                                   // [NT][steps][32 lanes] uint2: queries as second operands
  static constexpr int kOffRing = kOffFrags + NT * kSteps * 256;        // [rows][D] queries in the cache's type
  static constexpr int kOffStats = kOffRing + kRows * D * 2;             // [warps][rows] float2
  static constexpr int kOffRate = kOffStats + kWarps * kRows * 8;       // [rows] to units of log2 of a weight; in the end 1 / denominator
  static constexpr int kOffMerge = kOffRate + kRows * 4;                // [warps][8][stride] floats, or the weights of a merge
  static constexpr int kMergeBytes = kWarps * 8 * kMergeStride * 4;
  static constexpr int kWeightBytes = kRows * kMultiMaxPartials * 4;
  static constexpr int kSmem = kOffMerge + (kMergeBytes > kWeightBytes ? kMergeBytes : kWeightBytes);
};

__device__ __forceinline__ uint32_t q8_sub_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Bytes (flipped codes) 0 and 1, or 2 and 3, of x as two fp16.
template <int PAIR>
__device__ __forceinline__ uint32_t q8_halves(uint32_t x) {
  return q8_sub_half2(__byte_perm(x, 0x64646464u, PAIR == 0 ? 0x4140 : 0x4342), 0x64806480u);
}
template <typename T>
__device__ __forceinline__ void q8_mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void q8_mma_zero<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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

template <typename T, int D, int NT, bool kBlocks>
__global__ void __launch_bounds__(Q8Cfg<D, NT>::kThreads, Q8Cfg<D, NT>::kCtas) q8_mma_kernel(const Q8Params p, int row_tiles) {
  using Cfg = Q8Cfg<D, NT>;
  constexpr int kTile = kBalancedTileTokens;
  constexpr int kFar = 0x7fff0000;  // position of a token that nobody sees
  constexpr float kRingFactor = std::is_same_v<T, __half> ? 1.0f : 1.0f / 16384.0f;
  extern __shared__ __align__(16) uint8_t smem[];
  const uint2* frags = reinterpret_cast<const uint2*>(smem + Cfg::kOffFrags) + (threadIdx.x & 31);
  float* rate = reinterpret_cast<float*>(smem + Cfg::kOffRate);
  float2* stats = reinterpret_cast<float2*>(smem + Cfg::kOffStats);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  q8_let_next_start();
  q8_wait_for_previous();

  q8_for_each_segment<T, D, Cfg::kThreads, kBlocks>(p, row_tiles, [&](int64_t b, int kvh, int tile, int64_t t0, int64_t t1, const MultiPartial& part) {
  const Q8Stream st = q8_stream<Cfg::kRows>(p, b, kvh, tile);
  const int first_seen = (int)(st.len - p.tokens);  // newest key that query 0 sees
  const int packed_tiles = max(0, (int)(min(t1, st.packed) - t0 + kTile - 1)) / kTile;
  const int mine = packed_tiles > warp ? (packed_tiles - warp + Cfg::kWarps - 1) / Cfg::kWarps : 0;  // tiles of this warp: every kWarps-th

  // ---- pages of 32 of the warp's tiles, one a lane ------------------------------------------------------------------------------------
  struct Pages {
    const uint8_t* keys;
    int position;  // of the tile's first token in the sequence
    float2 scale;
  };
  auto find = [&](int from) {  // pages and positions; the scales are read by `scales`
    Pages x{p.pages, kFar, make_float2(0.0f, 0.0f)};
    const int i = from + lane;
    if (i < mine) {
      const int at = (int)t0 + (warp + i * Cfg::kWarps) * kTile;
      const int entry = p.block_shift >= 0 ? at >> p.block_shift : at / p.block_size, slot = at - entry * p.block_size;
      int block;
      const int64_t page = q8_page_at(p, st, b, kvh, entry, &block);
      if (page >= 0) {
        x.keys = p.pages + page + slot * D;
        x.position = block * p.block_size + slot;
      }
    }
    return x;
  };
  auto scales = [&](Pages& x) {
    // a tile's keys begin `slot` rows behind its page
    if (x.position != kFar)
      x.scale = __ldg(reinterpret_cast<const float2*>(x.keys + (int64_t)(2 * p.block_size - x.position % p.block_size) * D));
  };
  uint4 key[2][Cfg::kChunks];
  uint32_t val[4][Cfg::kVWords];
  auto load_keys = [&](const uint8_t* keys) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < Cfg::kChunks; ++c) key[i][c] = ldg_stream16(keys + (gid + 8 * i) * D + 64 * c + 16 * tig);
  };
  const int values_at = p.block_size * D;
  auto load_values = [&](const uint8_t* keys) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* from = keys + values_at + (2 * tig + (i & 1) + 8 * (i / 2)) * D + gid * (D / 8);
      if constexpr (D == 64) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(from));
        val[i][0] = v.x; val[i][1] = v.y;
      } else {
#pragma unroll
        for (int c = 0; c < D / 128; ++c) {
          const uint4 v = ldg_stream16(from + 16 * c);
          val[i][4 * c] = v.x; val[i][4 * c + 1] = v.y; val[i][4 * c + 2] = v.z; val[i][4 * c + 3] = v.w;
        }
      }
    }
  };
  auto broadcast = [&](const uint8_t* x, int from) {
    return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)x, from));
  };
  Pages now = find(0), next = now;
  const uint8_t* at = broadcast(now.keys, 0);
  if (mine > 0) {
    load_keys(at);
    load_values(at);
    scales(now);
    if (mine > 32) next = find(32);
  }

  // ---- queries -----------------------------------------------------------------------------------------------------------------------
  for (int i = warp; i < Cfg::kRows; i += Cfg::kWarps) {
    constexpr int E = D / 32;
    float x[E], top = 0.0f;
    const int row = st.row0 + min(i, st.count - 1), t = multi_token_of(p, row), h = kvh * p.groups + row - t * p.groups;
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_stride_b + h * p.q_stride_h + t * p.q_stride_t + lane * E;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      x[j] = ElemTraits<T>::to_float(q[j]);
      top = fmaxf(top, fabsf(x[j]));
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    int up = top > 0.0f && top < INFINITY ? 14 + 127 - (int)(__float_as_uint(top) >> 23) : 0;  // top * 2^up is in [2^14, 2^15)
    up = min(up, 126);
    const float factor = __uint_as_float((uint32_t)(up + 127) << 23);
    if (lane == 0) rate[i] = p.scaling * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int d = lane * E + j;
      const int place = ((i / 8 * Cfg::kSteps + d / 64 * 4 + d % 16 / 4) * 32 + i % 8 * 4 + d % 64 / 16) * 4 + d % 4;
      reinterpret_cast<__half*>(smem + Cfg::kOffFrags)[place] = __float2half_rn(x[j] * factor);
      // under 2^15 in fp16, under 2 in bf16, whose keys may be as large as a product
      reinterpret_cast<T*>(smem + Cfg::kOffRing)[i * D + d] = ElemTraits<T>::from_float(x[j] * factor * kRingFactor);
    }
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

  // Scores of 16 tokens (rows gid and gid + 8 of every column pair) become weights, at 2^14 times their size.
  auto softmax = [&](float (&s)[NT][4]) {
    bool more = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) more = more || fmaxf(s[j][k], s[j][k + 2]) > m_run[j][k];
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
        const float base = m_run[j][k] == -INFINITY ? 0.0f : m_run[j][k] - 14.0f;
        s[j][k] = q8_exp2(s[j][k] - base);
        s[j][k + 2] = q8_exp2(s[j][k + 2] - base);
        l_run[j][k] += s[j][k] + s[j][k + 2];
      }
  };

  // ---- packed tiles -------------------------------------------------------------------------------------------------------------------
  for (int i = 0; i < mine; ++i) {
    const int position = __shfl_sync(0xffffffffu, now.position, i & 31);
    const float2 scale = make_float2(__shfl_sync(0xffffffffu, now.scale.x, i & 31), __shfl_sync(0xffffffffu, now.scale.y, i & 31));
    if ((i & 31) == 31 && i + 1 < mine) {
      now = next;
      scales(now);
      if (i + 33 < mine) next = find(i + 33);
    }
    at = broadcast(now.keys, (i + 1) & 31);
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[j][r] = 0.0f;
#pragma unroll
    for (int c = 0; c < Cfg::kChunks; ++c) {
      const uint32_t wa[4] = {key[0][c].x, key[0][c].y, key[0][c].z, key[0][c].w};
      const uint32_t wb[4] = {key[1][c].x, key[1][c].y, key[1][c].z, key[1][c].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t ua = wa[x] ^ 0x80808080u, ub = wb[x] ^ 0x80808080u;
        const uint32_t a[4] = {q8_halves<0>(ua), q8_halves<0>(ub), q8_halves<1>(ua), q8_halves<1>(ub)};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint2 q = frags[(j * Cfg::kSteps + 4 * c + x) * 32];
          mma_m16n8k16<__half>(s[j], a, q.x, q.y);
        }
      }
    }
    if (i + 1 < mine) load_keys(at);
    float by[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x = scale.x * to_log2[j][k];
        s[j][k] *= x;
        s[j][k + 2] *= x;
        by[j][k] = scale.y;
      }
    if (position + kTile - 1 > first_seen) {  // tokens that some rows do not see, or a page that is none
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int last = limit(j, k);
          if (position + gid > last) s[j][k] = -INFINITY;
          if (position + gid + 8 > last) s[j][k + 2] = -INFINITY;
          if (position > last) by[j][k] = 0.0f;  // the scale may be NaN
        }
    }
    softmax(s);
    uint32_t w[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) w[j][k] = movmatrix_trans(pack2<__half>(s[j][2 * k], s[j][2 * k + 1]));
#pragma unroll
    for (int v = 0; v < Cfg::kVWords; ++v) {
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = val[k][v] ^ 0x80808080u;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t x = __byte_perm(u[0], u[1], half == 0 ? 0x5140 : 0x7362), z = __byte_perm(u[2], u[3], half == 0 ? 0x5140 : 0x7362);
        const uint32_t a[4] = {q8_halves<0>(x), q8_halves<1>(x), q8_halves<0>(z), q8_halves<1>(z)};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float sum[4];
          q8_mma_zero<__half>(sum, a, w[j][0], w[j][1]);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[j][2 * v + half][r] = fmaf(sum[r], by[j][r & 1], o[j][2 * v + half][r]);
        }
      }
    }
    if (i + 1 < mine) load_values(at);
  }

  // ---- tiles of the ring ----------------------------------------------------------------------------------------------------------------
  const int64_t ring_from = max(t0, st.packed);
  const int64_t slot = ring_from < t1 ? p.window_slots[b] : -1;
  if (slot >= 0 && slot < p.num_slots) {
    const T* keys = reinterpret_cast<const T*>(p.window) + (slot * 2 * p.kv_heads + kvh) * p.block_size * D;
    const T* values = keys + (int64_t)p.kv_heads * p.block_size * D;
    const int begin = (int)(ring_from - st.packed), end = (int)(t1 - st.packed), full = (int)st.full;  // ring slots; position of slot 0
    for (int from = begin + (warp + Cfg::kWarps - packed_tiles % Cfg::kWarps) % Cfg::kWarps * kTile; from < end; from += Cfg::kWarps * kTile) {
      const int valid = min(kTile, end - from), position = full + from;
      auto row_of = [&](int token) { return (int64_t)(from + min(token, valid - 1)) * D; };
      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[j][r] = 0.0f;
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
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int token = gid + 8 * (r / 2);
          s[j][r] = token >= valid || position + token > limit(j, r & 1) ? -INFINITY : s[j][r] * (to_log2[j][r & 1] / kRingFactor);
        }
      softmax(s);
      // weights as a sum of two of the type, so that they keep 16 bits and more
      uint32_t w[NT][2], rest[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float x = s[j][2 * k], y = s[j][2 * k + 1];
          const uint32_t most = pack2<T>(x, y);
          const T* parts = reinterpret_cast<const T*>(&most);
          w[j][k] = movmatrix_trans(most);
          rest[j][k] = movmatrix_trans(pack2<T>(x - ElemTraits<T>::to_float(parts[0]), y - ElemTraits<T>::to_float(parts[1])));
        }
      bool strange = false;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {  // 8 of a lane's dims
        uint32_t x[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int token = 2 * tig + (k & 1) + 8 * (k / 2);
          const uint4 got = token < valid ? *reinterpret_cast<const uint4*>(values + row_of(token) + gid * (D / 8) + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
          x[k][0] = got.x; x[k][1] = got.y; x[k][2] = got.z; x[k][3] = got.w;
#pragma unroll
          for (int v = 0; v < 4; ++v) {  // an infinite or NaN value must not meet a weight of 0: of a row that does not see it, of a rest
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
      if (__any_sync(0xffffffffu, strange)) {  // what was left out, for the rows that see it
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
    // a NaN among the scores has to stay one, so only a row without a key is zero
    rate[i] = part.count > 1 ? 1.0f : den == 0.0f ? 0.0f : 1.0f / den;
    if (part.count > 1 && i < st.count)
      reinterpret_cast<float2*>(p.stats)[multi_partial_row(part, part.mine, Cfg::kRows) + i] = make_float2(top * 0.6931471805599453f, den);
  }
  __syncthreads();
  float* merged = reinterpret_cast<float*>(smem + Cfg::kOffMerge);
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

Q8Shape q8_mma_shape(int head_dim, int rows) {
  auto of = [](auto cfg) { return Q8Shape{decltype(cfg)::kRows, decltype(cfg)::kCtas, decltype(cfg)::kWarps}; };
  if (head_dim == 64) return rows <= 8 ? of(Q8Cfg<64, 1>{}) : rows <= 16 ? of(Q8Cfg<64, 2>{}) : of(Q8Cfg<64, 4>{});
  if (head_dim == 128) return rows <= 8 ? of(Q8Cfg<128, 1>{}) : rows <= 16 ? of(Q8Cfg<128, 2>{}) : of(Q8Cfg<128, 4>{});
  return rows <= 8 ? of(Q8Cfg<256, 1>{}) : of(Q8Cfg<256, 2>{});
}

template <typename T, int D, int NT>
static int launch(const Q8Params& p, int row_tiles, int ctas, cudaStream_t stream) {
  using Cfg = Q8Cfg<D, NT>;
  auto kernel = p.blocks != nullptr ? q8_mma_kernel<T, D, NT, true> : q8_mma_kernel<T, D, NT, false>;
  ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
  return q8_launch("q8_mma_kernel", kernel, dim3((unsigned)ctas), Cfg::kThreads, Cfg::kSmem, stream, p, row_tiles);
}

int launch_q8_mma(const Q8Params& p, const Q8Plan& plan, int head_dim, int dtype, int ctas, cudaStream_t stream) {
  auto pick = [&](auto elem) -> int {
    using T = decltype(elem);
    if (head_dim == 64)
      return plan.rows == 8 ? launch<T, 64, 1>(p, plan.row_tiles, ctas, stream) : plan.rows == 16 ? launch<T, 64, 2>(p, plan.row_tiles, ctas, stream)
                                                                                                : launch<T, 64, 4>(p, plan.row_tiles, ctas, stream);
    if (head_dim == 128)
      return plan.rows == 8 ? launch<T, 128, 1>(p, plan.row_tiles, ctas, stream) : plan.rows == 16 ? launch<T, 128, 2>(p, plan.row_tiles, ctas, stream)
                                                                                                 : launch<T, 128, 4>(p, plan.row_tiles, ctas, stream);
    return plan.rows == 8 ? launch<T, 256, 1>(p, plan.row_tiles, ctas, stream) : launch<T, 256, 2>(p, plan.row_tiles, ctas, stream);
  };
  return dtype == ANNA_DTYPE_F16 ? pick(__half{}) : pick(__nv_bfloat16{});
}

}  // namespace anna
