// Tensor-core form of the multi-token decode over packed TurboQuant pages (16-bit caches, head_dim 64, 128 and 256).
//
// The T * G queries of a KV head are the 16-row A operand of mma.sync m16n8k16 (fp16 in, fp32 out), the tokens its columns, so a key
// that has been de-quantized serves 16 * MT rows and the probabilities of a tile are the A operand of the value product as they
// come out of the score product.  Per warp and step of two 16-token tiles:
//
//   packed bytes --bulk copy (cp.async.bulk, mbarrier)--> shared memory, two stages per warp
//   S[rows x tokens]  = Q1 . centroid(idx) + Q2 . (+-rnorm)       both products into one accumulator: K = 2 D
//       Q1 = fwht(s1*q), Q2 = sqrt(pi/2)/sqrt(D) * fwht(s2*Q1), each row scaled to a largest value of 1 and rounded to fp16
//   score (log2 units) = f_row * norm_token * S,   f_row = largest value of the row * |scaling| * log2(e) / D
//   online softmax in fp32 on the accumulators, P rounded to fp16
//   O[rows x D] += P . (code * scale + zero)                       value codes as fp16 by exponent bits
//
// The k-slots of the products and the columns of O are free to permute: a lane takes the coordinates whose codes it can unpack with
// the fewest instructions, and 2 * D/8 neighbouring dims of an output row.
//
// Bound: the packed bytes of a sequence from HBM, once for 16 or 32 of its queries; today the issue of instructions.  4 new tokens of 16 rows
// of 32768, 32/8 heads of 128, 4 bits: 269 us, 2.4 TB/s, 556 instructions per tile and warp (55 % of the issue slots, logic pipe 53 %,
// products 34 % of their pipe).  A CTA of eight warps splits a share's steps among them, so that a share of 32 tiles is two steps of each
// warp and the merge of their rows is one per share; two CTAs per SM (16 rows, up to 128 dims) is what the 128 registers of a thread
// leave.  32 rows a CTA (two row tiles) unpack a key once for both, with half the warps: 8 new tokens 419 us, twice 269 as two calls.
//
// What is rounded below 32 bits: the rotated queries, centroids and residual norms to fp16 (2^-12 of the row's largest value, of the
// centroid and of the norm), probabilities and values to fp16 (2^-12 of themselves; small probabilities: see kTopLog2).  Together they
// stay below the rounding of a bf16 output (2^-9 of the value); for fp16 see kSplit.  Values keep to fp16's range by powers of two (see
// `lift`): those of a bf16 cache that are small beside others of their dims in a warp's keys are off by 2^-19 of the largest, at most.
#pragma once

#include "mbarrier_utils.cuh"
#include "tq_multi_params.cuh"

namespace anna {

static __device__ int32_t g_tq_multi_faults;  // bumped when a bounded wait on a tile copy expires; one of each object

constexpr int kMultiMmaWarps = 8, kMultiMmaThreads = 32 * kMultiMmaWarps;
constexpr int kTile = 16;        // tokens
constexpr int kStepTiles = 2;    // tiles of a step: one softmax update
constexpr int kRingStages = 2;   // steps of a warp's ring
// Probabilities are fp16 in the value product, whose range goes from 2^15 down to 2^-24: the running maximum stands at 2^7, and may be
// exceeded by 2^8 before it moves.  So a weight has all its bits down to 2^-21 of the largest, and what is rounded below is at most
// 2^-32 of it: of n such keys together, n * 2^-32.  (With the maximum at 1, 2^-25 of it: beside one key of 99 % of the weight the others
// of 32768 were off by 2.5e-4 of the output, those of 99.9 % by 2.6e-2.)
constexpr float kMoveLimit = 8.0f, kTopLog2 = 7.0f;

template <typename T, int D, int BITS, int MT>
struct MultiCfg {
  // An fp16 output shows what Q1 and P lose as one fp16 each, so that they are sums of two there, with a product for either part: 16 rows
  // of 0.4-4 K tokens, 256 dims, 64 queries to a KV head, off by 2.8e-4 of the output instead of 3.9e-4 (2.1e-4 is its own rounding), 84 us
  // instead of 74; 16 rows of 32768 tokens, 128 dims, 328 instead of 269.  A bf16 output hides it.
  static constexpr bool kSplit = std::is_same_v<T, __half>;
  static constexpr int kPlanes = kSplit ? 3 : 2;
  static constexpr int kRows = 16 * MT;
  static constexpr int kSteps = D / 16;  // k-steps of one product
  static constexpr int kGroups = D / 32;
  static constexpr int kKeyBytes = D * BITS / 8;
  static constexpr int kValBytes = D / (BITS == 2 ? 4 : 2);
  // a tile in shared memory has the layout of a 16-token page
  static constexpr int kOffNorm = kTile * kKeyBytes;
  static constexpr int kOffRnorm = kOffNorm + 4 * kTile;
  static constexpr int kOffVal = kOffRnorm + 4 * kTile;
  static constexpr int kOffScale = kOffVal + kTile * kValBytes;
  static constexpr int kOffZero = kOffScale + kTile * kGroups * 2;
  static constexpr int kTileBytes = kOffZero + kTile * kGroups * 2;
  static constexpr int kTileStride = (kTileBytes + 127) / 128 * 128;
  static constexpr int kWarpRing = kRingStages * kStepTiles * kTileStride;
  static constexpr int kRing = kMultiMmaWarps * kWarpRing;
  static constexpr int kQuery = MT * kPlanes * kSteps * 32 * 16;  // A fragments of Q1, of Q2, of what is left of Q1
  // the merge of the warps: a row of O with its quarters 8 floats apart, so that the lanes that store together hit other banks
  static constexpr int kMergeStride = D + 8 * (D / 32) + 4;
  static constexpr int kMerge = kMultiMmaWarps * 16 * kMergeStride * 4;
  static constexpr int kWork = kRing + kQuery > kMerge ? kRing + kQuery : kMerge;
  static_assert(kWork >= kRows * kMultiMaxPartials * 4, "the weights of the partials lie there, too");
  static constexpr int kOffBars = kWork;                                  // mbarriers [warps][stages]
  static constexpr int kOffValid = kOffBars + kMultiMmaWarps * kRingStages * 8;  // tokens of the pieces [warps][stages][tiles or halves]
  static constexpr int kOffFactor = kOffValid + kMultiMmaWarps * kRingStages * kStepTiles * 8;  // f_row [rows]
  static constexpr int kOffLimit = kOffFactor + kRows * 4;                // newest key that the row sees [rows]
  static constexpr int kOffStats = kOffLimit + kRows * 4;                 // m, l of the warps [warps][rows][2]
  static constexpr int kOffStrange = kOffStats + kMultiMmaWarps * kRows * 8;  // see strange_values
  static constexpr int kSmem = kOffStrange + 8;
  static constexpr int kCtas = D <= 128 && MT == 1 ? 2 : 1;  // per SM
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_elem(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_elem<__half>(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) { mma_f16(d, a, b0, b1); }
template <>
__device__ __forceinline__ void mma_elem<__nv_bfloat16>(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 mul_f32x2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add_f32x2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}\n"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma_f32x2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 w, x, y, z;\n"
      " mov.b64 {%0, %1}, w;\n}\n"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
template <int LUT>
__device__ __forceinline__ uint32_t lop3(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, %4;\n" : "=r"(r) : "r"(a), "r"(b), "r"(c), "n"(LUT));
  return r;
}
constexpr int kAndOr = 0xEA, kAndXor = 0x6A;  // (a & b) | c, (a & b) ^ c
// Byte permute in PTX's default mode: nibble i of the low half of `sel` names byte i of the result among {a, b}.
__device__ __forceinline__ uint32_t permute(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;\n" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Larger of two values, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// x << n as a product: the multiply pipe has room, the logic pipe has not
__device__ __forceinline__ uint32_t times_power(uint32_t x, int n) {
  if (n == 0) return x;
  uint32_t r;
  asm("mul.lo.u32 %0, %1, %2;\n" : "=r"(r) : "r"(x), "r"(1u << n));
  return r;
}

// A value of the window that some rows see and others do not may be infinite or NaN, and zero times that is NaN: where a tile is cut by
// the rows' limits, such values go into the product as zeros, and the rows that see them get them at the end (strange_values).
template <typename T>
__device__ __forceinline__ uint32_t finite_halves(uint32_t pair) {  // all ones in the halves that are finite
  constexpr uint32_t kExp = std::is_same_v<T, __half> ? 0x7C007C00u : 0x7F807F80u, kOne = std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
  const uint32_t over = ((pair & kExp) + kOne) & 0x80008000u;  // the exponent's carry
  return ~((over >> 15) * 0xffffu);
}

// Of either half, the larger magnitude, NaN if either is (its sign is of no use).
template <typename T>
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>) asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* ptr, uint32_t (&dst)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(ptr)[i];
      dst[4 * i] = v.x; dst[4 * i + 1] = v.y; dst[4 * i + 2] = v.z; dst[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(ptr);
    dst[0] = v.x; dst[1] = v.y;
  } else {
    static_assert(N == 1, "unsupported word count");
    dst[0] = *reinterpret_cast<const uint32_t*>(ptr);
  }
}

// Where coordinate c of a row goes in the A fragments of a product: k-step, lane's tig, register (0: k 2tig.., 1: k 2tig + 8..), half.
struct FragSlot {
  int step, tig, reg, half;
};
// Centroids: eight codes of a nibble word are two k-steps, four neighbouring nibbles each.  A nibble word is a word of 4-bit codes, or
// the even or the odd fields of a word of 2-bit fields.
template <int D, int BITS>
__device__ __forceinline__ FragSlot index_slot(int c) {
  const int tig = c / (D / 4), j = c % (D / 4);
  const int word = BITS == 4 ? j / 8 : 2 * (j / 16) + (j & 1);
  const int i = BITS == 4 ? j % 8 : j % 16 / 2;
  return {2 * word + i / 4, tig, i % 4 / 2, i % 2};
}
// Signs: a mask leaves two bits of a word 16 positions apart, so halves of a register are four nibbles (16 bits of a plane) apart.
template <int D, int BITS>
__device__ __forceinline__ FragSlot sign_slot(int c) {
  const int tig = c / (D / 4), j = c % (D / 4);
  if (BITS == 3 && D == 64) return {j % 8 / 2, tig, j % 2, j / 8};  // 16 bits, spread to halves of 8
  if (BITS == 3) return {8 * (j / 32) + j % 16 / 2, tig, j % 2, j % 32 / 16};
  const int word = BITS == 4 ? j / 8 : 2 * (j / 16) + (j & 1);
  const int i = BITS == 4 ? j % 8 : j % 16 / 2;
  return {2 * word + i % 4 / 2, tig, i % 2, i / 4};
}

template <typename T, int D, int BITS, int MT, bool HALVED>
__global__ void __launch_bounds__(kMultiMmaThreads, MultiCfg<T, D, BITS, MT>::kCtas)
    tq_multi_mma_kernel(const TqMultiParams p, int row_tiles) {
  using Cfg = MultiCfg<T, D, BITS, MT>;
  constexpr int E = D / 32;
  constexpr int kKeyWords = BITS == 4 ? D / 32 : D / 64;  // of a lane's D/4 coordinates of a token: codes or indices
  constexpr int kSignWords = BITS == 3 && D > 64 ? D / 128 : 1;
  constexpr int kValWords = BITS == 2 && D > 64 ? D / 128 : D / 64;  // of a lane's D/8 dims of a token; of 64 2-bit codes, half a word
  constexpr int kCols = 2 * kStepTiles;                     // 8-token columns of a step
  extern __shared__ __align__(1024) uint8_t smem[];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  uint8_t* ring = smem + warp * Cfg::kWarpRing;
  const uint32_t bars = smem_u32(smem + Cfg::kOffBars) + warp * kRingStages * 8;
  volatile int* ring_valid = reinterpret_cast<volatile int*>(smem + Cfg::kOffValid) + warp * kRingStages * kStepTiles * 2;
  int* strange = reinterpret_cast<int*>(smem + Cfg::kOffStrange);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kRingStages; ++i) mbar_init(bars + 8 * i, 1);
    mbar_init_fence();
  }
  // The centroids are rounded to fp16; for an fp16 cache at the scale, of 512 between 1 and 2, that leaves the smallest squared error
  // over the codebook: as they are, their rounding was the largest error of its output.  A bf16 output hides it, and the search costs
  // 2 % of a long call (verification of 4 tokens over 16 rows of 32768: 259 -> 256 us without it).
  constexpr int kCentroids = 1 << (BITS - 1);
  float cent[kCentroids];
#pragma unroll
  for (int e = 0; e < kCentroids; ++e) cent[e] = __ldg(p.centroids + e);
  float cent_scale = 1.0f;
  if constexpr (std::is_same_v<T, __half>) {
    auto scale_of = [](uint32_t j) { return 1.0f + (float)j * (1.0f / 512.0f); };
    uint32_t best = 0xffffffffu;  // error (its lowest bits left out), number of the scale
#pragma unroll
    for (int i = 0; i < 512 / kMultiMmaThreads; ++i) {
      const uint32_t j = i * kMultiMmaThreads + threadIdx.x;
      float error = 0.0f;
#pragma unroll
      for (int e = 0; e < kCentroids; ++e) {
        const float x = cent[e] * scale_of(j), d = x - __half2float(__float2half_rn(x));
        error = fmaf(d, d, error);
      }
      error /= scale_of(j) * scale_of(j);
      best = min(best, (__float_as_uint(error) & ~511u) | j);
    }
    best = __reduce_min_sync(0xffffffffu, best);
    uint32_t* best_of = reinterpret_cast<uint32_t*>(smem + Cfg::kOffStats);
    if (lane == 0) best_of[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMultiMmaWarps; ++w) best = min(best, best_of[w]);
    cent_scale = scale_of(best & 511u);
  }
  // tables of the centroids' low and high bytes
  uint32_t lut_lo[2] = {0u, 0u}, lut_hi[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < kCentroids; ++e) {
    const uint32_t bits = __half_as_ushort(__float2half_rn(cent[e] * cent_scale));
    lut_lo[e / 4] |= (bits & 0xffu) << (8 * (e % 4));
    lut_hi[e / 4] |= (bits >> 8) << (8 * (e % 4));
  }
  uint32_t phase = 0;  // of the ring, which goes on from segment to segment
  int stage = 0;
  bool dead = false;  // a bounded wait expired: this warp consumes nothing any more

  multi_for_each_segment<T, D, kMultiMmaThreads>(p, row_tiles, [&](int b, int kvh, int tile, int t0, int t1, const MultiPartial& part) {
  const int row0 = tile * Cfg::kRows, count = min(Cfg::kRows, p.rows - row0);
  const int len = (int)max((int64_t)0, min(p.lengths[b], p.max_len));
  const int lq = max(0, len - p.residual_len);
  const int q_end = min(t1, lq);
  const int first_seen = len - p.tokens;  // newest key that query 0 sees
  if (threadIdx.x == 0) *strange = 0;

  // ---- copies of the first steps ---------------------------------------------------------------------------------------------
  const int tiles = q_end > t0 ? (q_end - t0 + kTile - 1) / kTile : 0;
  const int steps = (tiles + kStepTiles - 1) / kStepTiles;
  const int my_steps = steps > warp && !dead ? (steps - warp + kMultiMmaWarps - 1) / kMultiMmaWarps : 0;
  const int32_t* table = p.block_table + (int64_t)b * p.table_stride;
  // A piece is a run of tokens of one page: a tile, or half a tile where a page is no multiple of 16 tokens.
  // (Decided at run time, 16 rows of 32768 tokens took 264 us instead of 261.)
  constexpr int halved = HALVED ? 1 : 0, piece_tokens = kTile >> halved, group_steps = 16 >> halved;  // steps whose pieces are 32
  const int piece = lane & ((kStepTiles << halved) - 1);                                               // the lane's piece of a step
  // Page ids of the warp's next 32 pieces, one a lane, and those of the 32 behind them: a step that looks up its own waits for the table
  // before it can ask for the tokens.
  auto ids_of = [&](int group) {
    const int step = group * group_steps + (lane >> (1 + halved));
    const int ts = t0 + (step * kMultiMmaWarps + warp) * kStepTiles * kTile + piece * piece_tokens;
    if (ts >= q_end) return -1;
    const int blk = p.block_shift >= 0 ? ts >> p.block_shift : ts / p.block_size;
    return blk < p.max_blocks ? table[blk] : -1;
  };
  int32_t ids = ids_of(0), ids_next = ids_of(1);
  // A tile of a 16-token page is one run of bytes, other pieces are six (codes, norms, residual norms, value codes, scales, zeros).
  // The first lanes copy a piece each; lane 0 arms the barrier with the bytes of all.
  auto issue = [&](int step, int stage) {
    const int in_group = step & (group_steps - 1);
    if (in_group == 0 && step > 0) {
      ids = ids_next;
      ids_next = ids_of(step / group_steps + 1);
    }
    const int32_t pid = __shfl_sync(0xffffffffu, ids, (in_group << (1 + halved)) + piece);
    int valid = 0, at = 0;
    const uint8_t* page = nullptr;
    const bool copies = lane < kStepTiles << halved;
    if (copies) {
      const int ts = t0 + (step * kMultiMmaWarps + warp) * kStepTiles * kTile + piece * piece_tokens;
      if (pid >= 0 && pid < p.num_pages) {  // else a hole, or behind the end: nothing to copy
        valid = min(piece_tokens, q_end - ts);
        at = p.block_size == kTile ? 0 : p.block_shift >= 0 ? ts & (p.block_size - 1) : ts % p.block_size;
        page = p.pages + ((int64_t)pid * p.kv_heads + kvh) * p.layout.chunk_bytes;
      }
      ring_valid[stage * (kStepTiles << halved) + lane] = valid;
    }
    const uint32_t bar = bars + 8 * stage;
    const unsigned have = __ballot_sync(0xffffffffu, valid > 0);
    if (lane == 0) {
      if (have != 0u) mbar_expect_tx(bar, (uint32_t)__popc(have) * (Cfg::kTileBytes >> halved));
      else mbar_arrive(bar);  // the phase completes at once
    }
    __syncwarp();
    if (valid > 0) {
      const uint32_t dst = smem_u32(ring + (stage * kStepTiles + (lane >> halved)) * Cfg::kTileStride);
      if (p.block_size == kTile) {
        bulk_copy_g2s(dst, page, Cfg::kTileBytes, bar);
      } else {
        const int to = (lane & halved) * piece_tokens;
        bulk_copy_g2s(dst + to * Cfg::kKeyBytes, page + p.layout.off_kcodes + at * Cfg::kKeyBytes, piece_tokens * Cfg::kKeyBytes, bar);
        bulk_copy_g2s(dst + Cfg::kOffNorm + 4 * to, page + p.layout.off_knorm + 4 * at, 4 * piece_tokens, bar);
        bulk_copy_g2s(dst + Cfg::kOffRnorm + 4 * to, page + p.layout.off_krnorm + 4 * at, 4 * piece_tokens, bar);
        bulk_copy_g2s(dst + Cfg::kOffVal + to * Cfg::kValBytes, page + p.layout.off_vdata + at * Cfg::kValBytes,
                      piece_tokens * Cfg::kValBytes, bar);
        bulk_copy_g2s(dst + Cfg::kOffScale + to * Cfg::kGroups * 2, page + p.layout.off_vscale + at * Cfg::kGroups * 2,
                      piece_tokens * Cfg::kGroups * 2, bar);
        bulk_copy_g2s(dst + Cfg::kOffZero + to * Cfg::kGroups * 2, page + p.layout.off_vzero + at * Cfg::kGroups * 2,
                      piece_tokens * Cfg::kGroups * 2, bar);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kRingStages - 1; ++i)
    if (i < my_steps) issue(i, (stage + i) % kRingStages);

  // Scale and zero of this lane's column as B operand in one of the first tile's tokens 3, 7, 11 and 15, on their way behind the copies.
  T first_scale = T(0.0f), first_zero = T(0.0f);
  if constexpr (!std::is_same_v<T, __half>) {
    if (my_steps > 0) {
      const int in_tile = min(4 * tig + 3, q_end - 1 - t0 - warp * (kStepTiles * kTile)), ts = t0 + warp * (kStepTiles * kTile) + in_tile;
      const int32_t pid = __shfl_sync(0xffffffffu, ids, in_tile / piece_tokens);
      if (pid >= 0 && pid < p.num_pages) {
        const int at = p.block_shift >= 0 ? ts & (p.block_size - 1) : ts % p.block_size;
        const uint8_t* page = p.pages + ((int64_t)pid * p.kv_heads + kvh) * p.layout.chunk_bytes;
        const int where = at * Cfg::kGroups + gid * (D / 8) / 32;
        first_scale = reinterpret_cast<const T*>(page + p.layout.off_vscale)[where];
        first_zero = reinterpret_cast<const T*>(page + p.layout.off_vzero)[where];
      }
    }
  }

  // ---- rotated queries as A fragments ----------------------------------------------------------------------------------------
  float* factor = reinterpret_cast<float*>(smem + Cfg::kOffFactor);
  int* row_limit = reinterpret_cast<int*>(smem + Cfg::kOffLimit);
  __half* frags = reinterpret_cast<__half*>(smem + Cfg::kRing);
  {
    const float sign = p.scaling < 0.0f ? -1.0f : 1.0f;
    const float kappa = 1.2533141373155001f * rsqrt_dim_const<D>();
    float s1[E], s2[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      s1[j] = p.signs1[lane * E + j] * sign;
      s2[j] = p.signs2[lane * E + j];
    }
    for (int i = warp; i < Cfg::kRows; i += kMultiMmaWarps) {
      const int up = i % 16 / 8, m = i / 16, row_lane = 4 * (i % 8);
      if (i >= count) {  // a row that is not there: zeros, which see no key
        if (lane == 0) {
          row_limit[i] = -1;
          factor[i] = 1e-30f;
        }
        for (int k = lane; k < Cfg::kPlanes * Cfg::kSteps * 4; k += 32) {
          uint32_t* words = reinterpret_cast<uint32_t*>(frags) + ((m * Cfg::kPlanes * Cfg::kSteps + k / 4) * 32 + row_lane + k % 4) * 4 + up;
          words[0] = words[2] = 0u;
        }
        continue;
      }
      const int row = row0 + i;
      const int t = multi_token_of(p, row);
      const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_stride_b + (int64_t)(kvh * p.groups + row - t * p.groups) * p.q_stride_h +
                   (int64_t)t * p.q_stride_t + lane * E;
      float w1[E], w2[E];
      lane_load<T, E>(q, w1);
#pragma unroll
      for (int j = 0; j < E; ++j) w1[j] *= s1[j];
      warp_fwht<E>(w1, lane);
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        top = max_nan(top, fabsf(w1[j]));
        w2[j] = w1[j] * s2[j];
      }
      warp_fwht<E>(w2, lane);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        w2[j] *= kappa;
        top = max_nan(top, fabsf(w2[j]));
      }
      // as integers, non-negative floats keep their order and a NaN is above all of them
      top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
      const float inv = top == 0.0f ? 0.0f : 1.0f / top;
      // a factor of zero (a zero query, no scaling) would make NaN of hidden scores
      if (lane == 0) row_limit[i] = first_seen + t;
      if (lane == 0) factor[i] = max_nan(top * fabsf(p.scaling) * (1.4426950408889634f / (float)D) / cent_scale, 1e-30f);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const FragSlot a = index_slot<D, BITS>(lane * E + j), c = sign_slot<D, BITS>(lane * E + j);
        const __half most = __float2half_rn(w1[j] * inv);
        __half* to = frags + (((m * Cfg::kPlanes * Cfg::kSteps + a.step) * 32 + row_lane + a.tig) * 4 + 2 * a.reg + up) * 2 + a.half;
        to[0] = most;
        if constexpr (Cfg::kSplit) to[2 * Cfg::kSteps * 32 * 8] = __float2half_rn(fmaf(w1[j], inv, -__half2float(most)));
        frags[(((m * Cfg::kPlanes * Cfg::kSteps + Cfg::kSteps + c.step) * 32 + row_lane + c.tig) * 4 + 2 * c.reg + up) * 2 + c.half] =
            __float2half_rn(w2[j] * inv);
      }
    }
  }
  __syncthreads();

  // rows gid and gid + 8 of every 16
  float m_run[MT][2], l_run[MT][2];
  float o[MT][D / 8][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m_run[m][k] = -INFINITY;
      l_run[m][k] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[m][j][r] = 0.0f;
  }
  // Column c of a tile's first or second eight is token c ^ ((c >> 1) & 1): rows of codes that are read together then lie in different
  // halves of the shared-memory banks.
  const int tok = gid ^ ((gid >> 1) & 1);              // this lane's column as B operand of the scores
  const int tok_a = 2 * tig + (tig & 1), tok_b = 2 * tig + 1 - (tig & 1);  // its two columns of the accumulators
  const uint4* frag = reinterpret_cast<const uint4*>(smem + Cfg::kRing) + lane;  // [m][Q1 steps, Q2 steps][lane]

  // Scores of the columns, in units of the rows' factors, through the online softmax; leaves the probabilities in s.
  auto softmax = [&](auto& s, auto cols) {
    constexpr int N = decltype(cols)::value;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float f_row[2] = {factor[16 * m + gid], factor[16 * m + gid + 8]};
      float top[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        top[k] = fmaxf(s[m][0][2 * k], s[m][0][2 * k + 1]);
#pragma unroll
        for (int c = 1; c < N; ++c) top[k] = fmaxf(top[k], fmaxf(s[m][c][2 * k], s[m][c][2 * k + 1]));
        top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
        top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2));
      }
      const bool moves = top[0] > m_run[m][0] && !(f_row[0] * (top[0] - m_run[m][0]) <= kMoveLimit);
      const bool moves1 = top[1] > m_run[m][1] && !(f_row[1] * (top[1] - m_run[m][1]) <= kMoveLimit);
      if (__any_sync(0xffffffffu, moves || moves1)) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float next = fmaxf(m_run[m][k], top[k]);
          const float by = next == -INFINITY ? 1.0f : exp2_approx(f_row[k] * (m_run[m][k] - next));
          m_run[m][k] = next;
          l_run[m][k] *= by;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            o[m][j][2 * k] *= by;
            o[m][j][2 * k + 1] *= by;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float base = m_run[m][k] == -INFINITY ? 0.0f : fmaf(f_row[k], m_run[m][k], -kTopLog2);
        float2 sum = make_float2(l_run[m][k], 0.0f);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const float2 x = fma_f32x2(make_float2(f_row[k], f_row[k]), make_float2(s[m][c][2 * k], s[m][c][2 * k + 1]),
                                     make_float2(-base, -base));
          const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
          s[m][c][2 * k] = e.x;
          s[m][c][2 * k + 1] = e.y;
          sum = add_f32x2(sum, e);
        }
        l_run[m][k] = sum.x + sum.y;
      }
    }
  };

  // Values are fp16 in the product, where those of a finite group may not fit.  So a column of O (a lane's column as B operand: dims of
  // one group) has its values at a power of two, which falls when one could pass 2^15.  A step that the rows' limits cut is another
  // matter: what is infinite or NaN there, or takes the power below 1, must not touch the rows that do not see it, and zero times it
  // would.  From such a tile on the values are added in 32 bits, each to the rows that give it a weight.
  constexpr float kCodes = BITS == 2 ? 4.0f : 16.0f;  // above all codes
  float lift = 1.0f;
  bool exact = false, lifted = false;  // lifted: not every column at 1, or exact
  auto lift_for = [&](float reach) {  // takes reach * kCodes to between 2^11 and 2^12
    return __uint_as_float((uint32_t)(127 + 11 + 127 - (BITS == 2 ? 2 : 4)) * (1u << 23) - (__float_as_uint(fmaxf(reach, 0x1p-100f)) & 0x7f800000u));
  };
  // A bf16 cache may hold values far below fp16's range, too: a column whose first values stay below 2^-6 (or are zero, or in a hole) begins at
  // a power above 1.  An fp16 cache's scales and zeros are multiples of 2^-24, and so are its values.
  if constexpr (!std::is_same_v<T, __half>) {
    const float a = fabsf(ElemTraits<T>::to_float(first_scale)), z = fabsf(ElemTraits<T>::to_float(first_zero));
    float reach = a < INFINITY && z < INFINITY ? fmaf(z, 1.0f / kCodes, a) : 0.0f;
    reach = fmaxf(reach, __shfl_xor_sync(0xffffffffu, reach, 1));
    reach = fmaxf(reach, __shfl_xor_sync(0xffffffffu, reach, 2));
    if (my_steps > 0 && reach < 0.015625f / kCodes) lift = lift_for(reach);
    lifted = __any_sync(0xffffffffu, lift != 1.0f) != 0;
  }
  // Steps whose scales and zeros stay below 2^14 (over the codes) look no further as long as no column is lifted: 2^14 in the type's bits,
  // each half with a bit on top that a larger magnitude, infinity and NaN take away.
  constexpr uint32_t kOne = std::is_same_v<T, __half> ? 15 << 10 : 127 << 7, kPower = std::is_same_v<T, __half> ? 1 << 10 : 1 << 7;
  constexpr uint32_t kMostZero = (0x8000u + kOne + 14 * kPower) * 0x10001u, kMostScale = (0x8000u + kOne + (BITS == 2 ? 12 : 10) * kPower) * 0x10001u;
  auto lift_columns = [&](float by) {  // the columns of O that this lane holds, by the factors of their lanes
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float of_column = __shfl_sync(0xffffffffu, by, 4 * (2 * tig + h));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[m][j][h] *= of_column;
          o[m][j][2 + h] *= of_column;
        }
    }
  };
  // Four tokens of the eight from `base` on of the tile at `at`: those that the lanes of a quad hold in their column `r`.
  auto exact_tokens = [&](auto&& weight, const uint8_t* at, int base, int r) {
    constexpr int kWidth = BITS == 2 ? 2 : 4;
#pragma unroll 1
    for (int from = 0; from < 4; ++from) {
      const int t = base + 2 * from + ((from ^ r) & 1);
      float p_of[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < 2; ++k) p_of[m][k] = __shfl_sync(0xffffffffu, weight(m, k), (lane & ~3) + from);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int column = 2 * tig + h, group = column * (D / 8) / 32;
        const float scale = ElemTraits<T>::to_float(reinterpret_cast<const T*>(at + Cfg::kOffScale)[t * Cfg::kGroups + group]);
        const float zero = ElemTraits<T>::to_float(reinterpret_cast<const T*>(at + Cfg::kOffZero)[t * Cfg::kGroups + group]);
        const uint8_t* codes = at + Cfg::kOffVal + t * Cfg::kValBytes + column * (Cfg::kValBytes / 8);
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          const float v = fmaf((float)((codes[j * kWidth / 8] >> (j * kWidth % 8)) & ((1 << kWidth) - 1)), scale, zero);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (p_of[m][k] != 0.0f) o[m][j][2 * k + h] = fmaf(p_of[m][k], v, o[m][j][2 * k + h]);
        }
      }
    }
  };

  // ---- packed prefix -----------------------------------------------------------------------------------------------------------
  for (int n = 0; n < my_steps; ++n) {
    __syncwarp();  // every lane is done with the stage that is re-armed next
    if (n + kRingStages - 1 < my_steps) issue(n + kRingStages - 1, (stage + kRingStages - 1) % kRingStages);
    if (!mbar_wait(bars + 8 * stage, phase)) {
      if (lane == 0) atomicAdd(&g_tq_multi_faults, 1);
      // wait (bounded) for the copies still in flight before the merge reuses the ring, then give this chunk up
      for (int k = 1; k < kRingStages && n + k < my_steps; ++k)
        (void)mbar_wait(bars + 8 * ((stage + k) % kRingStages), stage + k >= kRingStages ? phase ^ 1u : phase);
      dead = true;
      break;
    }
    const uint8_t* st = ring + stage * kStepTiles * Cfg::kTileStride;
    constexpr int kPieces = kStepTiles << halved;
    int valid[kPieces], total = 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      valid[i] = ring_valid[stage * kPieces + i];
      total += valid[i];
    }
    // tokens of column c, eight of a tile, that are there
    auto there = [&](int c) { return HALVED ? valid[c % kPieces] : valid[c / 2] - 8 * (c & 1); };
    if (++stage == kRingStages) { stage = 0; phase ^= 1u; }
    if (total == 0) continue;  // holes only
    const int ts = t0 + (n * kMultiMmaWarps + warp) * kStepTiles * kTile;

    // ---- scores ----
    float s[MT][kCols][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][c][r] = 0.0f;
    {
      // a lane's words of a token are loaded in two halves: the others' registers are the products' (128 dims have 128 registers a thread)
      constexpr int kHalfWords = kKeyWords > 1 ? kKeyWords / 2 : 1, kPerLoad = BITS == 4 ? kHalfWords : 2 * kHalfWords;  // nibble words
      uint32_t words[kCols][kHalfWords], flips[kCols];  // flips: the residual norm at the centroids' scale, negative, twice in fp16
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const uint8_t* at = st + c / 2 * Cfg::kTileStride;
        const int t = tok + 8 * (c & 1);
        const uint32_t r = __half_as_ushort(__float2half_rn(-cent_scale * *reinterpret_cast<const float*>(at + Cfg::kOffRnorm + 4 * t)));
        flips[c] = r | r << 16;
      }
      constexpr int kNibbleWords = D / 32;
#pragma unroll
      for (int w = 0; w < kNibbleWords; ++w) {
        if (w % kPerLoad == 0) {
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            load_words<kHalfWords>(st + c / 2 * Cfg::kTileStride + (tok + 8 * (c & 1)) * Cfg::kKeyBytes + tig * (4 * kKeyWords) +
                                       w / kPerLoad * (4 * kHalfWords), words[c]);
        }
        const int at = BITS == 4 ? w % kHalfWords : w / 2 % kHalfWords;  // the nibble word's word
        // a k-step at a time, column by column: a product runs while the next column is unpacked, and one column's products are four apart
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint4 a[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) a[m] = frag[(m * Cfg::kPlanes * Cfg::kSteps + 2 * w + i) * 32];
          uint4 rest[MT];
          if constexpr (Cfg::kSplit) {
#pragma unroll
            for (int m = 0; m < MT; ++m) rest[m] = frag[((m * Cfg::kPlanes + 2) * Cfg::kSteps + 2 * w + i) * 32];
          }
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            uint32_t sel = (BITS == 2 || BITS == 3) && (w & 1) != 0 ? words[c][at] >> (i == 0 ? 2 : 18) : i == 0 ? words[c][at] : words[c][at] >> 16;
            sel &= BITS == 4 ? 0x7777u : BITS == 3 ? 0x3333u : 0x1111u;
            const uint32_t lo = permute(lut_lo[0], lut_lo[1], sel), hi = permute(lut_hi[0], lut_hi[1], sel);
            const uint32_t k0 = permute(lo, hi, 0x5140), k1 = permute(lo, hi, 0x7362);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              mma_f16(s[m][c], a[m], k0, k1);
              if constexpr (Cfg::kSplit) mma_f16(s[m][c], rest[m], k0, k1);
            }
          }
        }
        if constexpr (BITS != 3) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint4 a[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) a[m] = frag[(m * Cfg::kPlanes * Cfg::kSteps + Cfg::kSteps + 2 * w + i) * 32];
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              uint32_t k[2];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                // the sign of nibble n is its top bit; of a 2-bit field, the upper bit of the even or the odd ones
                const int up = 12 - 4 * (2 * i + r) + (BITS == 2 && (w & 1) == 0 ? 2 : 0);
                k[r] = lop3<kAndXor>(times_power(words[c][at], up), 0x80008000u, flips[c]);
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) mma_f16(s[m][c], a[m], k[0], k[1]);
            }
          }
        }
      }
      if constexpr (BITS == 3) {
        uint32_t signs[kCols][kSignWords];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const uint8_t* bits = st + c / 2 * Cfg::kTileStride + (tok + 8 * (c & 1)) * Cfg::kKeyBytes + D / 4 + tig * (D / 32);
          if constexpr (D == 64) {
            const uint32_t both = *reinterpret_cast<const uint16_t*>(bits);
            signs[c][0] = both | both << 8;
          } else {
            load_words<kSignWords>(bits, signs[c]);
          }
        }
#pragma unroll
        for (int x = 0; x < Cfg::kSteps; ++x) {
          uint4 a[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) a[m] = frag[(m * Cfg::kPlanes * Cfg::kSteps + Cfg::kSteps + x) * 32];
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const uint32_t word = signs[c][x / 8];
            const int up = 15 - 2 * (x % 8);
            const uint32_t k0 = lop3<kAndXor>(times_power(word, up), 0x80008000u, flips[c]);
            const uint32_t k1 = lop3<kAndXor>(times_power(word, up - 1), 0x80008000u, flips[c]);
#pragma unroll
            for (int m = 0; m < MT; ++m) mma_f16(s[m][c], a[m], k0, k1);
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const float2 two = *reinterpret_cast<const float2*>(st + c / 2 * Cfg::kTileStride + Cfg::kOffNorm + 4 * (2 * tig + 8 * (c & 1)));
      const float norm[2] = {(tig & 1) ? two.y : two.x, (tig & 1) ? two.x : two.y};
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 x = mul_f32x2(make_float2(s[m][c][2 * k], s[m][c][2 * k + 1]), make_float2(norm[0], norm[1]));
          s[m][c][2 * k] = x.x;
          s[m][c][2 * k + 1] = x.y;
        }
    }
    const bool full = total == kStepTiles * kTile;
    const bool cut = ts + kStepTiles * kTile - 1 > first_seen;
    if (!full || cut) {  // tokens that are not there, or that some rows do not see
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = (r & 1) ? tok_b : tok_a;
            if (t >= there(c) || ts + 8 * c + t > row_limit[16 * m + gid + 8 * (r / 2)]) s[m][c][r] = -INFINITY;
          }
    }
    softmax(s, std::integral_constant<int, kCols>{});

    // ---- values ----
    // In two forms, so that what a column's power takes costs the ordinary one nothing (in one, 16 rows of 32768 tokens took 280 us instead of 267).
    bool careful = lifted;
    if (!careful) {  // scales and zeros of two tokens of the step a lane
      uint32_t words[Cfg::kGroups];
      load_words<Cfg::kGroups>(st + (lane >> 4) * Cfg::kTileStride + Cfg::kOffScale + (lane & 15) * (4 * Cfg::kGroups), words);
#pragma unroll
      for (int i = 1; i < Cfg::kGroups; ++i) words[0] = max_magnitudes<T>(words[0], words[i]);
      const uint32_t room = ((lane & 8) != 0 ? kMostZero : kMostScale) - (words[0] & 0x7fff7fffu);
      careful = __any_sync(0xffffffffu, (room & 0x80008000u) != 0x80008000u) != 0;
    }
    auto values = [&](auto careful_way) {
      constexpr bool kCareful = decltype(careful_way)::value;
#pragma unroll
      for (int u = 0; u < kStepTiles; ++u) {
        const uint8_t* at = st + u * Cfg::kTileStride;
        uint4 pa[MT], rest[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          pa[m] = make_uint4(pack2<__half>(s[m][2 * u][0], s[m][2 * u][1]), pack2<__half>(s[m][2 * u][2], s[m][2 * u][3]),
                             pack2<__half>(s[m][2 * u + 1][0], s[m][2 * u + 1][1]), pack2<__half>(s[m][2 * u + 1][2], s[m][2 * u + 1][3]));
          if constexpr (Cfg::kSplit) {
            const uint32_t most[4] = {pa[m].x, pa[m].y, pa[m].z, pa[m].w};
            uint32_t left[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&most[i]));
              left[i] = pack2<__half>(s[m][2 * u + i / 2][2 * (i % 2)] - x.x, s[m][2 * u + i / 2][2 * (i % 2) + 1] - x.y);
            }
            rest[m] = make_uint4(left[0], left[1], left[2], left[3]);
          }
        }
        uint32_t scale[2], zero[2], words[2][2][kValWords];
        float sc[2][2], ze[2][2];  // of tokens tok_a and tok_b, of the tile's first and second eight
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int ta = tok_a + 8 * i, tb = tok_b + 8 * i;
          const int group = gid * (D / 8) / 32;
          const T* scales = reinterpret_cast<const T*>(at + Cfg::kOffScale) + group;
          const T* zeros = reinterpret_cast<const T*>(at + Cfg::kOffZero) + group;
          sc[i][0] = ElemTraits<T>::to_float(scales[ta * Cfg::kGroups]); sc[i][1] = ElemTraits<T>::to_float(scales[tb * Cfg::kGroups]);
          ze[i][0] = ElemTraits<T>::to_float(zeros[ta * Cfg::kGroups]); ze[i][1] = ElemTraits<T>::to_float(zeros[tb * Cfg::kGroups]);
          if (!full) {  // the bytes of tokens that are not there may be anything
            if (tok_a >= there(2 * u + i)) sc[i][0] = ze[i][0] = 0.0f;
            if (tok_b >= there(2 * u + i)) sc[i][1] = ze[i][1] = 0.0f;
          }
          const uint8_t* codes = at + Cfg::kOffVal + gid * (Cfg::kValBytes / 8);
          if constexpr (BITS == 2 && D == 64) {
            words[i][0][0] = *reinterpret_cast<const uint16_t*>(codes + ta * Cfg::kValBytes);
            words[i][1][0] = *reinterpret_cast<const uint16_t*>(codes + tb * Cfg::kValBytes);
          } else {
            load_words<kValWords>(codes + ta * Cfg::kValBytes, words[i][0]);
            load_words<kValWords>(codes + tb * Cfg::kValBytes, words[i][1]);
          }
        }
        if constexpr (kCareful) {
          const float most_scale = max_nan(max_nan(fabsf(sc[0][0]), fabsf(sc[0][1])), max_nan(fabsf(sc[1][0]), fabsf(sc[1][1])));
          const float most_zero = max_nan(max_nan(fabsf(ze[0][0]), fabsf(ze[0][1])), max_nan(fabsf(ze[1][0]), fabsf(ze[1][1])));
          if (__any_sync(0xffffffffu, !exact && !(fmaf(most_zero, 1.0f / kCodes, most_scale) * lift <= 32768.0f / kCodes))) {
            float reach = 0.0f;  // the column's largest value, in codes
            bool fine = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float a = fabsf(sc[i / 2][i % 2]), z = fabsf(ze[i / 2][i % 2]);
              if (a < INFINITY && z < INFINITY) reach = fmaxf(reach, fminf(fmaf(z, 1.0f / kCodes, a), 3.0e38f));
              else fine = false;
            }
            reach = fmaxf(reach, __shfl_xor_sync(0xffffffffu, reach, 1));
            reach = fmaxf(reach, __shfl_xor_sync(0xffffffffu, reach, 2));
            float next = lift;
            if (reach * lift > 32768.0f / kCodes) next = lift_for(reach);
            exact = __any_sync(0xffffffffu, cut && (!fine || (next != lift && next < 1.0f))) != 0;
            if (exact) next = 1.0f;
            lift_columns(next / lift);
            lift = next;
            lifted = exact || __any_sync(0xffffffffu, lift != 1.0f) != 0;
          }
          if (exact) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
              for (int r = 0; r < 2; ++r) exact_tokens([&](int m, int k) { return s[m][2 * u + i][2 * k + r]; }, at, 8 * i, r);
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              sc[i][k] *= lift;
              ze[i][k] *= lift;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          scale[i] = pack2<__half>(sc[i][0], sc[i][1]);
          zero[i] = pack2<__half>(ze[i][0], ze[i][1]);
        }
        // A code in the lowest bits under the exponent of 1024 reads as 1024 + code in fp16, one a field higher under the exponent of 64
        // (2-bit codes: 256) as 64 + code, and taking that off is exact.  So one shift serves the two fields of a byte: the logic pipe,
        // which binds this kernel, has one operation per register of two values and a shift per four, instead of two.
        constexpr int kWidth = BITS == 2 ? 2 : 4, kPerWord = 32 / kWidth;
        constexpr uint32_t kField = (1u << kWidth) - 1u;
#pragma unroll
        for (int w = 0; w < kValWords; ++w)
#pragma unroll
          for (int h = 0; h < (BITS == 2 && D == 64 ? 1 : 2); ++h) {
            uint32_t x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = permute(words[i][0][w], words[i][1][w], h == 0 ? 0x5410 : 0x7632);
#pragma unroll
            for (int f = 0; f < kPerWord / 2; f += 2) {
#pragma unroll
              for (int up = 0; up < 2; ++up) {
                uint32_t v[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t mask = kField << (kWidth * up) | kField << (kWidth * up + 16);
                  const uint32_t base = up == 0 ? 0x64006400u : BITS == 2 ? 0x5C005C00u : 0x54005400u;
                  v[i] = sub_f16x2(lop3<kAndOr>(x[i], mask, base), base);
                  v[i] = fma_f16x2(v[i], scale[i], zero[i]);
                }
                const int j = w * kPerWord + h * (kPerWord / 2) + f + up;
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                  mma_f16(o[m][j], pa[m], v[0], v[1]);
                  if constexpr (Cfg::kSplit) mma_f16(o[m][j], rest[m], v[0], v[1]);
                }
              }
#pragma unroll
              for (int i = 0; i < 2; ++i) x[i] >>= 2 * kWidth;
            }
          }
      }
    };
    if (careful) values(std::true_type{});
    else values(std::false_type{});
  }

  if (lifted) lift_columns(1.0f / lift);

  // ---- un-quantized window ring ------------------------------------------------------------------------------------------------
  const int w0 = max(t0, lq);
  for (int ts = w0 + warp * kTile; ts < t1; ts += kMultiMmaWarps * kTile) {
    const int valid = min(kTile, t1 - ts);
    const int R = p.residual_len;
    const T* keys = reinterpret_cast<const T*>(p.window) + (p.window_slots[b] * 2 * p.kv_heads + kvh) * R * D;
    const T* values = keys + (int64_t)p.kv_heads * R * D;
    auto ring_row = [&](int t) { return (int64_t)((ts + min(t, valid - 1)) % R) * D; };
    float s[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][c][r] = 0.0f;
    {
      const T* k0 = keys + ring_row(tok) + tig * (D / 4);
      const T* k1 = keys + ring_row(tok + 8) + tig * (D / 4);
      const T* q[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row = row0 + min(16 * m + gid + 8 * k, count - 1);
          const int t = multi_token_of(p, row);
          q[m][k] = reinterpret_cast<const T*>(p.q) + (int64_t)b * p.q_stride_b + (int64_t)(kvh * p.groups + row - t * p.groups) * p.q_stride_h +
                    (int64_t)t * p.q_stride_t + tig * (D / 4);
        }
      // 8 coordinates of this lane are two k-steps
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        const uint4 ka = *reinterpret_cast<const uint4*>(k0 + 8 * x), kb = *reinterpret_cast<const uint4*>(k1 + 8 * x);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 lo = *reinterpret_cast<const uint4*>(q[m][0] + 8 * x), hi = *reinterpret_cast<const uint4*>(q[m][1] + 8 * x);
          const uint4 a0 = make_uint4(lo.x, hi.x, lo.y, hi.y), a1 = make_uint4(lo.z, hi.z, lo.w, hi.w);
          mma_elem<T>(s[m][0], a0, ka.x, ka.y);
          mma_elem<T>(s[m][0], a1, ka.z, ka.w);
          mma_elem<T>(s[m][1], a0, kb.x, kb.y);
          mma_elem<T>(s[m][1], a1, kb.z, kb.w);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int in_tile = 8 * c + ((r & 1) ? tok_b : tok_a);
          // to the units of the row's factor
          const float x = s[m][c][r] * (p.scaling * 1.4426950408889634f / factor[16 * m + gid + 8 * (r / 2)]);
          s[m][c][r] = in_tile >= valid || ts + in_tile > row_limit[16 * m + gid + 8 * (r / 2)] ? -INFINITY : x;
        }
    softmax(s, std::integral_constant<int, 2>{});
    // probabilities as a sum of two of the type, so that they keep 16 bits and more
    uint4 pa[MT], pb[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t* hi = &pa[m].x;
      uint32_t* lo = &pb[m].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[m][i / 2][2 * (i % 2)], y = s[m][i / 2][2 * (i % 2) + 1];
        hi[i] = pack2<T>(x, y);
        if constexpr (std::is_same_v<T, __half>) {
          const float2 most = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
          lo[i] = pack2<T>(x - most.x, y - most.y);
        } else {
          lo[i] = pack2<T>(x - __uint_as_float(hi[i] << 16), y - __uint_as_float(hi[i] & 0xffff0000u));
        }
      }
    }
    const T* v[4] = {values + ring_row(tok_a) + gid * (D / 8), values + ring_row(tok_b) + gid * (D / 8),
                     values + ring_row(tok_a + 8) + gid * (D / 8), values + ring_row(tok_b + 8) + gid * (D / 8)};
    const bool cut = ts + kTile - 1 > first_seen;
    const bool there[4] = {tok_a < valid, tok_b < valid, tok_a + 8 < valid, tok_b + 8 < valid};
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
      uint32_t w[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 got = there[i] ? *reinterpret_cast<const uint4*>(v[i] + 8 * x) : make_uint4(0u, 0u, 0u, 0u);
        w[i][0] = got.x; w[i][1] = got.y; w[i][2] = got.z; w[i][3] = got.w;
      }
      if (cut) {
        uint32_t all = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t fine = finite_halves<T>(w[i][k]);
            w[i][k] &= fine;
            all &= fine;
          }
        if (all != 0xffffffffu) *strange = 1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v0 = permute(w[0][i / 2], w[1][i / 2], i % 2 == 0 ? 0x5410 : 0x7632);
        const uint32_t v1 = permute(w[2][i / 2], w[3][i / 2], i % 2 == 0 ? 0x5410 : 0x7632);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma_elem<T>(o[m][8 * x + i], pa[m], v0, v1);
          mma_elem<T>(o[m][8 * x + i], pb[m], v0, v1);
        }
      }
    }
  }

  // Adds the infinite and NaN values of the window that its products left out, at the row's dims d .. d + 3.
  auto strange_values = [&](int row, int d, float4& sum) {
    const int seen = min(t1 - 1, first_seen + multi_token_of(p, row)), w0 = max(t0, lq);
    for (int t = max(w0, first_seen - kTile); t <= seen; ++t) {
      if (w0 + (t - w0) / kTile * kTile + kTile - 1 <= first_seen) continue;  // of a tile that was not cut
      const T* value = reinterpret_cast<const T*>(p.window) +
                       (((p.window_slots[b] * 2 + 1) * p.kv_heads + kvh) * p.residual_len + t % p.residual_len) * D + d;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = ElemTraits<T>::to_float(value[i]);
        if (isfinite(v[i])) v[i] = 0.0f;  // is in the product
      }
      sum.x += v[0]; sum.y += v[1]; sum.z += v[2]; sum.w += v[3];
    }
  };

  // ---- the warps' rows together ---------------------------------------------------------------------------------------------
  float2* stats = reinterpret_cast<float2*>(smem + Cfg::kOffStats);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      l_run[m][k] += __shfl_xor_sync(0xffffffffu, l_run[m][k], 1);
      l_run[m][k] += __shfl_xor_sync(0xffffffffu, l_run[m][k], 2);
      if (tig == 0) stats[warp * Cfg::kRows + 16 * m + gid + 8 * k] = make_float2(m_run[m][k], l_run[m][k]);
    }
  __syncthreads();  // and nobody reads the ring or the queries any more
  // a thread per row: what each warp's sums count, in place of its maximum; the row's 1 / denominator, or 1 where the partials of
  // several CTAs are merged, in place of its factor
  if (threadIdx.x < Cfg::kRows) {
    const int i = threadIdx.x;
    const float f = factor[i];
    float top = -INFINITY, den = 0.0f;
#pragma unroll
    for (int w = 0; w < kMultiMmaWarps; ++w) top = fmaxf(top, stats[w * Cfg::kRows + i].x);
#pragma unroll
    for (int w = 0; w < kMultiMmaWarps; ++w) {
      const float2 x = stats[w * Cfg::kRows + i];
      // a warp without a key for the row has no sums; where none has, a NaN may be in them
      const float by = top == -INFINITY ? 1.0f : x.x == -INFINITY ? 0.0f : exp2_approx(f * (x.x - top));
      stats[w * Cfg::kRows + i].x = by;
      den = fmaf(x.y, by, den);
    }
    const bool alone = part.count == 1;
    // a NaN among the scores has to stay one, so only a row without a key is zero
    factor[i] = alone ? (den == 0.0f ? 0.0f : 1.0f / den) : 1.0f;
    if (!alone && i < count)
      reinterpret_cast<float2*>(p.stats)[multi_partial_row(part, part.mine, Cfg::kRows) + i] =
          make_float2(top * f * 0.6931471805599453f, den);  // natural units
  }
  __syncthreads();
  float* merged = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float by = stats[warp * Cfg::kRows + 16 * m + gid + 8 * k].x;
      float* to = merged + (warp * 16 + gid + 8 * k) * Cfg::kMergeStride;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < D / 8; j += 4) {
          const int d = (2 * tig + h) * (D / 8) + j;
          *reinterpret_cast<float4*>(to + d + 8 * (d / 32)) =
              make_float4(o[m][j][2 * k + h] * by, o[m][j + 1][2 * k + h] * by, o[m][j + 2][2 * k + h] * by, o[m][j + 3][2 * k + h] * by);
        }
    }
    __syncthreads();
    const int rows = min(16, count - 16 * m);
    for (int item = threadIdx.x; item < rows * (D / 4); item += kMultiMmaThreads) {
      const int i = item / (D / 4), d = 4 * (item % (D / 4));
      const float* from = merged + i * Cfg::kMergeStride + d + 8 * (d / 32);
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kMultiMmaWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(from + w * 16 * Cfg::kMergeStride);
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
      const int row = row0 + 16 * m + i;
      if (*strange != 0) strange_values(row, d, sum);
      if (part.count == 1) {
        const float inv = factor[16 * m + i];
        const float out[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
        multi_store<T, 4>(p, b, kvh, row, d, out);
      } else {
        *reinterpret_cast<float4*>(p.values + (multi_partial_row(part, part.mine, Cfg::kRows) + 16 * m + i) * D + d) = sum;
      }
    }
    __syncthreads();
  }
  if (part.count > 1) multi_merge<T, D, kMultiMmaWarps, Cfg::kRows>(p, b, kvh, tile, row_tiles, count, part, merged);
  // the next segment's copies land where the merge and the queries were
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  __syncthreads();
  });
}

template <typename T, int D, int BITS, int MT, bool HALVED>
static int launch(const TqMultiParams& p, cudaStream_t stream) {
  using Cfg = MultiCfg<T, D, BITS, MT>;
  static_assert(148 * Cfg::kCtas <= kMultiMaxCtas && Cfg::kCtas * Cfg::kRows <= 2 * kMultiScratchRows, "partials of more rows than there is room for");
  const int row_tiles = (p.rows + Cfg::kRows - 1) / Cfg::kRows;
  auto kernel = tq_multi_mma_kernel<T, D, BITS, MT, HALVED>;
  ANNA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
  kernel<<<multi_ctas(p, row_tiles, Cfg::kCtas), kMultiMmaThreads, Cfg::kSmem, stream>>>(p, row_tiles);
  return check_launch("tq_multi_mma_kernel");
}

template <bool HALVED>
static int launch_pages_of(const TqMultiParams& p, int head_dim, int bits, int dtype, cudaStream_t stream) {
  auto pick = [&](auto elem) -> int {
    using T = decltype(elem);
    return ANNA_DISPATCH_TQ_BITS(bits, BITS, [&]() -> int {
      if (head_dim == 64) return p.rows > 16 ? launch<T, 64, BITS, 2, HALVED>(p, stream) : launch<T, 64, BITS, 1, HALVED>(p, stream);
      if (head_dim == 128) return p.rows > 16 ? launch<T, 128, BITS, 2, HALVED>(p, stream) : launch<T, 128, BITS, 1, HALVED>(p, stream);
      return launch<T, 256, BITS, 1, HALVED>(p, stream);
    });
  };
  return dtype == ANNA_DTYPE_F16 ? pick(__half{}) : pick(__nv_bfloat16{});
}

static int multi_mma_faults(int* count) {
  int32_t value = 0;
  ANNA_CUDA_CHECK(cudaMemcpyFromSymbol(&value, g_tq_multi_faults, sizeof(value)));
  *count = value;
  return ANNA_OK;
}

}  // namespace anna
