// Append to the 8-bit paged cache, and its dense view.
//
// Append: a warp takes the keys or the values of one page of one KV head.  It reads the page's tokens (from the ring those in front of
// the new ones), keeps the largest and the smallest value of every dim, from which the page's largest magnitude follows, and writes
// the codes; the bounds of the keys are the codes of those extremes, as rounding keeps the order.  The warp of a row's first page then
// writes the tokens of the unfinished page to the ring: it has read the ring before, and no other warp reads it.
//
// Bound: HBM; every token is read once, 2 D e bytes, and written once, 2 D.
//
// A code is the whole number next to 127 x / m, ties to even, of the quotient itself: x and m have at most 11 significant bits (fp16),
// so 254 x - (odd) m, unless zero, is at least 2^-19 of the quotient's power of two away from a tie, while x * fl(127 / m) is off by
// 2^-22.4 of it at most.  Rounded to 21 bits (Veltkamp's splitting: c = 9 q, c - (c - q)) a tie is one again, and all else stays on its
// side.  fp32 values take the same steps in 64 bits (24 significant bits, rounded to 41).
#include "q8_common.cuh"
#include "tq_bulk.cuh"

#include <type_traits>

namespace anna {

struct Q8AppendParams {
  const void* in[2];  // keys, values
  int64_t stride_b[2], stride_h[2], stride_t[2];
  uint8_t* pages;
  const int32_t* page_table;
  int64_t table_stride;
  void* window;
  const int64_t* window_slots;
  const int64_t* past_lengths;
  int64_t* new_lengths;
  int batch, kv_heads, tokens, block_size, units;
  int page_bytes;
  int64_t num_pages, max_blocks, num_slots;
  int32_t* status;
};

constexpr int kQ8AppendWarps = 4;
constexpr int64_t kQ8MaxLength = 1ll << 30;  // of a row, a table, and a call's tokens

// The larger and the smaller of the values in a word, one or two; a NaN stays one.
template <typename T>
__device__ __forceinline__ uint32_t q8_larger(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, float>) asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else if constexpr (std::is_same_v<T, __half>) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t q8_smaller(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, float>) asm("min.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else if constexpr (std::is_same_v<T, __half>) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Running extremes of a lane's dims, 16 bytes each, in the cache's type.
template <typename T>
struct Q8Extremes {
  uint4 high, low;
  __device__ __forceinline__ void start() {
    constexpr uint32_t kInf = std::is_same_v<T, float> ? 0x7f800000u : std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t kSigns = std::is_same_v<T, float> ? 0x80000000u : 0x80008000u;
    low = make_uint4(kInf, kInf, kInf, kInf);
    high = make_uint4(kInf | kSigns, kInf | kSigns, kInf | kSigns, kInf | kSigns);
  }
  __device__ __forceinline__ void take(const uint4& h, const uint4& l) {
    high = make_uint4(q8_larger<T>(high.x, h.x), q8_larger<T>(high.y, h.y), q8_larger<T>(high.z, h.z), q8_larger<T>(high.w, h.w));
    low = make_uint4(q8_smaller<T>(low.x, l.x), q8_smaller<T>(low.y, l.y), q8_smaller<T>(low.z, l.z), q8_smaller<T>(low.w, l.w));
  }
  __device__ __forceinline__ void exchange(int mask) {
    auto other = [&](uint32_t x) { return __shfl_xor_sync(0xffffffffu, x, mask); };
    const uint4 h = make_uint4(other(high.x), other(high.y), other(high.z), other(high.w));
    take(h, make_uint4(other(low.x), other(low.y), other(low.z), other(low.w)));
  }
  // the largest magnitude, of one dim or of two
  __device__ __forceinline__ uint32_t magnitude() const {
    constexpr uint32_t kValue = std::is_same_v<T, float> ? 0x7fffffffu : 0x7fff7fffu;
    auto larger = [](uint32_t a, uint32_t b) { return q8_larger<T>(a & kValue, b & kValue); };
    return larger(larger(larger(high.x, low.x), larger(high.y, low.y)), larger(larger(high.z, low.z), larger(high.w, low.w)));
  }
};

// Turns 16 bytes of values into codes (see above), of which the lowest byte is looked at.  Two at a time, as the GPU has packed products; 9 q is
// 8 q + q, and a packed product with a sum behind it, which may be contracted, is one of the first step alone, where that rounds once less.  Tiny pages are
// lifted, so that 127 / m is finite.
template <typename T>
struct Q8Coder {
  float lift, rate;
  __device__ __forceinline__ explicit Q8Coder(float top) {
    lift = top < 8.6736174e-19f ? 1.2676506e30f : 1.0f;  // 2^-60, 2^100
    rate = __fdiv_rn(127.0f, top * lift);
  }
  __device__ __forceinline__ void codes(const uint4& raw, float sign, int (&code)[8]) const {
    float x[8];
    widen16<T>(raw, x);
    if (lift != 1.0f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= lift;
    }
    const uint64_t rates = pair_of(sign * rate, sign * rate), eight = pair_of(8.0f, 8.0f), minus = pair_of(-1.0f, -1.0f);
    const uint64_t to_whole = pair_of(12582912.0f, 12582912.0f);  // 1.5 * 2^23
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t q = mul_pair(pair_of(x[i], x[i + 1]), rates), c = fma_pair(q, eight, q);
      const uint64_t tie = add_pair(c, fma_pair(c, minus, q));
      float a, b;
      halves_of(add_pair(tie, to_whole), a, b);
      code[i] = __float_as_int(a);
      code[i + 1] = __float_as_int(b);
    }
  }
};
template <>
struct Q8Coder<float> {
  double rate;
  __device__ __forceinline__ explicit Q8Coder(float top) { rate = 127.0 / (double)top; }
  __device__ __forceinline__ void codes(const uint4& raw, float sign, int (&code)[4]) const {
    float x[4];
    widen16<float>(raw, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double q = __dmul_rn((double)(sign * x[i]), rate), c = __dmul_rn(q, 4097.0);
      code[i] = (int)rint(__dsub_rn(c, __dsub_rn(c, q)));
    }
  }
};

template <int N>
__device__ __forceinline__ void q8_store_codes(uint8_t* to, const int (&code)[N]) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint32_t lo = __byte_perm(code[4 * i], code[4 * i + 1], 0x0040), hi = __byte_perm(code[4 * i + 2], code[4 * i + 3], 0x0040);
    w[i] = __byte_perm(lo, hi, 0x5410);
  }
  if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(to) = w[0];
}

// PER warps, one or all of the CTA, to an item.
template <typename T, int D, int PER>
__global__ void __launch_bounds__(kQ8AppendWarps * 32) q8_append_kernel(const Q8AppendParams p) {
  static_assert(PER == 1 || PER == kQ8AppendWarps, "a warp or a CTA");
  constexpr int kN = ElemTraits<T>::kVec;
  constexpr int kVecs = D / kN;                               // of a token
  constexpr int kLanes = kVecs < 32 ? kVecs : 32;              // that share a token
  constexpr int kCols = kVecs / kLanes;                        // vectors of a lane and token
  constexpr int kAtOnce = PER * (32 / kLanes);                 // tokens of the item's warps
  constexpr int kHeld = (PER == 1 ? 8 : 16) / kCols;           // rounds whose values stay in registers
  __shared__ uint4 s_extremes[PER == 1 ? 1 : 2 * PER * kVecs];
  q8_wait_for_previous();
  const int lane = threadIdx.x & 31, part = PER == 1 ? 0 : threadIdx.x >> 5;
  const uint32_t item = PER == 1 ? blockIdx.x * kQ8AppendWarps + (threadIdx.x >> 5) : blockIdx.x;
  const int which = (int)(item & 1u);  // keys, values
  uint32_t rest = item >> 1;
  const int unit = (int)(rest % (uint32_t)p.units);
  rest /= (uint32_t)p.units;
  const int h = (int)(rest % (uint32_t)p.kv_heads);
  const int64_t b = rest / (uint32_t)p.kv_heads;
  if (b >= p.batch) return;
  const int S = p.block_size;
  const int64_t past_length = p.past_lengths[b];
  if (p.new_lengths != nullptr && unit == 0 && h == 0 && which == 0 && lane == 0 && part == 0) p.new_lengths[b] = past_length + p.tokens;
  if (past_length < 0) return;
  if (past_length >= kQ8MaxLength - p.tokens) {  // behind any table
    if (p.status != nullptr && unit == 0 && lane == 0) atomicOr(p.status, (int)ANNA_DEV_BAD_PAGE);
    return;
  }
  const int past = (int)past_length, total = past + p.tokens, block = past / S + unit;
  const T* fresh = reinterpret_cast<const T*>(p.in[which]) + b * p.stride_b[which] + h * p.stride_h[which];
  const int64_t step = p.stride_t[which];
  const int64_t slot = unit == 0 ? p.window_slots[b] : -1;
  T* ring = slot >= 0 && slot < p.num_slots ? reinterpret_cast<T*>(p.window) + ((slot * 2 + which) * p.kv_heads + h) * S * D : nullptr;
  const int begin = block * S;  // position of the page's first token
  const int col = lane % kLanes * kN, row = part * (32 / kLanes) + lane / kLanes;

  const bool closes = begin + S <= total;
  int32_t pid = -1;
  if (closes && block < p.max_blocks) pid = p.page_table[b * p.table_stride + block];
  const bool there = pid >= 0 && pid < p.num_pages;
  const bool needs_ring = unit == 0 && (past % S != 0 || total % S != 0);
  if (p.status != nullptr && lane == 0 && part == 0 && ((closes && !there) || (needs_ring && ring == nullptr)))
    atomicOr(p.status, (int)ANNA_DEV_BAD_PAGE);
  if (closes && there && (begin >= past || ring != nullptr)) {
    uint8_t* page = p.pages + ((int64_t)pid * p.kv_heads + h) * p.page_bytes;
    uint8_t* codes = page + which * S * D;
    auto source = [&](int token) {
      const int at = begin + token;
      return at < past ? ring + token * D : fresh + (at - past) * step;
    };
    const int rounds = (S + kAtOnce - 1) / kAtOnce;
    Q8Extremes<T> seen[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) seen[c].start();
    // a token past the page's end counts as its last one again
    auto finish = [&](auto&& each) {
#pragma unroll
      for (int mask = kLanes; mask < 32; mask *= 2)
#pragma unroll
        for (int c = 0; c < kCols; ++c) seen[c].exchange(mask);
      if constexpr (PER > 1) {
        uint4* mine = s_extremes + part * 2 * kVecs + lane;
        if (lane < kLanes) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            mine[c * 32] = seen[c].high;
            mine[kVecs + c * 32] = seen[c].low;
          }
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < PER; ++w)
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const uint4* theirs = s_extremes + w * 2 * kVecs + lane % kLanes + c * 32;
            seen[c].take(theirs[0], theirs[kVecs]);
          }
      }
      uint32_t word = seen[0].magnitude();
#pragma unroll
      for (int c = 1; c < kCols; ++c) word = q8_larger<T>(word, seen[c].magnitude());
#pragma unroll
      for (int mask = 1; mask < kLanes; mask *= 2) word = q8_larger<T>(word, __shfl_xor_sync(0xffffffffu, word, mask));
      float pair[kN];
      widen16<T>(make_uint4(word, word, word, word), pair);
      const float top = __uint_as_float(q8_larger<float>(__float_as_uint(pair[0]), __float_as_uint(pair[1])));
      const bool fine = top < INFINITY;  // neither an infinity nor a NaN
      const bool some = fine && top > 0.0f;
      if (lane == 0 && part == 0)
        reinterpret_cast<float*>(page + q8_scale_offset(D, S))[which] = fine ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fc00000);
      const Q8Coder<T> coder(some ? top : 1.0f);
      auto put = [&](const uint4& raw, float sign, uint8_t* to) {
        int code[kN] = {};
        if (some) coder.codes(raw, sign, code);
        q8_store_codes<kN>(to, code);
      };
      each([&](const uint4& v, int token, int c) {
        if (token < S) put(v, 1.0f, codes + token * D + c * 32 * kN + col);
      });
      if (which == 0 && row == 0) {
        uint8_t* bounds = page + q8_bounds_offset(D, S);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          put(seen[c].high, 1.0f, bounds + c * 32 * kN + col);
          put(seen[c].low, -1.0f, bounds + D + c * 32 * kN + col);
        }
      }
    };
    if (rounds <= kHeld) {
      uint4 held[kHeld][kCols];
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
        if (r < rounds) {
          const T* from = source(min(r * kAtOnce + row, S - 1));
#pragma unroll
          for (int c = 0; c < kCols; ++c) held[r][c] = *reinterpret_cast<const uint4*>(from + c * 32 * kN + col);
        }
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
        if (r < rounds) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) seen[c].take(held[r][c], held[r][c]);
        }
      finish([&](auto&& one) {
#pragma unroll
        for (int r = 0; r < kHeld; ++r)
          if (r < rounds) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) one(held[r][c], r * kAtOnce + row, c);
          }
      });
    } else {  // pages of more than the registers hold are read twice, the second time from L1 or L2
      auto walk = [&](auto&& one) {
#pragma unroll 8
        for (int r = 0; r < rounds; ++r) {
          const int token = r * kAtOnce + row;
          const T* from = source(min(token, S - 1));
#pragma unroll
          for (int c = 0; c < kCols; ++c) one(*reinterpret_cast<const uint4*>(from + c * 32 * kN + col), token, c);
        }
      };
      walk([&](const uint4& v, int, int c) { seen[c].take(v, v); });
      finish(walk);
    }
  }
  if (unit != 0 || ring == nullptr) return;
  if constexpr (PER == 1) __syncwarp();  // the ring has been read
  else __syncthreads();
  const int open = total / S * S;  // first position of the unfinished page
  for (int at = max(past, open) + row; at < total; at += kAtOnce)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      *reinterpret_cast<uint4*>(ring + (at - open) * D + c * 32 * kN + col) =
          *reinterpret_cast<const uint4*>(fresh + (at - past) * step + c * 32 * kN + col);
}

struct Q8GatherParams {
  const uint8_t* pages;
  const int32_t* page_table;
  int64_t table_stride;
  const void* window;
  const int64_t* window_slots;
  const int64_t* lengths;
  void* out[2];
  int64_t stride_b, stride_h, stride_t;
  int batch, kv_heads, block_size, page_bytes;
  int shares;  // of a block
  int spans;   // blocks
  int64_t num_pages, max_blocks, num_slots, max_len;
};
constexpr int kQ8GatherPieces = 128;  // of 16 codes, of a warp

// Dense view: a warp writes 2048 keys' or values' dims of one block of one KV head; a lane de-quantizes 16 codes, which is 32 bytes of a
// 16-bit cache, at a time.  Bound: HBM, of which the output is two thirds.
template <typename T, int D>
__global__ void __launch_bounds__(128) q8_gather_kernel(const Q8GatherParams p) {
  constexpr int kN = ElemTraits<T>::kVec;
  constexpr int kPieces = D / 16;  // of a token
  q8_wait_for_previous();
  const int lane = threadIdx.x & 31;
  const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int which = (int)(item & 1u);
  uint32_t rest = item >> 1;
  const int share = (int)(rest % (uint32_t)p.shares);
  rest /= (uint32_t)p.shares;
  const int block = (int)(rest % (uint32_t)p.spans);
  rest /= (uint32_t)p.spans;
  const int h = (int)(rest % (uint32_t)p.kv_heads);
  const int64_t b = rest / (uint32_t)p.kv_heads;
  if (b >= p.batch) return;
  const int S = p.block_size;
  const int64_t length = p.lengths[b];
  const int len = (int)max((int64_t)0, min(length, p.max_len)), begin = block * S;
  const bool full = begin + S <= length;
  const uint8_t* codes = nullptr;
  const T* ring = nullptr;
  float scale = 0.0f;
  if (full) {
    const int32_t pid = block < p.max_blocks ? p.page_table[b * p.table_stride + block] : -1;
    if (pid >= 0 && pid < p.num_pages) {
      const uint8_t* page = p.pages + ((int64_t)pid * p.kv_heads + h) * p.page_bytes;
      codes = page + which * S * D;
      scale = reinterpret_cast<const float*>(page + q8_scale_offset(D, S))[which];
    }
  } else if (begin < len) {
    const int64_t slot = p.window_slots[b];
    if (slot >= 0 && slot < p.num_slots) ring = reinterpret_cast<const T*>(p.window) + ((slot * 2 + which) * p.kv_heads + h) * S * D;
  }
  T* out = reinterpret_cast<T*>(p.out[which]) + b * p.stride_b + h * p.stride_h;
  const int pieces = min(S, (int)p.max_len - begin) * kPieces;
  const int end = min(pieces, (share + 1) * kQ8GatherPieces);
#pragma unroll
  for (int round = 0; round < kQ8GatherPieces / 32; ++round) {
    const int i = share * kQ8GatherPieces + round * 32 + lane;
    if (i >= end) break;
    const int token = i / kPieces, d = i % kPieces * 16;
    uint4 x[16 / kN];
    if (codes != nullptr) {
      const uint4 c = *reinterpret_cast<const uint4*>(codes + token * D + d);
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
      T v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = ElemTraits<T>::from_float(scale * (float)(int8_t)(w[j / 4] >> (8 * (j % 4))));
#pragma unroll
      for (int j = 0; j < 16 / kN; ++j) x[j] = *reinterpret_cast<const uint4*>(v + j * kN);
    } else {
#pragma unroll
      for (int j = 0; j < 16 / kN; ++j)
        x[j] = ring != nullptr && begin + token < len ? *reinterpret_cast<const uint4*>(ring + token * D + d + j * kN) : make_uint4(0u, 0u, 0u, 0u);
    }
    T* to = out + (int64_t)(begin + token) * p.stride_t + d;
#pragma unroll
    for (int j = 0; j < 16 / kN; ++j) *reinterpret_cast<uint4*>(to + j * kN) = x[j];
  }
}

}  // namespace anna

using namespace anna;

extern "C" int anna_q8_page_bytes(int head_dim, int block_size, int64_t* bytes) {
  const char* what = "anna_q8_page_bytes";
  ANNA_REQUIRE(bytes != nullptr, "%s: null pointer argument", what);
  if (!q8_head_dim(head_dim)) return set_error(ANNA_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %d", what, head_dim);
  ANNA_REQUIRE(block_size > 0 && block_size <= kQ8MaxBlockSize, "%s: block_size must be in [1, %d], got %d", what, kQ8MaxBlockSize, block_size);
  *bytes = q8_page_bytes(head_dim, block_size);
  return ANNA_OK;
}

extern "C" int anna_q8_append(const void* k_new, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t, const void* v_new,
                              int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, uint8_t* pages, const int32_t* page_table,
                              int64_t table_stride, void* window, const int64_t* window_slots, const int64_t* past_lengths,
                              int64_t* new_lengths, int batch, int kv_heads, int new_tokens, int head_dim, int block_size,
                              int64_t num_pages, int64_t max_blocks, int64_t num_slots, int dtype, int32_t* status, anna_stream_t stream) {
  const char* what = "anna_q8_append";
  int64_t bytes = 0;
  if (const int rc = anna_q8_page_bytes(head_dim, block_size, &bytes)) return rc;
  ANNA_REQUIRE(batch >= 0 && kv_heads > 0 && new_tokens > 0 && max_blocks >= 0 && num_pages >= 0 && num_slots >= 0, "%s: bad sizes", what);
  if (batch == 0) return ANNA_OK;
  ANNA_REQUIRE(k_new && v_new && window && window_slots && past_lengths, "%s: null pointer argument", what);
  ANNA_REQUIRE(new_lengths != past_lengths, "%s: new_lengths must not be past_lengths", what);
  ANNA_REQUIRE(max_blocks == 0 || (pages && page_table), "%s: a block table needs pages", what);
  ANNA_REQUIRE(dtype == ANNA_DTYPE_F32 || dtype == ANNA_DTYPE_F16 || dtype == ANNA_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  const int vec = 16 / dtype_bytes_of(dtype);
  ANNA_REQUIRE(aligned_to(k_new, 16) && aligned_to(v_new, 16) && aligned_to(window, 16) && aligned_to(pages, 16),
               "%s: keys, values, pages and window must be 16-byte aligned", what);
  ANNA_REQUIRE((batch == 1 || (k_stride_b % vec == 0 && v_stride_b % vec == 0)) && (kv_heads == 1 || (k_stride_h % vec == 0 && v_stride_h % vec == 0)) &&
               (new_tokens <= 1 || (k_stride_t % vec == 0 && v_stride_t % vec == 0)), "%s: strides must be multiples of 16 bytes", what);
  Q8AppendParams p{};
  p.in[0] = k_new; p.in[1] = v_new;
  // the stride of a dim of one entry may be anything
  p.stride_b[0] = batch > 1 ? k_stride_b : 0; p.stride_b[1] = batch > 1 ? v_stride_b : 0;
  p.stride_h[0] = kv_heads > 1 ? k_stride_h : 0; p.stride_h[1] = kv_heads > 1 ? v_stride_h : 0;
  p.stride_t[0] = new_tokens > 1 ? k_stride_t : 0; p.stride_t[1] = new_tokens > 1 ? v_stride_t : 0;
  p.pages = pages; p.page_table = page_table; p.table_stride = table_stride;
  p.window = window; p.window_slots = window_slots; p.past_lengths = past_lengths; p.new_lengths = new_lengths;
  p.batch = batch; p.kv_heads = kv_heads; p.tokens = new_tokens; p.block_size = block_size;
  p.units = (int)(((int64_t)new_tokens + block_size - 2) / block_size) + 1;
  p.page_bytes = (int)bytes; p.num_pages = num_pages; p.max_blocks = max_blocks; p.num_slots = num_slots; p.status = status;
  // A CTA to an item where a warp would have more than 8 vectors a lane, or where the GPU has room for that: 512 tokens of 256 dims in pages of 32
  // take 4.5 us so, 7.8 with a warp to an item, 3001 such tokens 6.6 and 12.6, one token of 8 KV heads that fills its page 3.5 and 3.7.  A warp otherwise: 8 rows
  // of 2048 tokens of 128 dims in pages of 16 take 16.4 us so, 45.7 with CTAs.
  const int64_t items = (int64_t)batch * kv_heads * p.units * 2;
  ANNA_REQUIRE(new_tokens < kQ8MaxLength && max_blocks < kQ8MaxLength / block_size && items < (1ll << 31), "%s: too many tokens", what);
  const bool whole = block_size * head_dim / vec > 256 || items <= 148 * 8;
  const int64_t ctas = whole ? items : (items + kQ8AppendWarps - 1) / kQ8AppendWarps;
  return ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
      return q8_launch("q8_append_kernel", whole ? q8_append_kernel<T, D, kQ8AppendWarps> : q8_append_kernel<T, D, 1>, dim3((unsigned)ctas),
                       kQ8AppendWarps * 32, 0, (cudaStream_t)stream, p);
    });
  });
}

extern "C" int anna_q8_gather(const uint8_t* pages, const int32_t* page_table, int64_t table_stride, const void* window,
                              const int64_t* window_slots, const int64_t* lengths, void* key_out, void* value_out, int64_t out_stride_b,
                              int64_t out_stride_h, int64_t out_stride_t, int batch, int kv_heads, int head_dim, int block_size,
                              int64_t num_pages, int64_t max_blocks, int64_t num_slots, int64_t max_len, int dtype, anna_stream_t stream) {
  const char* what = "anna_q8_gather";
  int64_t bytes = 0;
  if (const int rc = anna_q8_page_bytes(head_dim, block_size, &bytes)) return rc;
  ANNA_REQUIRE(batch >= 0 && kv_heads > 0 && max_len >= 0 && max_blocks >= 0 && num_pages >= 0 && num_slots >= 0, "%s: bad sizes", what);
  if (batch == 0 || max_len == 0) return ANNA_OK;
  ANNA_REQUIRE(window && window_slots && lengths && key_out && value_out, "%s: null pointer argument", what);
  ANNA_REQUIRE(max_blocks == 0 || (pages && page_table), "%s: a block table needs pages", what);
  ANNA_REQUIRE(dtype == ANNA_DTYPE_F32 || dtype == ANNA_DTYPE_F16 || dtype == ANNA_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  const int vec = 16 / dtype_bytes_of(dtype);
  ANNA_REQUIRE(aligned_to(key_out, 16) && aligned_to(value_out, 16) && aligned_to(window, 16) && aligned_to(pages, 16),
               "%s: outputs, pages and window must be 16-byte aligned", what);
  ANNA_REQUIRE(out_stride_b % vec == 0 && out_stride_h % vec == 0 && out_stride_t % vec == 0, "%s: strides must be multiples of 16 bytes", what);
  Q8GatherParams p{};
  p.pages = pages; p.page_table = page_table; p.table_stride = table_stride;
  p.window = window; p.window_slots = window_slots; p.lengths = lengths;
  p.out[0] = key_out; p.out[1] = value_out;
  p.stride_b = out_stride_b; p.stride_h = out_stride_h; p.stride_t = out_stride_t;
  p.batch = batch; p.kv_heads = kv_heads; p.block_size = block_size; p.page_bytes = (int)bytes;
  p.num_pages = num_pages; p.max_blocks = max_blocks; p.num_slots = num_slots; p.max_len = max_len;
  ANNA_REQUIRE(max_len < kQ8MaxLength, "%s: too many tokens", what);
  p.spans = (int)((max_len + block_size - 1) / block_size);
  p.shares = (block_size * head_dim / 16 + kQ8GatherPieces - 1) / kQ8GatherPieces;
  const int64_t warps = (int64_t)batch * kv_heads * p.spans * p.shares * 2;
  ANNA_REQUIRE(warps < (1ll << 31), "%s: too many tokens", what);
  return ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    return ANNA_DISPATCH_TQ_DIM(head_dim, D, [&]() -> int {
      return q8_launch("q8_gather_kernel", q8_gather_kernel<T, D>, dim3((unsigned)((warps + 3) / 4)), 128, 0, (cudaStream_t)stream, p);
    });
  });
}
