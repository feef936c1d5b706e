// Rotary positions with several axes, and the same with the rotated keys and the values written into un-quantized pages.
//
// Pair i of a head is its dims (i, i + R/2), R = rotary_dim; a token turns it by the angle a_i = position[axis_i] * rate_i:
//   x1' = x1 cos(a_i) - x2 sin(a_i)     x2' = x2 cos(a_i) + x1 sin(a_i)
// and the head_dim - R dims behind the pairs stay as they are.
//
// Bound: HBM (every vector is read and written once; 3 operations an element).  The angles are the same for all heads of a
// token, so a CTA is a token: R/2 threads work them out, all threads then turn the heads.  The first vectors of a thread are on
// their way before it waits for the angles.  A position times the rate, in turns, is formed in 64 bits and reduced to half a
// turn before it is rounded to 32 bits: at position 262144 the product in 32 bits would be off by up to 0.008 of a radian.
#include "common.cuh"

namespace anna {

struct RotaryRows {  // [batch, heads, tokens, head_dim] with the last dim contiguous
  const void* base;
  int64_t stride_b, stride_h, stride_t;
};

struct RotaryParams {
  RotaryRows q, k, v, q_out, k_out;  // k_out and v: of one of the two forms only
  int q_heads, kv_heads;
  const int64_t* positions;  // [axes, batch, tokens]; nullptr: past + token (+ delta) on every axis
  int64_t pos_stride_a, pos_stride_b, pos_stride_t;
  const int64_t* rope_deltas;
  int64_t delta_stride;
  const double* rates;  // turns per position, [R / 2]
  const int32_t* axes;  // [R / 2]
  float scale;
  int tokens, head_dim, half;  // half = R / 2
  int pieces;                  // of a head: (half + head_dim - R) / VEC
  uint32_t pieces_inverse;     // ceil(2^32 / pieces)
  int items, items_per_cta;
  // paged form
  void* key_pages;
  void* value_pages;
  const int32_t* page_table;
  int64_t table_stride;
  const int64_t* past_lengths;
  int64_t* new_lengths;
  int block_size;
  int64_t num_pages, max_blocks;
  int32_t* status;
};

constexpr int kRotaryThreads = 256;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotaryPiece {
  T x[VEC];
};

// VEC: elements per access.  kPaged: keys go to pages, and the heads behind those of the keys are the values, which do not turn.
template <typename T, int VEC, bool kPaged>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
  using Piece = RotaryPiece<T, VEC>;
  extern __shared__ __align__(16) float sm_angle[];  // cos [half], sin [half]
  float* sm_cos = sm_angle;
  float* sm_sin = sm_angle + p.half;
  const int64_t b = blockIdx.x / p.tokens;
  const int t = (int)(blockIdx.x % p.tokens);

  int64_t page_row = -1;  // of head 0, in elements
  const int64_t past = kPaged || p.positions == nullptr ? p.past_lengths[b] : 0;
  if constexpr (kPaged) {
    const int64_t at = past + t;
    const int64_t blk = at / p.block_size;
    int32_t pid = -1;
    if (at >= 0 && blk < p.max_blocks) pid = p.page_table[b * p.table_stride + blk];
    if (pid >= 0 && pid < p.num_pages)
      page_row = (((int64_t)pid * p.kv_heads) * p.block_size + (at - blk * p.block_size)) * p.head_dim;
    if (blockIdx.y == 0 && threadIdx.x == 0) {
      if (page_row < 0 && p.status != nullptr) atomicOr(p.status, (int)ANNA_DEV_BAD_PAGE);
      if (p.new_lengths != nullptr && t == 0) p.new_lengths[b] = past + p.tokens;
    }
  }

  struct Item {
    const T* src;
    T* dst;  // nullptr: nothing to do
    int at;  // first dim of the piece; of a pair, of its first half
    bool turns, pair;
  };
  auto row = [&](const RotaryRows& r, int h) {
    return reinterpret_cast<T*>(const_cast<void*>(r.base)) + b * r.stride_b + (int64_t)h * r.stride_h + (int64_t)t * r.stride_t;
  };
  const int last = min(p.items, ((int)blockIdx.y + 1) * p.items_per_cta);
  auto find = [&](int item) {
    Item it{nullptr, nullptr, 0, true, true};
    if (item >= last) return it;
    int h = p.pieces == 1 ? item : (int)__umulhi((uint32_t)item, p.pieces_inverse);
    const int piece = item - h * p.pieces;
    it.at = piece * VEC;
    it.pair = it.at < p.half;
    if (!it.pair) it.at += p.half;
    if (h < p.q_heads) {
      it.src = row(p.q, h);
      it.dst = row(p.q_out, h);
    } else {
      h -= p.q_heads;
      if constexpr (kPaged) {
        const bool value = h >= p.kv_heads;
        if (value) h -= p.kv_heads;
        it.turns = !value;
        it.src = row(value ? p.v : p.k, h);
        if (page_row >= 0)
          it.dst = reinterpret_cast<T*>(value ? p.value_pages : p.key_pages) + page_row + (int64_t)h * p.block_size * p.head_dim;
      } else {
        it.src = row(p.k, h);
        it.dst = row(p.k_out, h);
      }
    }
    if (!it.pair && it.src == it.dst) it.dst = nullptr;  // in place
    return it;
  };
  auto load = [&](const Item& it, Piece& x1, Piece& x2) {
    if (it.dst == nullptr) return;
    x1 = *reinterpret_cast<const Piece*>(it.src + it.at);
    if (it.pair) x2 = *reinterpret_cast<const Piece*>(it.src + it.at + p.half);
  };
  auto finish = [&](const Item& it, Piece& x1, Piece& x2) {
    if (it.dst == nullptr) return;
    if (it.pair && it.turns) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float c = sm_cos[it.at + i], s = sm_sin[it.at + i];
        const float a = ElemTraits<T>::to_float(x1.x[i]), z = ElemTraits<T>::to_float(x2.x[i]);
        x1.x[i] = ElemTraits<T>::from_float(fmaf(a, c, -(z * s)));
        x2.x[i] = ElemTraits<T>::from_float(fmaf(z, c, a * s));
      }
    }
    *reinterpret_cast<Piece*>(it.dst + it.at) = x1;
    if (it.pair) *reinterpret_cast<Piece*>(it.dst + it.at + p.half) = x2;
  };

  constexpr int U = 2;
  Item it[U];
  Piece x1[U], x2[U];
  const int first = (int)blockIdx.y * p.items_per_cta + (int)threadIdx.x;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    it[u] = find(first + u * kRotaryThreads);
    load(it[u], x1[u], x2[u]);
  }
  for (int i = threadIdx.x; i < p.half; i += kRotaryThreads) {
    int64_t position;
    if (p.positions != nullptr) {
      position = p.positions[p.axes[i] * p.pos_stride_a + b * p.pos_stride_b + t * p.pos_stride_t];
    } else {
      position = past + t + (p.rope_deltas != nullptr ? p.rope_deltas[b * p.delta_stride] : 0);
    }
    double turns = (double)position * p.rates[i];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    sm_cos[i] = c * p.scale;
    sm_sin[i] = s * p.scale;
  }
  __syncthreads();
  for (int base = first;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) finish(it[u], x1[u], x2[u]);
    base += U * kRotaryThreads;
    if (base >= last) break;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      it[u] = find(base + u * kRotaryThreads);
      load(it[u], x1[u], x2[u]);
    }
  }
}

// The same for many tokens, where a vector is 4, 8, 16 or 32 pieces of 16 bytes: a lane holds a piece, and the other half of its pairs
// comes from another lane, so that a vector is one load and one store of neighbouring lanes and its addresses are worked out once.
// A CTA takes several tokens, and a lane has kRowsAhead vectors on their way.  (With the kernel above, 222 instructions per 32 pieces:
// 16383 tokens of 20 heads of 256 dims, 64 turned, 156 us; 66 us so,
// 5.1 TB/s.  Two or eight vectors ahead, four or sixteen tokens a CTA: as fast or slower.)
constexpr int kManyTokens = 8, kRowsAhead = 4;

struct RotaryToken {
  int64_t q, k, v, q_out, k_out;  // element offsets of head 0
  int64_t page;                   // of head 0 in the pools, -1: not written
  int64_t start;                  // position where none are given
  int64_t given;                  // offset of the token's positions
};

template <typename T, int PIECES, bool kPaged>
__global__ void __launch_bounds__(kRotaryThreads) rotary_rows_kernel(const RotaryParams p, int64_t all_tokens, int per_cta,
                                                                     uint32_t half_inverse) {
  constexpr int VEC = 16 / (int)sizeof(T), kRows = 32 / PIECES;  // vectors of a warp
  constexpr int kStep = kRotaryThreads / 32 * kRows;
  extern __shared__ __align__(16) float sm_angle[];  // cos [tokens][half], sin [tokens][half]
  __shared__ RotaryToken sm_token[kManyTokens];
  const int64_t first = (int64_t)blockIdx.x * per_cta;
  const int count = (int)min((int64_t)per_cta, all_tokens - first);
  float* sm_cos = sm_angle;
  float* sm_sin = sm_angle + per_cta * p.half;
  if ((int)threadIdx.x < count) {
    const int64_t b = (first + threadIdx.x) / p.tokens, t = (first + threadIdx.x) - b * p.tokens;
    RotaryToken token{b * p.q.stride_b + t * p.q.stride_t, b * p.k.stride_b + t * p.k.stride_t, b * p.v.stride_b + t * p.v.stride_t,
                      b * p.q_out.stride_b + t * p.q_out.stride_t, b * p.k_out.stride_b + t * p.k_out.stride_t, -1, 0,
                      b * p.pos_stride_b + t * p.pos_stride_t};
    const int64_t past = kPaged || p.positions == nullptr ? p.past_lengths[b] : 0;
    if (p.positions == nullptr) token.start = past + t + (p.rope_deltas != nullptr ? p.rope_deltas[b * p.delta_stride] : 0);
    if constexpr (kPaged) {
      const int64_t at = past + t, blk = at / p.block_size;
      int32_t pid = -1;
      if (at >= 0 && blk < p.max_blocks) pid = p.page_table[b * p.table_stride + blk];
      if (pid >= 0 && pid < p.num_pages)
        token.page = (((int64_t)pid * p.kv_heads) * p.block_size + (at - blk * p.block_size)) * p.head_dim;
      else if (p.status != nullptr)
        atomicOr(p.status, (int)ANNA_DEV_BAD_PAGE);
      if (p.new_lengths != nullptr && t == 0) p.new_lengths[b] = past + p.tokens;
    }
    sm_token[threadIdx.x] = token;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * p.half; i += kRotaryThreads) {
    const int token = p.half == 1 ? i : (int)__umulhi((uint32_t)i, half_inverse), pair = i - token * p.half;
    const int64_t position = p.positions != nullptr ? p.positions[p.axes[pair] * p.pos_stride_a + sm_token[token].given] : sm_token[token].start;
    double turns = (double)position * p.rates[pair];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    sm_cos[i] = c * p.scale;
    sm_sin[i] = s * p.scale;
  }
  __syncthreads();

  const int lane = threadIdx.x & 31, at = lane % PIECES * VEC;  // first dim of this lane's piece
  const int heads = p.q_heads + p.kv_heads * (kPaged ? 2 : 1);
  const bool low = at < p.half, turns = at < 2 * p.half;
  const int partner = turns ? lane + (low ? p.half / VEC : -(p.half / VEC)) : lane;
  const int angle = low ? at : at - p.half;
  int token = 0, h = (int)(threadIdx.x >> 5) * kRows + lane / PIECES;  // of this lane's next vector
  while (h >= heads) { h -= heads; ++token; }
  for (int rest = count * heads - (int)(threadIdx.x >> 5) * kRows; rest > 0; rest -= kRowsAhead * kStep) {
    uint4 x[kRowsAhead];
    T* dst[kRowsAhead];         // nullptr: nothing to do
    int angles[kRowsAhead];     // negative: the vector does not turn
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      dst[u] = nullptr;
      angles[u] = -1;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      if (token < count) {
        const RotaryToken& tk = sm_token[token];
        const T* src;
        angles[u] = token * p.half + angle;
        if (h < p.q_heads) {
          src = reinterpret_cast<const T*>(p.q.base) + tk.q + (int64_t)h * p.q.stride_h + at;
          dst[u] = reinterpret_cast<T*>(const_cast<void*>(p.q_out.base)) + tk.q_out + (int64_t)h * p.q_out.stride_h + at;
        } else {
          int kh = h - p.q_heads;
          if constexpr (kPaged) {
            const bool value = kh >= p.kv_heads;
            if (value) {
              kh -= p.kv_heads;
              angles[u] = -1;
            }
            src = value ? reinterpret_cast<const T*>(p.v.base) + tk.v + (int64_t)kh * p.v.stride_h + at
                        : reinterpret_cast<const T*>(p.k.base) + tk.k + (int64_t)kh * p.k.stride_h + at;
            if (tk.page >= 0)
              dst[u] = reinterpret_cast<T*>(value ? p.value_pages : p.key_pages) + tk.page + kh * p.block_size * p.head_dim + at;
          } else {
            src = reinterpret_cast<const T*>(p.k.base) + tk.k + (int64_t)kh * p.k.stride_h + at;
            dst[u] = reinterpret_cast<T*>(const_cast<void*>(p.k_out.base)) + tk.k_out + (int64_t)kh * p.k_out.stride_h + at;
          }
        }
        if (dst[u] != nullptr) x[u] = *reinterpret_cast<const uint4*>(src);
      }
      h += kStep;
      while (h >= heads) { h -= heads; ++token; }
    }
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      uint4 other;
      other.x = __shfl_sync(0xffffffffu, x[u].x, partner);
      other.y = __shfl_sync(0xffffffffu, x[u].y, partner);
      other.z = __shfl_sync(0xffffffffu, x[u].z, partner);
      other.w = __shfl_sync(0xffffffffu, x[u].w, partner);
      if (turns && angles[u] >= 0) {
        float mine[VEC], theirs[VEC];
        widen16<T>(x[u], mine);
        widen16<T>(other, theirs);
        T* out = reinterpret_cast<T*>(&x[u]);
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {  // half is a multiple of VEC, so the angles of a piece are aligned
          const float4 c = *reinterpret_cast<const float4*>(sm_cos + angles[u] + i), s = *reinterpret_cast<const float4*>(sm_sin + angles[u] + i);
          const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            out[i + k] = ElemTraits<T>::from_float(fmaf(mine[i + k], cs[k], low ? -(theirs[i + k] * sn[k]) : theirs[i + k] * sn[k]));
        }
      }
      if (dst[u] != nullptr) *reinterpret_cast<uint4*>(dst[u]) = x[u];
    }
  }
}

// Widest access in bytes that rows of this kind allow.
static size_t rotary_access(const RotaryRows& r, size_t elem) {
  size_t bytes = 16;
  for (const uint64_t v : {(uint64_t)reinterpret_cast<uintptr_t>(r.base), (uint64_t)(r.stride_b * (int64_t)elem),
                           (uint64_t)(r.stride_h * (int64_t)elem), (uint64_t)(r.stride_t * (int64_t)elem)})
    while (v % bytes != 0) bytes /= 2;
  return bytes;
}

static int launch_rotary(RotaryParams& p, int batch, int rotary_dim, int dtype, bool paged, const char* what, cudaStream_t stream) {
  ANNA_REQUIRE(p.q.base && p.q_out.base && p.k.base && p.rates && p.axes, "%s: null pointer argument", what);
  ANNA_REQUIRE(batch > 0 && p.q_heads > 0 && p.kv_heads > 0 && p.tokens > 0 && p.head_dim > 0, "%s: sizes must be positive", what);
  ANNA_REQUIRE(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= p.head_dim && p.head_dim <= 4096,
               "%s: rotary_dim %d must be even and at most head_dim %d (at most 4096)", what, rotary_dim, p.head_dim);
  ANNA_REQUIRE((int64_t)batch * p.tokens < (1ll << 31), "%s: too many tokens", what);
  ANNA_REQUIRE(dtype == ANNA_DTYPE_F32 || dtype == ANNA_DTYPE_F16 || dtype == ANNA_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
  const size_t elem = dtype == ANNA_DTYPE_F32 ? 4 : 2;
  p.half = rotary_dim / 2;
  size_t access = 16;
  auto narrow = [&](size_t to) { access = to < access ? to : access; };
  for (const RotaryRows* r : {&p.q, &p.q_out, &p.k}) narrow(rotary_access(*r, elem));
  if (paged) {
    narrow(rotary_access(p.v, elem));
    const RotaryRows keys{p.key_pages, 0, p.head_dim, 0}, values{p.value_pages, 0, p.head_dim, 0};
    narrow(rotary_access(keys, elem));
    narrow(rotary_access(values, elem));
  } else {
    narrow(rotary_access(p.k_out, elem));
  }
  ANNA_REQUIRE(access >= elem, "%s: tensors must be aligned to their elements", what);
  while (p.half * elem % access != 0 || (p.head_dim - rotary_dim) * elem % access != 0) access /= 2;
  const int vec = (int)(access / elem);
  p.pieces = (p.half + p.head_dim - rotary_dim) / vec;
  p.pieces_inverse = (uint32_t)(((1ull << 32) + p.pieces - 1) / p.pieces);  // of one piece: not read
  const int heads = p.q_heads + p.kv_heads * (paged ? 2 : 1);
  // the quotient by the rounded inverse is exact while items * pieces < 2^32
  ANNA_REQUIRE((int64_t)heads * p.pieces * p.pieces < (1ll << 32), "%s: %d heads of %d dims are not supported", what,
               heads, p.head_dim);
  p.items = heads * p.pieces;
  // A token's heads go to several CTAs where the tokens alone leave SMs without one.
  const int64_t tokens = (int64_t)batch * p.tokens;
  int splits = (p.items + kRotaryThreads - 1) / kRotaryThreads;
  while (splits > 1 && tokens * splits > 148 * 4) --splits;
  p.items_per_cta = ((p.items + splits - 1) / splits + 31) / 32 * 32;
  const dim3 grid((unsigned)tokens, (unsigned)((p.items + p.items_per_cta - 1) / p.items_per_cta));
  const size_t smem = 2 * p.half * sizeof(float);
  // Many tokens: several a CTA, as long as that leaves four CTAs for each of the eight that an SM holds.
  const int row_pieces = access == 16 ? p.head_dim / vec : 0;
  int per_cta = (int)(tokens / (148 * 8) < kManyTokens ? tokens / (148 * 8) : kManyTokens);
  while (per_cta > 1 && per_cta * (int64_t)p.half > 2048) --per_cta;
  const bool rows = per_cta > 1 && p.half <= 2048 && (row_pieces == 4 || row_pieces == 8 || row_pieces == 16 || row_pieces == 32) &&
                    (!paged || (int64_t)p.kv_heads * p.block_size * p.head_dim < (1ll << 31));
  const uint32_t half_inverse = (uint32_t)(((1ull << 32) + p.half - 1) / p.half);  // exact below 2^32 / half
  return ANNA_DISPATCH_DTYPE(dtype, T, [&]() -> int {
    if (rows) {
      const unsigned ctas = (unsigned)((tokens + per_cta - 1) / per_cta);
      auto many = [&](auto pieces) {
        constexpr int PIECES = decltype(pieces)::value;
        if (paged) rotary_rows_kernel<T, PIECES, true><<<ctas, kRotaryThreads, per_cta * smem, stream>>>(p, tokens, per_cta, half_inverse);
        else rotary_rows_kernel<T, PIECES, false><<<ctas, kRotaryThreads, per_cta * smem, stream>>>(p, tokens, per_cta, half_inverse);
      };
      if (row_pieces == 4) many(std::integral_constant<int, 4>{});
      if (row_pieces == 8) many(std::integral_constant<int, 8>{});
      if (row_pieces == 16) many(std::integral_constant<int, 16>{});
      if (row_pieces == 32) many(std::integral_constant<int, 32>{});
      return check_launch("rotary_rows_kernel");
    }
    auto launch = [&](auto width) {
      constexpr int VEC = decltype(width)::value;
      if (paged) rotary_kernel<T, VEC, true><<<grid, kRotaryThreads, smem, stream>>>(p);
      else rotary_kernel<T, VEC, false><<<grid, kRotaryThreads, smem, stream>>>(p);
    };
    if constexpr (sizeof(T) == 2) {
      if (vec == 8) launch(std::integral_constant<int, 8>{});
    }
    if (vec == 4) launch(std::integral_constant<int, 4>{});
    if (vec == 2) launch(std::integral_constant<int, 2>{});
    if (vec == 1) launch(std::integral_constant<int, 1>{});
    return check_launch("rotary_kernel");
  });
}

}  // namespace anna

using namespace anna;

extern "C" int anna_multi_axis_rotary(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, void* q_out,
                                      int64_t qo_stride_b, int64_t qo_stride_h, int64_t qo_stride_t, const void* k,
                                      int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t, void* k_out,
                                      int64_t ko_stride_b, int64_t ko_stride_h, int64_t ko_stride_t, const int64_t* positions,
                                      int64_t pos_stride_a, int64_t pos_stride_b, int64_t pos_stride_t,
                                      const int64_t* past_lengths, const int64_t* rope_deltas, int64_t delta_stride,
                                      const double* rates, const int32_t* axes, float scale, int batch, int q_heads, int kv_heads, int tokens,
                                      int head_dim, int rotary_dim, int dtype, anna_stream_t stream) {
  ANNA_REQUIRE((positions != nullptr || past_lengths != nullptr) && k_out != nullptr, "anna_multi_axis_rotary: null pointer argument");
  RotaryParams p{};
  p.past_lengths = past_lengths; p.rope_deltas = rope_deltas; p.delta_stride = delta_stride;
  p.q = {q, q_stride_b, q_stride_h, q_stride_t};
  p.q_out = {q_out, qo_stride_b, qo_stride_h, qo_stride_t};
  p.k = {k, k_stride_b, k_stride_h, k_stride_t};
  p.k_out = {k_out, ko_stride_b, ko_stride_h, ko_stride_t};
  p.positions = positions;
  p.pos_stride_a = pos_stride_a; p.pos_stride_b = pos_stride_b; p.pos_stride_t = pos_stride_t;
  p.rates = rates; p.axes = axes; p.scale = scale;
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.tokens = tokens; p.head_dim = head_dim;
  return launch_rotary(p, batch, rotary_dim, dtype, false, "anna_multi_axis_rotary", (cudaStream_t)stream);
}

extern "C" int anna_rotary_paged_kv_write(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t, void* q_out,
                                          int64_t qo_stride_b, int64_t qo_stride_h, int64_t qo_stride_t, const void* k,
                                          int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t, const void* v,
                                          int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, void* key_pages,
                                          void* value_pages, const int32_t* page_table, int64_t table_stride,
                                          const int64_t* past_lengths, int64_t* new_lengths, const int64_t* positions,
                                          int64_t pos_stride_a, int64_t pos_stride_b, int64_t pos_stride_t,
                                          const int64_t* rope_deltas, int64_t delta_stride, const double* rates,
                                          const int32_t* axes, float scale, int batch, int q_heads, int kv_heads, int tokens,
                                          int head_dim, int rotary_dim, int block_size, int64_t num_pages, int64_t max_blocks,
                                          int dtype, int32_t* status, anna_stream_t stream) {
  ANNA_REQUIRE(v && key_pages && value_pages && page_table && past_lengths, "anna_rotary_paged_kv_write: null pointer argument");
  ANNA_REQUIRE(new_lengths != past_lengths, "anna_rotary_paged_kv_write: new_lengths must not alias past_lengths");
  ANNA_REQUIRE(block_size > 0 && num_pages > 0 && max_blocks > 0, "anna_rotary_paged_kv_write: sizes must be positive");
  RotaryParams p{};
  p.q = {q, q_stride_b, q_stride_h, q_stride_t};
  p.q_out = {q_out, qo_stride_b, qo_stride_h, qo_stride_t};
  p.k = {k, k_stride_b, k_stride_h, k_stride_t};
  p.v = {v, v_stride_b, v_stride_h, v_stride_t};
  p.key_pages = key_pages; p.value_pages = value_pages;
  p.page_table = page_table; p.table_stride = table_stride;
  p.past_lengths = past_lengths; p.new_lengths = new_lengths;
  p.positions = positions;
  p.pos_stride_a = pos_stride_a; p.pos_stride_b = pos_stride_b; p.pos_stride_t = pos_stride_t;
  p.rope_deltas = rope_deltas; p.delta_stride = delta_stride;
  p.rates = rates; p.axes = axes; p.scale = scale;
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.tokens = tokens; p.head_dim = head_dim;
  p.block_size = block_size; p.num_pages = num_pages; p.max_blocks = max_blocks; p.status = status;
  return launch_rotary(p, batch, rotary_dim, dtype, true, "anna_rotary_paged_kv_write", (cudaStream_t)stream);
}
