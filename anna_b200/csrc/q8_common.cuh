// The 8-bit paged cache: layout of a page and what its kernels share (q8_append.cu, q8_attention.cu, q8_attention_mma.cu, q8_select.cu).
//
// A page holds S tokens of one KV head: key codes int8 [S, D], value codes int8 [S, D], their two scales, and the bounds of the key
// codes, int8 [2, D].  Codes of keys and values lie next to one another and the scales behind them, so that a kernel that reads all of
// a page reads one run; the bounds, which the selection alone reads, are next to the scale that it needs, too.
#pragma once

#include "tq_multi_params.cuh"

namespace anna {

constexpr int kQ8MaxBlockSize = 1024;

__host__ __device__ __forceinline__ int q8_scale_offset(int head_dim, int block_size) { return 2 * block_size * head_dim; }
__host__ __device__ __forceinline__ int q8_bounds_offset(int head_dim, int block_size) { return 2 * block_size * head_dim + 16; }
__host__ __device__ __forceinline__ int q8_page_bytes(int head_dim, int block_size) {
  return (2 * block_size * head_dim + 16 + 2 * head_dim + 127) / 128 * 128;
}
inline bool q8_head_dim(int head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }

// Attention (q8_attention.cu): the multi-token decode's parameters, of which packed codes, signs and centroids are not used.  The keys of
// a stream lie on an axis: its full pages, or with `blocks` the pages that its list names, `width` of them; behind those the tokens of
// the ring.  Row tiles: of all rows, or with `blocks` of the rows of one query token, since each has a list of its own.
struct Q8Params : TqMultiParams {
  int page_bytes;
  const int32_t* blocks;  // [B, Hkv, T, width]
  int width;
  int tiles_per_token;    // row tiles of one query token (blocks only)
  int splits;             // CTAs of a stream (blocks only)
  int64_t num_slots;
};

// What a stream reads: rows row0 .. row0 + count - 1 (row = token * groups + head of the group).
struct Q8Stream {
  int len, full;        // tokens of the sequence, of those in full pages
  int packed;           // tokens of the axis that lie in pages
  int row0, count;
  const int32_t* list;  // the blocks on the axis, or null: all in order
};

template <int ROWS>
__device__ __forceinline__ Q8Stream q8_stream(const Q8Params& p, int64_t b, int kvh, int tile, int len) {
  Q8Stream s;
  s.len = len;
  const int blocks = p.block_shift >= 0 ? len >> p.block_shift : len / p.block_size;
  s.full = blocks * p.block_size;
  s.list = nullptr;
  if (p.blocks == nullptr) {
    s.packed = s.full;
    s.row0 = tile * ROWS;
    s.count = min(ROWS, p.rows - s.row0);
  } else {
    const int token = tile / p.tiles_per_token, part = tile - token * p.tiles_per_token;
    s.packed = p.width * p.block_size;
    s.row0 = token * p.groups + part * ROWS;
    s.count = min(ROWS, p.groups - part * ROWS);
    s.list = p.blocks + ((b * p.kv_heads + kvh) * p.tokens + token) * p.width;
  }
  return s;
}

// Page of entry `entry` of the axis, in bytes from the pool's start, -1: none; *block is its place in the sequence.
__device__ __forceinline__ int64_t q8_page_at(const Q8Params& p, const Q8Stream& s, int64_t b, int kvh, int entry, int* block) {
  const int j = s.list != nullptr ? s.list[entry] : entry;
  *block = j;
  if (j < 0 || (int64_t)j * p.block_size >= s.full) return -1;  // a sequence has no more full pages than the table has columns
  const int32_t pid = p.block_table[b * p.table_stride + j];
  return pid >= 0 && pid < p.num_pages ? ((int64_t)pid * p.kv_heads + kvh) * p.page_bytes : -1;
}

// Calls segment(b, kvh, tile, t0, t1, length, partial) for this CTA's part of the axes.
//
// With blocks all axes are as long, and the host has cut them: `splits` CTAs to a stream, 16-token tiles dealt evenly.  Else CTAs take even shares of a
// line of all streams, as multi_for_each_segment cuts it; at most 32 rows are lined up by every warp by itself, without barriers and with one read of
// the lengths (one row of 4000 tokens 9.9 us either way; 12.3 and 11.7 when its tiles were scored with four warps).
template <typename T, int D, int THREADS, bool kBlocks, typename Fn>
__device__ __forceinline__ void q8_for_each_segment(const Q8Params& p, int row_tiles, Fn&& segment) {
  if constexpr (kBlocks) {
    const int stream = blockIdx.x / p.splits, split = blockIdx.x - stream * p.splits;
    const int rest = stream / row_tiles, tile = stream - rest * row_tiles, b = rest / p.kv_heads, head = rest - b * p.kv_heads;
    const int len = (int)max((int64_t)0, min(p.lengths[b], p.max_len));
    const int ring = p.block_shift >= 0 ? len & (p.block_size - 1) : len % p.block_size, end = p.width * p.block_size + ring;
    const int tiles = (end + kBalancedTileTokens - 1) / kBalancedTileTokens, each = tiles / p.splits, more = tiles - each * p.splits;
    const int t0 = (each * split + min(split, more)) * kBalancedTileTokens, t1 = min(end, t0 + (each + (split < more ? 1 : 0)) * kBalancedTileTokens);
    segment(b, head, tile, t0, t1, len, MultiPartial{stream * p.splits, p.splits, split});
  } else {
    __shared__ int s_prefix[kBalancedMaxRows + 1];
    const bool few = p.batch <= 32;
    const int per_row = p.kv_heads * row_tiles;
    WarpLine line{};
    int total, most;
    if (few) {
      line.load(p.lengths, p.max_len, p.batch, 0);
      total = line.scan(per_row, p.stream_tiles, 0);
      most = __reduce_max_sync(0xffffffffu, line.tiles);
    } else {
      int tiles[kBalancedRowsPerThread<THREADS>], streams;
      balanced_load_tiles<THREADS>(p.lengths, p.max_len, p.batch, 0, tiles);
      most = balanced_scan<THREADS>(tiles, p.batch, per_row, s_prefix, p.stream_tiles, 0, &streams);
      total = s_prefix[p.batch];
    }
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {  // rows without a key
      if (few ? __shfl_sync(0xffffffffu, line.tiles, b & 31) != 0 : s_prefix[b + 1] != s_prefix[b]) continue;
      for (int item = threadIdx.x; item < p.kv_heads * p.rows * (D / 4); item += THREADS) {
        const float zeros[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int row = item / (D / 4);
        multi_store<T, 4>(p, b, row / p.rows, row % p.rows, item % (D / 4) * 4, zeros);
      }
    }
    const int share = max(max((total + (int)gridDim.x - 1) / (int)gridDim.x, p.min_share), (most + kMultiMaxPartials - 3) / (kMultiMaxPartials - 2));
    int pos = (int)min((int64_t)blockIdx.x * share, (int64_t)total), b = 0;
    const int end = min(pos + share, total);
    if (!few && pos < end) {
      int above = p.batch;  // s_prefix[b] <= pos < s_prefix[above]
      while (above - b > 1) {
        const int mid = (b + above) >> 1;
        if (s_prefix[mid] <= pos) b = mid;
        else above = mid;
      }
    }
    while (pos < end) {
      int len, first_of_row;
      if (few) {
        b = __popc(__ballot_sync(0xffffffffu, line.next <= pos));  // rows that end at or before it (never all: pos < total)
        len = __shfl_sync(0xffffffffu, line.len, b);
        first_of_row = __shfl_sync(0xffffffffu, line.first, b);
      } else {
        while (s_prefix[b + 1] <= pos) ++b;
        len = (int)max((int64_t)0, min(p.lengths[b], p.max_len));
        first_of_row = s_prefix[b];
      }
      const int n = (len + kBalancedTileTokens - 1) / kBalancedTileTokens + p.stream_tiles;
      const int stream = (pos - first_of_row) / n, at = pos - first_of_row - stream * n, stop = min(n, at + end - pos);
      if (stop > p.stream_tiles) {
        const int begin = first_of_row + stream * n, first = (begin + p.stream_tiles) / share;
        const int head = stream / row_tiles;
        segment(b, head, stream - head * row_tiles, max(0, at - p.stream_tiles) * kBalancedTileTokens,
                min(len, (stop - p.stream_tiles) * kBalancedTileTokens), len,
                MultiPartial{first, (begin + n - 1) / share - first + 1, (int)blockIdx.x - first});
      }
      pos += stop - at;
    }
  }
}

// Launches of this cache follow one another (append, selection, choice, attention), each of a few microseconds.  They go out with leave to be set up
// while the kernel in front of them ends, and touch no memory before that has ended and its writes are there.  No kernel lets the next one start ahead of
// its own end, as CTAs that wait beside it cost more than that saves: an append and attention of one row of 4000 tokens 11.9 us, 12.5 with early starts, 16.4
// without leave; choice of 128 pages of 32 rows and attention 71.6, 81.7, 79.3; dense view of a prompt behind its append 10.8, 10.8, 14.4.
//
// A kernel may be on the GPU all the same while the one in front of it still writes pages, and pages change their contents between two kernels on one SM: what is read
// of the pool goes by coherent loads alone (__ldg and ld.global.nc are for memory that stays as it is while the kernel lives).
__device__ __forceinline__ void q8_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
int q8_launch(const char* what, void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = (size_t)smem;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
  if (err != cudaSuccess) return set_error(ANNA_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(err));
  return ANNA_OK;
}

// Rows of a tile, CTAs and the scratch of a call; q8_attention.cu plans, both kernels go by it.
struct Q8Plan {
  bool tensor_cores;
  int rows;       // of a row tile
  int warps;      // of a CTA (tensor cores)
  int row_tiles;  // of a (sequence, KV head)
  int tiles_per_token, splits;
  int64_t ctas;   // at most
  int64_t floats;
  int counters;
};

// Tensor-core form (q8_attention_mma_body.cuh): pages of a multiple of 8 tokens.
struct Q8Shape {
  int rows, ctas, warps;  // of a row tile; of an SM; of a CTA
};
Q8Shape q8_mma_shape(int head_dim, int rows, bool few);  // few: one row tile, and no more key tiles than a CTA to an SM has quick work of
template <typename T>
int launch_q8_mma_of(const Q8Params& p, const Q8Plan& plan, int head_dim, int ctas, cudaStream_t stream);

}  // namespace anna
