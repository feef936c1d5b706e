// Copies of whole pages within and between page pools, any number of pools in one launch: forks of sequences (window rings, partly
// filled pages of all layers) and compaction (the live pages of all layers move to smaller pools).
//
// Bound: HBM for large copies (each page read once and written once), the launch for small ones: 224 pages of 32 pools as tensor
// operations are 32 gathers, 32 scatters and the upload of the ids.  What a launch has to know travels in its parameters where it
// fits (128 pools and 2816 pairs of ids, 29 KB), so that an ordinary fork uploads nothing.
//
// The work is cut into units of at most kUnitBytes of one page, whatever the pages' sizes; a CTA finds the pool of a unit by bisection
// over the pools' first units, which it keeps in shared memory.
#include "common.cuh"

#include <cstring>

namespace anna {

constexpr int kCopyThreads = 256;
constexpr int kCopyInFlight = 4;  // accesses per thread before the first store
constexpr int kUnitBytes = kCopyThreads * kCopyInFlight * 16;

struct CopyPool {
  const uint8_t* src;
  uint8_t* dst;
  int64_t page_bytes;
  int64_t first_unit;
  int32_t src_pages, dst_pages;
  int32_t first_pair;
  int32_t units_per_page;
  int32_t access;      // bytes
  int32_t unit_bytes;  // the page's bytes dealt evenly, in whole 512
};

template <int POOLS, int PAIRS>
struct CopyTables {
  CopyPool pools[POOLS];
  int2 pairs[PAIRS > 0 ? PAIRS : 1];  // (source page, target page); PAIRS == 0: in device memory
};

template <typename W>
__device__ __forceinline__ void copy_unit(const uint8_t* src, uint8_t* dst, int64_t bytes) {
  const W* from = reinterpret_cast<const W*>(src);
  W* to = reinterpret_cast<W*>(dst);
  const int64_t words = bytes / (int64_t)sizeof(W);
  for (int64_t base = threadIdx.x; base < words; base += kCopyThreads * kCopyInFlight) {
    W held[kCopyInFlight];
#pragma unroll
    for (int i = 0; i < kCopyInFlight; ++i)
      if (base + i * kCopyThreads < words) held[i] = __ldcs(from + base + i * kCopyThreads);
#pragma unroll
    for (int i = 0; i < kCopyInFlight; ++i)
      if (base + i * kCopyThreads < words) __stcs(to + base + i * kCopyThreads, held[i]);
  }
}

template <int POOLS, int PAIRS>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ CopyTables<POOLS, PAIRS> t, int num_pools,
                                                                 int64_t units, const int2* device_pairs, int32_t* status) {
  __shared__ int64_t first_unit[POOLS];
  for (int i = threadIdx.x; i < num_pools; i += kCopyThreads) first_unit[i] = t.pools[i].first_unit;
  __syncthreads();
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    int lo = 0, hi = num_pools - 1;  // the last pool that starts at or before the unit
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first_unit[mid] <= unit) lo = mid;
      else hi = mid - 1;
    }
    const CopyPool& pool = t.pools[lo];
    const int64_t mine = unit - pool.first_unit;
    const int64_t copy = mine / pool.units_per_page;
    const int64_t at = (mine - copy * pool.units_per_page) * pool.unit_bytes;
    const int2 pair = PAIRS > 0 ? t.pairs[PAIRS > 0 ? pool.first_pair + copy : 0] : device_pairs[pool.first_pair + copy];
    if (pair.x < 0 || pair.x >= pool.src_pages || pair.y < 0 || pair.y >= pool.dst_pages) {
      if (status != nullptr && threadIdx.x == 0) atomicOr(status, (int)ANNA_DEV_BAD_PAGE);
      continue;
    }
    const uint8_t* src = pool.src + pair.x * pool.page_bytes + at;
    uint8_t* dst = pool.dst + pair.y * pool.page_bytes + at;
    const int64_t bytes = min((int64_t)pool.unit_bytes, pool.page_bytes - at);
    if (pool.access == 16) copy_unit<uint4>(src, dst, bytes);
    else if (pool.access >= 4) copy_unit<uint32_t>(src, dst, bytes);
    else copy_unit<uint8_t>(src, dst, bytes);
  }
}

template <int POOLS, int PAIRS>
static int launch_copies(const CopyPool* pools, int num_pools, const int2* pairs, int num_pairs, const int2* device_pairs, int64_t units,
                         int32_t* status, cudaStream_t stream) {
  CopyTables<POOLS, PAIRS> t;
  memcpy(t.pools, pools, sizeof(CopyPool) * num_pools);
  if (PAIRS > 0) memcpy(t.pairs, pairs, sizeof(int2) * num_pairs);
  // a CTA per unit: 300 window rings of four layers 201 us (6.2 TB/s), 228 with eight CTAs per SM that go on from unit to unit
  const int64_t ctas = units < INT32_MAX ? units : INT32_MAX;
  page_copy_kernel<POOLS, PAIRS><<<(unsigned)ctas, kCopyThreads, 0, stream>>>(t, num_pools, units, device_pairs, status);
  return check_launch("page_copy_kernel");
}

constexpr int kCopyMaxPools = 128, kCopyMaxPairs = 2816;
constexpr int kCopyFewPools = 32, kCopyFewPairs = 256;

}  // namespace anna

using namespace anna;

extern "C" int anna_page_copy_max_pairs(void) { return kCopyMaxPairs; }

extern "C" int anna_page_copy(const anna_page_pool* pools, int num_pools, const int32_t* pairs, int64_t num_pairs,
                              const int32_t* device_pairs, int32_t* status, anna_stream_t stream) {
  ANNA_REQUIRE(num_pools >= 0 && (num_pools == 0 || pools != nullptr), "anna_page_copy: pools missing");
  ANNA_REQUIRE(num_pairs >= 0 && num_pairs < (1ll << 31), "anna_page_copy: bad number of pairs");
  ANNA_REQUIRE(device_pairs != nullptr || (num_pairs <= kCopyMaxPairs && (num_pairs == 0 || pairs != nullptr)),
               "anna_page_copy: more than %d pairs of page ids have to be in device memory", kCopyMaxPairs);
  ANNA_REQUIRE(device_pairs == nullptr || aligned_to(device_pairs, 8), "anna_page_copy: device_pairs must be 8-byte aligned");
  for (int i = 0; i < num_pools; ++i) {
    const anna_page_pool& g = pools[i];
    ANNA_REQUIRE(g.count >= 0 && g.first_pair >= 0 && g.first_pair + (int64_t)g.count <= num_pairs,
                 "anna_page_copy: pool %d names pairs that are not there", i);
    ANNA_REQUIRE(g.page_bytes >= 0 && g.src_pages >= 0 && g.dst_pages >= 0, "anna_page_copy: pool %d has negative sizes", i);
    ANNA_REQUIRE(g.count == 0 || g.page_bytes == 0 || (g.src != nullptr && g.dst != nullptr), "anna_page_copy: pool %d has no memory", i);
    ANNA_REQUIRE((g.page_bytes + kUnitBytes - 1) / kUnitBytes < (1ll << 31), "anna_page_copy: pages of pool %d are too large", i);
  }
  for (int at = 0; at < num_pools;) {
    CopyPool some[kCopyMaxPools];
    int n = 0;
    int64_t units = 0;
    for (; at < num_pools && n < kCopyMaxPools; ++at) {
      const anna_page_pool& g = pools[at];
      if (g.count == 0 || g.page_bytes == 0) continue;
      CopyPool& c = some[n++];
      c = CopyPool{};
      c.src = static_cast<const uint8_t*>(g.src);
      c.dst = static_cast<uint8_t*>(g.dst);
      c.page_bytes = g.page_bytes;
      c.first_unit = units;
      c.src_pages = g.src_pages;
      c.dst_pages = g.dst_pages;
      c.first_pair = g.first_pair;
      c.units_per_page = (int32_t)((g.page_bytes + kUnitBytes - 1) / kUnitBytes);
      c.unit_bytes = (int32_t)(((g.page_bytes + c.units_per_page - 1) / c.units_per_page + 511) / 512 * 512);
      c.access = 16;
      while (reinterpret_cast<uintptr_t>(g.src) % c.access || reinterpret_cast<uintptr_t>(g.dst) % c.access || g.page_bytes % c.access)
        c.access /= 2;
      units += (int64_t)c.units_per_page * g.count;
    }
    if (n == 0) continue;
    const int2* host = reinterpret_cast<const int2*>(pairs);
    const int2* device = reinterpret_cast<const int2*>(device_pairs);
    int rc;
    if (device_pairs != nullptr) rc = launch_copies<kCopyMaxPools, 0>(some, n, nullptr, 0, device, units, status, (cudaStream_t)stream);
    else if (n <= kCopyFewPools && num_pairs <= kCopyFewPairs)
      rc = launch_copies<kCopyFewPools, kCopyFewPairs>(some, n, host, (int)num_pairs, nullptr, units, status, (cudaStream_t)stream);
    else rc = launch_copies<kCopyMaxPools, kCopyMaxPairs>(some, n, host, (int)num_pairs, nullptr, units, status, (cudaStream_t)stream);
    if (rc != ANNA_OK) return rc;
  }
  return ANNA_OK;
}
