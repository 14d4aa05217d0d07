// Block tables and slot maps from request lengths (cutt_pages_build), and rows stored into and
// loaded from pages (cutt_pages_store, cutt_pages_load).
#include <cooperative_groups.h>
#include <stdint.h>

#include "rows.h"

namespace cuttb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// Exclusive prefix sums of (tokens, pages) over the block: tokens saturate, pages cannot overflow
// (a table has fewer than 2^30 entries).
__device__ __forceinline__ uint2 block_scan2(uint2 v, uint2* s, uint2& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  uint2 x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned t = __shfl_up_sync(kFull, x.x, d), p = __shfl_up_sync(kFull, x.y, d);
    if (lane >= d) {
      x.x = add_up_to_int(x.x, t);
      x.y += p;
    }
  }
  uint2 before;                  // exclusive within the warp
  before.x = __shfl_up_sync(kFull, x.x, 1);
  before.y = __shfl_up_sync(kFull, x.y, 1);
  if (lane == 0) before = make_uint2(0, 0);
  if (lane == 31) s[w] = x;
  __syncthreads();
  uint2 y = lane < nw ? s[lane] : make_uint2(0, 0);      // every warp scans the warps' sums
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned t = __shfl_up_sync(kFull, y.x, d), p = __shfl_up_sync(kFull, y.y, d);
    if (lane >= d) {
      y.x = add_up_to_int(y.x, t);
      y.y += p;
    }
  }
  total.x = __shfl_sync(kFull, y.x, nw - 1);
  total.y = __shfl_sync(kFull, y.y, nw - 1);
  const unsigned bx = __shfl_sync(kFull, y.x, w > 0 ? w - 1 : 0), by = __shfl_sync(kFull, y.y, w > 0 ? w - 1 : 0);
  if (w > 0) {
    before.x = add_up_to_int(before.x, bx);
    before.y += by;
  }
  __syncthreads();
  return before;
}

// Prefix sums of the new tokens and of the pages they take, by one block: to shared memory (toks,
// pags) where those are given, to tokenOffset and pageOffset where `writes` is set.
struct Pool {
  int first, limit, entries;      // next free entry and number of entries of the free list, clamped; as given
};
__device__ __forceinline__ Pool read_pool(const PagesBuild& p, const int* poolIn) {
  Pool r = {0, 0, 0};
  if (p.freeList) {
    r.first = clamp_pool(poolIn[0]);
    r.entries = poolIn[1];
    r.limit = clamp_pool(r.entries);
  }
  return r;
}
__device__ __forceinline__ uint2 scan_requests(const PagesBuild& p, const Pool& pool, int* tokenOffset, int* pageOffset, bool writes,
                                               int* toks, int* pags) {
  __shared__ uint2 s[32];
  unsigned tokens = 0, pages = pool.first;
  for (int b0 = 0; b0 < p.s.requests; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const bool in = b < p.s.requests;
    const int n = in ? max(0, p.added[b]) : 0;
    const int g = in && p.freeList ? pages_taken(p.held[b], n, p.s.divPage, p.s.tableWidth) : 0;
    uint2 total;
    const uint2 at = block_scan2(make_uint2(n, g), s, total);
    if (in) {
      const int t = (int)add_up_to_int(tokens, at.x), f = (int)(pages + at.y);
      if (writes) {
        tokenOffset[b] = t;
        if (p.freeList) pageOffset[b] = f;
      }
      if (toks) {
        toks[b] = t;
        pags[b] = f;
      }
    }
    tokens = add_up_to_int(tokens, total.x);
    pages += total.y;
  }
  if (threadIdx.x == 0) {
    if (writes) {
      tokenOffset[p.s.requests] = (int)tokens;
      if (p.freeList) pageOffset[p.s.requests] = (int)pages;
    }
    if (toks) {
      toks[p.s.requests] = (int)tokens;
      pags[p.s.requests] = (int)pages;
    }
  }
  return make_uint2(tokens, pages);
}
__device__ __forceinline__ void write_pool(const PagesBuild& p, const Pool& pool, unsigned pages, int* poolOut) {
  if (!p.freeList || threadIdx.x != 0) return;
  poolOut[0] = min((int)pages, max(pool.first, pool.limit));
  poolOut[1] = pool.entries;
}

// Slots and new table entries, a part of them for each of `blocks` blocks.
__device__ __forceinline__ void expand_requests(const PagesBuild& p, int limit, int block, int blocks) {
  const int stride = blocks * blockDim.x, at = block * blockDim.x + threadIdx.x;
  const int tokens = p.tokenOffset[p.s.requests];
#pragma unroll 2
  for (int q = at; q < p.s.maxTokens; q += stride) {
    long long slot = -1;
    if (q < tokens) slot = slot_of_token(p, last_at_or_before(p.tokenOffset, p.s.requests + 1, q), q, limit);
    p.slot[q] = slot;
  }
  if (!p.freeList) return;
  const int end = p.pageOffset[p.s.requests];
  for (long long f = (long long)p.pageOffset[0] + at; f < end; f += stride)      // end may be close to 2^31
    take_page(p, last_at_or_before(p.pageOffset, p.s.requests + 1, (int)f), (int)f, limit);
}

// One kernel.  Every block makes all prefix sums for itself, in shared memory: a few kilobytes of
// lengths, and no exchange.  Table entries that are read (pages of held tokens) and written (new ones)
// differ, and slots of new pages come from the free list, so blocks wait for nothing - unless the
// pool is updated in place (`inPlace`): then the blocks are one cluster, and the pool is written
// after all of them have read it.
constexpr int kSharedRequests = 4096;

__global__ void __launch_bounds__(1024)
pages_build(const __grid_constant__ PagesBuild p, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset, bool inPlace) {
  extern __shared__ int smem[];
  begin_row_kernel();
  int* toks = smem;
  int* pags = smem + p.s.requests + 1;
  const Pool pool = read_pool(p, poolIn);
  const uint2 sums = scan_requests(p, pool, tokenOffset, pageOffset, blockIdx.x == 0, toks, pags);
  if (inPlace) cooperative_groups::this_cluster().sync();
  else __syncthreads();
  if (blockIdx.x == 0) write_pool(p, pool, sums.y, poolOut);
  PagesBuild q = p;
  q.tokenOffset = toks;
  q.pageOffset = pags;
  expand_requests(q, pool.limit, blockIdx.x, gridDim.x);
}

// Two kernels: prefix sums by one block, then the rest by many.
__global__ void __launch_bounds__(1024)
pages_scan(const __grid_constant__ PagesBuild p, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset) {
  begin_row_kernel();
  const Pool pool = read_pool(p, poolIn);
  const uint2 sums = scan_requests(p, pool, tokenOffset, pageOffset, true, nullptr, nullptr);
  __syncthreads();          // every thread has read the pool, which may be updated in place
  write_pool(p, pool, sums.y, poolOut);
}

constexpr int kExpandThreads = 256;

__global__ void __launch_bounds__(kExpandThreads) pages_expand(const __grid_constant__ PagesBuild p) {
  begin_row_kernel();
  expand_requests(p, p.freeList ? clamp_pool(p.pool[1]) : 0, blockIdx.x, gridDim.x);
}

template <int VB> struct Raw;
template <> struct Raw<16> { typedef uint4 T; };
template <> struct Raw<8> { typedef uint2 T; };
template <> struct Raw<4> { typedef uint32_t T; };
template <> struct Raw<2> { typedef uint16_t T; };
template <> struct Raw<1> { typedef uint8_t T; };

struct PagedLaunch {
  PagedItems p;
  PagedMove m;
};

// grid.x: groups of perBlock tokens, grid.y: tensors.  A thread's loads are all issued before its first
// store.  Memory bounds it: 131072 K and V rows of 2 KB take 165 us, 6.5 TB/s.  Measured there: blocks of
// 64, 128, 256, 512 threads with four loads each 166, 165, 182, 224; 128 threads with 6, 8 loads 173, 183;
// 256 threads with 1, 2, 3 loads 222, 197, 181.  Loads and stores are marked as not to be used again
// (ld.cs, st.cs): 8192 rows stored before 131072 are loaded 192 instead of 207 us (256 threads), since the
// marked lines make room for one another.
// STORE is a template parameter: with a flag the loads of a thread are no longer in flight at once (204
// instead of 165 us).
// A row is read only once its slot is known to be one of the cache's: k and v may end before the tokens whose
// slots are not.  FIRST: a thread looks up the slots of all its accesses before the first of them, else one by
// one (which takes fewer registers); kFirstBlocks says when.
template <int VB, bool STORE, bool FIRST>
__global__ void __launch_bounds__(kPagedThreads) paged_kernel(const __grid_constant__ PagedLaunch l) {
  typedef typename Raw<VB>::T R;
  begin_row_kernel();
  const int q0 = blockIdx.x * l.p.perBlock;
  const unsigned char* src = l.m.src[blockIdx.y];
  unsigned char* dst = l.m.dst[blockIdx.y];
  const uint32_t items = (uint32_t)min(l.p.perBlock, l.p.s.tokens - q0) * l.p.vecs;
  for (uint32_t i0 = threadIdx.x; i0 < items; i0 += kPagedThreads * kPagedItems) {
    R value[kPagedItems];
    R* to[kPagedItems];
    if (FIRST) {
      PagedPlace place[kPagedItems];
      long long slot[kPagedItems];
#pragma unroll
      for (int k = 0; k < kPagedItems; k++) {
        const uint32_t i = i0 + k * kPagedThreads;
        slot[k] = -1;
        if (i >= items) continue;
        place[k] = paged_place(l.p, q0, i);
        slot[k] = l.m.slot[place[k].token];
      }
#pragma unroll
      for (int k = 0; k < kPagedItems; k++) {
        long long row, cache;
        to[k] = nullptr;
        if (!paged_access(l.p, place[k], slot[k], row, cache)) continue;
        value[k] = __ldcs((const R*)(src + (STORE ? row : cache)));
        to[k] = (R*)(dst + (STORE ? cache : row));
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPagedItems; k++) {
        const uint32_t i = i0 + k * kPagedThreads;
        to[k] = nullptr;
        if (i >= items) continue;
        const PagedPlace a = paged_place(l.p, q0, i);
        long long row, cache;
        if (!paged_access(l.p, a, l.m.slot[a.token], row, cache)) continue;
        value[k] = __ldcs((const R*)(src + (STORE ? row : cache)));
        to[k] = (R*)(dst + (STORE ? cache : row));
      }
    }
#pragma unroll
    for (int k = 0; k < kPagedItems; k++)
      if (to[k]) __stcs(to[k], value[k]);
  }
}

// Blocks for an SM up to which a store looks up its slots first: with few blocks the time is the chain of slot and
// row, with many it is how many of them an SM holds (58 registers a thread instead of 48, with narrow accesses 50
// instead of 40).  K and V rows, us in a graph, slots first and one by one:
//   8 heads of 128 bf16       256 rows 2.5, 3.1    8192 rows 13.6, 13.8    65536 rows 87.0, 86.2
//   8 heads of 33 bf16        256 rows 2.1, 2.5    2048 rows 6.6, 6.6      65536 rows 153, 139
// 8192 and 2048 rows are the same number of blocks there, 4096.  Loads: 131072 rows 167, 165.
constexpr int kFirstBlocks = 28;

template <int VB>
cudaError_t paged_typed(const PagedLaunch& l, int numSM, cudaStream_t stream) {
  const dim3 grid((unsigned)((l.p.s.tokens + l.p.perBlock - 1) / l.p.perBlock), l.m.tensors, 1);
  if (!l.m.store) return launch_row_kernel(paged_kernel<VB, false, false>, grid, kPagedThreads, 0, 0, stream, l);
  if ((long long)grid.x * grid.y <= (long long)kFirstBlocks * numSM)
    return launch_row_kernel(paged_kernel<VB, true, true>, grid, kPagedThreads, 0, 0, stream, l);
  return launch_row_kernel(paged_kernel<VB, true, false>, grid, kPagedThreads, 0, 0, stream, l);
}

}  // namespace

// Tokens of a block.
constexpr int kBlockTokens = 1024;
// With the pool updated in place: up to this many tokens a cluster, above two kernels.  Measured, 61 requests:
// 8192 tokens 5.0 against 5.7 us, 16384 tokens 4.8 against 5.7, 32768 tokens 5.6 against 5.7, 131072 tokens 10.9
// against 5.8; 256 requests with one token each 3.3 against 5.2.
constexpr int kClusterTokens = 16384;

// Blocks and threads of the one kernel.
int build_blocks(const PagesShape& s, int most) {
  int blocks = 1;
  while (blocks * 2 <= most && s.maxTokens > blocks * kBlockTokens) blocks *= 2;
  return blocks;
}
int build_threads(const PagesShape& s) { return s.requests > 512 || s.maxTokens > 512 ? 1024 : 512; }

int pages_build_clusters(const PagesShape& s, cudaStream_t stream) {
  if (s.requests > kSharedRequests || s.maxTokens > kClusterTokens) return kMostClusterBlocks;     // two kernels
  const int blocks = build_blocks(s, kMostClusterBlocks);
  return blocks <= kPortableBlocks || cluster_fits(pages_build, blocks, build_threads(s), 8 * (s.requests + 1), stream) ? kMostClusterBlocks
                                                                                                                     : kPortableBlocks;
}

cudaError_t launch_pages_build(const PagesBuild& b, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset,
                               int numSM, int cluster, cudaStream_t stream) {
  const bool inPlace = b.freeList && poolIn == poolOut;
  if (b.s.requests <= kSharedRequests && (!inPlace || b.s.maxTokens <= kClusterTokens)) {
    const int blocks = build_blocks(b.s, inPlace ? cluster : numSM);
    return launch_row_kernel(pages_build, dim3(blocks), build_threads(b.s), 8 * (b.s.requests + 1), inPlace ? blocks : 0, stream, b, poolIn,
                             poolOut, tokenOffset, pageOffset, inPlace);
  }
  const cudaError_t e = launch_row_kernel(pages_scan, dim3(1), 1024, 0, 0, stream, b, poolIn, poolOut, tokenOffset, pageOffset);
  if (e != cudaSuccess) return e;
  const int want = (b.s.maxTokens + kExpandThreads - 1) / kExpandThreads, most = numSM * 8;
  return launch_row_kernel(pages_expand, dim3(want < 1 ? 1 : want < most ? want : most), kExpandThreads, 0, 0, stream, b);
}

cudaError_t launch_paged(const PagedShape& s, const PagedMove& m, int numSM, cudaStream_t stream) {
  if (s.tokens == 0) return cudaSuccess;
  unsigned long long addresses = 0;
  for (int i = 0; i < m.tensors; i++) addresses |= (uintptr_t)m.src[i] | (uintptr_t)m.dst[i];
  const PagedLaunch l{paged_items(s, m.tokenStride, m.headStride, addresses), m};
  switch (l.p.access) {
    case 16: return paged_typed<16>(l, numSM, stream);
    case 8: return paged_typed<8>(l, numSM, stream);
    case 4: return paged_typed<4>(l, numSM, stream);
    case 2: return paged_typed<2>(l, numSM, stream);
    default: return paged_typed<1>(l, numSM, stream);
  }
}

}  // namespace cuttb
