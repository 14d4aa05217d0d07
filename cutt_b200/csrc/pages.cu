// Block tables and slot maps from request lengths (cutt_pages_build), and rows stored into and
// loaded from pages (cutt_pages_store, cutt_pages_load).
#include <stdint.h>

#include "kernels.h"
#include "rows.h"

namespace cuttb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ long long block_scan64(long long v, long long* s, long long& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long x = v;
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(kFull, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) s[w] = x;
  __syncthreads();
  if (w == 0) {
    long long t = lane < nw ? s[lane] : 0;
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(kFull, t, d);
      if (lane >= d) t += y;
    }
    if (lane < nw) s[lane] = t;
  }
  __syncthreads();
  const long long before = w ? s[w - 1] : 0;
  total = s[nw - 1];
  __syncthreads();
  return before + x - v;
}

// Prefix sums of the new tokens and of the pages they take (a block).
__device__ void scan_requests(const PagesBuild& p, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset) {
  __shared__ long long s[33];
  long long tokens = 0, pages = 0;
  int limit = 0, first = 0;
  if (p.freeList) {
    first = clamp_pool(poolIn[0]);
    limit = clamp_pool(poolIn[1]);
    pages = first;
  }
  for (int b0 = 0; b0 < p.s.requests; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    const int n = b < p.s.requests ? max(0, p.added[b]) : 0;
    long long total;
    const long long at = tokens + block_scan64(n, s, total);
    tokens += total;
    if (b < p.s.requests) tokenOffset[b] = saturate(at);
    if (p.freeList) {
      const int g = b < p.s.requests ? pages_taken(p.held[b], n, p.s.pageSize, p.s.tableWidth) : 0;
      const long long f = pages + block_scan64(g, s, total);
      pages += total;
      if (b < p.s.requests) pageOffset[b] = (int)f;   // below 2^31: the table's entries and the pool are at most 2^30
    }
  }
  if (threadIdx.x == 0) {
    tokenOffset[p.s.requests] = saturate(tokens);
    if (p.freeList) {
      pageOffset[p.s.requests] = (int)pages;
      poolOut[0] = min((int)pages, max(first, limit));
      poolOut[1] = poolIn[1];
    }
  }
}

__device__ void expand_requests(const PagesBuild& p, int limit, int block, int blocks) {
  const int stride = blocks * blockDim.x, at = block * blockDim.x + threadIdx.x;
  const int tokens = p.tokenOffset[p.s.requests];
  for (int q = at; q < p.s.maxTokens; q += stride) {
    long long slot = -1;
    if (q < tokens) slot = slot_of_token(p, last_at_or_before(p.tokenOffset, p.s.requests + 1, q), q, limit);
    p.slot[q] = slot;
  }
  if (!p.freeList) return;
  const int end = p.pageOffset[p.s.requests];
  for (int f = p.pageOffset[0] + at; f < end; f += stride)
    take_page(p, last_at_or_before(p.pageOffset, p.s.requests + 1, f), f, limit);
}

__global__ void __launch_bounds__(1024)
pages_one_block(const __grid_constant__ PagesBuild p, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset) {
  scan_requests(p, poolIn, poolOut, tokenOffset, pageOffset);
  __syncthreads();
  expand_requests(p, p.freeList ? clamp_pool(poolOut[1]) : 0, 0, 1);
}

template <int VB> struct Raw;
template <> struct Raw<16> { typedef uint4 T; };
template <> struct Raw<8> { typedef uint2 T; };
template <> struct Raw<4> { typedef uint32_t T; };
template <> struct Raw<2> { typedef uint16_t T; };
template <> struct Raw<1> { typedef uint8_t T; };

struct PagedLaunch {
  PagedShape s;
  PagedMove m;
  FastDiv divPage, divRow, divHead;   // by pageSize, by accesses of a token, by accesses of a head
  int perBlock;                       // tokens of a block
  int vecs;                           // accesses of a token
};

constexpr int kPagedThreads = 256;

// grid.x: groups of perBlock tokens, grid.y: tensors.
template <int VB>
__global__ void __launch_bounds__(kPagedThreads) paged_kernel(const __grid_constant__ PagedLaunch p) {
  typedef typename Raw<VB>::T R;
  const int q0 = blockIdx.x * p.perBlock;
  const int nq = min(p.perBlock, p.s.tokens - q0);
  const unsigned char* src = p.m.src[blockIdx.y];
  unsigned char* dst = p.m.dst[blockIdx.y];
  const uint32_t items = (uint32_t)nq * p.vecs;
  for (uint32_t i = threadIdx.x; i < items; i += kPagedThreads) {
    const uint32_t q = fdiv(i, p.divRow), r = i - q * p.vecs;
    const uint32_t h = fdiv(r, p.divHead), v = r - h * p.divHead.d;
    const long long at = cache_offset(p.s, p.m.slot[q0 + q], p.divPage);
    if (at < 0) continue;
    const long long c = (at + h * p.s.headStride) * p.s.elt + (long long)v * VB;
    const long long x = (long long)(q0 + q) * p.m.tokenStride + h * p.m.headStride + (long long)v * VB;
    if (p.m.store) *(R*)(dst + c) = *(const R*)(src + x);
    else *(R*)(dst + x) = *(const R*)(src + c);
  }
}

template <int VB>
cudaError_t paged_vec(PagedLaunch& p, cudaStream_t stream) {
  const int perHead = p.s.headSize * p.s.elt / VB;
  p.vecs = perHead * p.s.heads;
  p.divHead = make_fastdiv(perHead);
  p.divRow = make_fastdiv(p.vecs);
  p.perBlock = p.vecs >= kPagedThreads ? 1 : kPagedThreads / p.vecs;
  const dim3 grid((unsigned)((p.s.tokens + p.perBlock - 1) / p.perBlock), p.m.tensors, 1);
  paged_kernel<VB><<<grid, kPagedThreads, 0, stream>>>(p);
  count_launch();
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_pages_build(const PagesBuild& b, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset,
                               int, cudaStream_t stream) {
  pages_one_block<<<1, 1024, 0, stream>>>(b, poolIn, poolOut, tokenOffset, pageOffset);
  count_launch();
  return cudaGetLastError();
}

cudaError_t launch_paged(const PagedShape& s, const PagedMove& m, int, cudaStream_t stream) {
  if (s.tokens == 0) return cudaSuccess;
  PagedLaunch p;
  p.s = s;
  p.m = m;
  p.divPage = make_fastdiv(s.pageSize);
  unsigned long long bits = (unsigned long long)s.headSize * s.elt | (unsigned long long)m.tokenStride |
                            (unsigned long long)m.headStride | (unsigned long long)(s.pageStride * s.elt) |
                            (unsigned long long)(s.slotStride * s.elt) | (unsigned long long)(s.headStride * s.elt);
  for (int i = 0; i < m.tensors; i++) bits |= (uintptr_t)m.src[i] | (uintptr_t)m.dst[i];
  switch (access_bytes(bits, s.elt)) {
    case 16: return paged_vec<16>(p, stream);
    case 8: return paged_vec<8>(p, stream);
    case 4: return paged_vec<4>(p, stream);
    case 2: return paged_vec<2>(p, stream);
    default: return paged_vec<1>(p, stream);
  }
}

}  // namespace cuttb
