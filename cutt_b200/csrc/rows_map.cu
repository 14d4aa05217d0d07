// The map of rows sorted by expert (cutt_rows_sort).
//
// row(s) = start of s's expert + number of earlier slots of that expert: a stable counting sort.
// Every warp owns a contiguous range of slots; __match_any_sync finds, 32 slots at a time, which
// lanes name the same expert, so one warp-private histogram in shared memory gives each slot its
// rank without atomics: the result does not depend on timing.  Two passes over the slots (count,
// then rank) around a scan over (expert, range).
#include <stdint.h>

#include "kernels.h"
#include "rows.h"

namespace cuttb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// Adds the slots lo .. hi-1 to this warp's histogram.
template <typename I>
__device__ __forceinline__ void warp_count(const I* ids, int lo, int hi, int first, int experts, int* hist) {
  const int lane = threadIdx.x & 31;
  for (int base = lo; base < hi; base += 32) {
    const int i = base + lane;
    const int e = i < hi ? local_expert((long long)ids[i], first, experts) : -1;
    const unsigned same = __match_any_sync(kFull, e);
    if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
  }
}

// Gives the slots lo .. hi-1 their rows; hist[e] is the next row of expert e for this warp.
template <typename I>
__device__ __forceinline__ void warp_rank(const I* ids, int lo, int hi, int first, int experts, int capacity, int* hist,
                                          int* rowOf, int* slotOf) {
  const int lane = threadIdx.x & 31;
  for (int base = lo; base < hi; base += 32) {
    const int i = base + lane;
    const int e = i < hi ? local_expert((long long)ids[i], first, experts) : -1;
    const unsigned same = __match_any_sync(kFull, e);
    int row = -1;
    if (e >= 0) row = hist[e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
    if (row >= capacity) row = -1;
    if (i < hi) {
      rowOf[i] = row;
      if (row >= 0) slotOf[row] = i;
    }
  }
}

// Exclusive prefix sum over the block; `total` is the sum.  s: one int per warp and one more.
__device__ __forceinline__ int block_scan(int v, int* s, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int x = v;
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(kFull, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) s[w] = x;
  __syncthreads();
  if (w == 0) {
    int t = lane < nw ? s[lane] : 0;
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(kFull, t, d);
      if (lane >= d) t += y;
    }
    if (lane < nw) s[lane] = t;
  }
  __syncthreads();
  const int before = w ? s[w - 1] : 0;
  total = s[nw - 1];
  __syncthreads();
  return before + x - v;
}

// Rows of a segment that no slot owns, and rows behind the last segment: slotOf = -1.
__device__ __forceinline__ void fill_gaps(int experts, int capacity, const int* count, const int* offset, int* slotOf,
                                          int block, int blocks) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int e = block * nw + w; e < experts; e += blocks * nw)
    for (int r = offset[e] + count[e] + lane; r < offset[e + 1]; r += 32) slotOf[r] = -1;
  for (int r = offset[experts] + block * blockDim.x + threadIdx.x; r < capacity; r += blocks * blockDim.x) slotOf[r] = -1;
}

// Whole map in one block.  Shared memory: warps * experts histogram words.
template <typename I>
__global__ void __launch_bounds__(1024)
sort_one_block(RowsShape s, const I* __restrict__ ids, int* count, int* offset, int* rowOf, int* slotOf) {
  extern __shared__ int hist[];
  __shared__ int scratch[33];
  const int w = threadIdx.x >> 5, nw = blockDim.x >> 5, E = s.experts;
  const int n = s.tokens * s.choices;
  const int per = ((n + nw - 1) / nw + 31) & ~31;
  const int lo = min(n, w * per), hi = min(n, lo + per);
  for (int i = threadIdx.x; i < nw * E; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  warp_count(ids, lo, hi, s.first, E, hist + w * E);
  __syncthreads();
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int n_e = 0;
    if (e < E)
      for (int k = 0; k < nw; k++) n_e += hist[k * E + e];
    int total;
    const int o = carry + block_scan(align_rows(n_e, s.align), scratch, total);
    carry += total;
    if (e < E) {
      count[e] = held_rows(o, n_e, s.capacity);
      offset[e] = clip_row(o, s.capacity);
      int at = o;
      for (int k = 0; k < nw; k++) {
        const int h = hist[k * E + e];
        hist[k * E + e] = at;
        at += h;
      }
    }
  }
  if (threadIdx.x == 0) offset[E] = clip_row(carry, s.capacity);
  __syncthreads();
  warp_rank(ids, lo, hi, s.first, E, s.capacity, hist + w * E, rowOf, slotOf);
  fill_gaps(E, s.capacity, count, offset, slotOf, 0, 1);
}

template <typename I>
cudaError_t sort_typed(const RowsShape& s, const I* ids, int* count, int* offset, int* rowOf, int* slotOf, cudaStream_t stream) {
  int warps = 32;
  while (warps > 1 && warps * s.experts * 4 > 160 * 1024) warps >>= 1;
  const int smem = warps * s.experts * 4;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(sort_one_block<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  sort_one_block<I><<<1, warps * 32, smem, stream>>>(s, ids, count, offset, rowOf, slotOf);
  count_launch();
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rows_sort(const RowsShape& s, const void* expertOf, int indexBytes, int* count, int* offset,
                             int* rowOf, int* slotOf, int, cudaStream_t stream) {
  if (indexBytes == 4) return sort_typed(s, (const int*)expertOf, count, offset, rowOf, slotOf, stream);
  return sort_typed(s, (const long long*)expertOf, count, offset, rowOf, slotOf, stream);
}

}  // namespace cuttb
