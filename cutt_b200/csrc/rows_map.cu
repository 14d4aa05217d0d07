// The map of rows sorted by expert (cutt_rows_sort).
//
// row(s) = start of s's expert + number of earlier slots of that expert: a stable counting sort.
// Every warp owns a contiguous range of slots and takes 32 of them at a time.  Its lanes set their
// bits in a shared word of their expert, which so holds the lanes that name the same expert; with a
// warp-private histogram that gives each slot its rank among the warp's slots.  Bits and sums do
// not depend on the order of the additions, so the result does not depend on timing.  Scans over
// (expert, warp, block) turn ranks into rows.
// (Other ways to find the lanes: __match_any_sync, which an SM completes once in about 62 cycles -
// 8192 slots of 256 experts took 22 us in one block; a ballot for each bit of the expert's number,
// about 45 instructions for 32 slots.)
#include <cooperative_groups.h>
#include <stdint.h>

#include "rows.h"

namespace cuttb {

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xffffffffu;

// Loads of a warp that are in flight at once: 32 slots each.  One at a time, every 32 slots would
// wait for a round trip to memory.
constexpr int kAhead = 8;

// A slot's expert as device memory has it.  sort_rows reads the indices before its wait for the kernels
// before it.  That the kernel which wrote them has ended and its writes are in device memory (L2) is known all
// the same: sort_count waited for that before it let sort_starts begin, which lets sort_rows begin.  But only
// a kernel's own wait promises that its SM's L1 holds no older copy of a line, so the loads must not be served
// from there: these are coherent at the scope of the device.  Ranks made after the wait instead took 17.6 us
// where these take 12.6 (524288 slots, 256 experts, 64-bit indices; plain loads 13.1).
__device__ __forceinline__ int load_index(const int* p) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ long long load_index(const long long* p) {
  long long v;
  asm volatile("ld.relaxed.gpu.global.s64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

// Experts of the slots base .. base + 32 * kAhead - 1, one of each 32 in a lane; `experts` where
// the slot is dropped or not below hi.
template <typename I>
__device__ __forceinline__ void load_experts(const I* ids, int base, int hi, int first, int experts, int (&e)[kAhead]) {
  const int lane = threadIdx.x & 31;
  I raw[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; k++) {
    const int i = base + k * 32 + lane;
    if (i < hi) raw[k] = load_index(ids + i);
  }
#pragma unroll
  for (int k = 0; k < kAhead; k++) {
    const int i = base + k * 32 + lane;
    const int l = i < hi ? local_expert(raw[k], first, experts) : -1;
    e[k] = l < 0 ? experts : l;
  }
}

// A slot's expert and rank in one word.  13 bits of expert (`experts` itself: dropped), 19 of rank:
// a block has at most 2^19 slots.
constexpr int kRankBits = 19;

// Ranks the slots lo .. hi-1 among this warp's slots of their expert; hist: this warp's, zero at
// first, the counts at the end; lanes: this warp's words for the lanes of an expert, zero before and
// after.
template <typename I>
__device__ __forceinline__ void warp_rank(const I* ids, int lo, int hi, int first, int experts, int* hist, unsigned* lanes,
                                          unsigned* packed) {
  const int lane = threadIdx.x & 31;
  for (int base = lo; base < hi; base += 32 * kAhead) {
    int e[kAhead];
    load_experts(ids, base, hi, first, experts, e);
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const int i = base + k * 32 + lane;
      if (base + k * 32 >= hi) break;
      const bool live = e[k] < experts;
      if (live) atomicOr(&lanes[e[k]], 1u << lane);
      __syncwarp();
      const unsigned same = live ? lanes[e[k]] : 0;
      const int before = live ? hist[e[k]] : 0;
      __syncwarp();
      if (live && lane == __ffs(same) - 1) {
        hist[e[k]] = before + __popc(same);
        lanes[e[k]] = 0;
      }
      __syncwarp();
      if (i < hi) packed[i - lo] = ((unsigned)e[k] << kRankBits) | (unsigned)(before + __popc(same & ((1u << lane) - 1)));
    }
  }
}

// Exclusive prefix sums of pairs over the block; `total` is the sum.  s: one pair per warp.
__device__ __forceinline__ int2 block_scan(int2 v, int2* s, int2& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int2 x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(kFull, x.x, d), b = __shfl_up_sync(kFull, x.y, d);
    if (lane >= d) { x.x += a; x.y += b; }
  }
  if (lane == 31) s[w] = x;
  __syncthreads();
  int2 y = lane < nw ? s[lane] : make_int2(0, 0);      // every warp scans the warps' sums
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(kFull, y.x, d), b = __shfl_up_sync(kFull, y.y, d);
    if (lane >= d) { y.x += a; y.y += b; }
  }
  total.x = __shfl_sync(kFull, y.x, nw - 1);
  total.y = __shfl_sync(kFull, y.y, nw - 1);
  const int at = w > 0 ? w - 1 : 0;
  const int bx = __shfl_sync(kFull, y.x, at), by = __shfl_sync(kFull, y.y, at);
  __syncthreads();
  return make_int2((w > 0 ? bx : 0) + x.x - v.x, (w > 0 ? by : 0) + x.y - v.y);
}

// Rows of a segment that no slot owns, and rows behind the last segment: slotOf = -1.
__device__ __forceinline__ void fill_gaps(int experts, int capacity, const int* count, const int* offset, int* slotOf,
                                          int block, int blocks) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int e = block * nw + w; e < experts; e += blocks * nw)
    for (int r = offset[e] + count[e] + lane; r < offset[e + 1]; r += 32) slotOf[r] = -1;
  for (int r = offset[experts] + block * blockDim.x + threadIdx.x; r < capacity; r += blocks * blockDim.x) slotOf[r] = -1;
}

__device__ __forceinline__ void warp_range(int lo, int hi, int& from, int& to) {
  const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int per = ((hi - lo + nw - 1) / nw + 31) & ~31;
  from = min(hi, lo + w * per);
  to = min(hi, from + per);
}

// Shared memory of a block that ranks `slots` slots.
struct Ranked {
  unsigned* packed;     // a word for each slot
  unsigned* sorted;     // a word for each slot
  int* hist;            // warps x experts
  unsigned* lanes;      // warps x experts
  int* total;           // experts: slots of this block
  int* shift;           // experts: row of a slot less its place among the block's sorted slots
};
__device__ __forceinline__ Ranked carve(int* smem, int slots, int warps, int experts) {
  Ranked r;
  r.packed = (unsigned*)smem;
  r.sorted = r.packed + slots;
  r.hist = (int*)(r.sorted + slots);
  r.lanes = (unsigned*)(r.hist + warps * experts);
  r.total = (int*)(r.lanes + warps * experts);
  r.shift = r.total + experts;
  return r;
}

// Ranks the block's slots lo .. hi-1 and sums the warps' counts: hist becomes, for every warp, the
// slots of the warps before it, total the block's counts.
template <typename I>
__device__ void rank_block(const RowsShape& s, const I* ids, int lo, int hi, const Ranked& r) {
  const int w = threadIdx.x >> 5, nw = blockDim.x >> 5, E = s.experts;
  int from, to;
  warp_range(lo, hi, from, to);
  for (int i = threadIdx.x; i < 2 * nw * E; i += blockDim.x) r.hist[i] = 0;      // and lanes
  __syncthreads();
  warp_rank(ids, from, to, s.first, E, r.hist + w * E, r.lanes + w * E, r.packed + (from - lo));
  __syncthreads();
  // one thread for an expert walks over the warps; the loads do not wait for one another
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int at = 0;
#pragma unroll 8
    for (int k = 0; k < nw; k++) {
      const int n = r.hist[k * E + e];
      r.hist[k * E + e] = at;
      at += n;
    }
    r.total[e] = at;
  }
  __syncthreads();
}

// Writes the rows.  shift[e] + place among the block's sorted slots = row, and start[e] (left in
// total) is the place of the block's first slot of expert e.  The slots are sorted in shared memory
// first: written as they come, every lane of a warp would write a line of its own.
__device__ void write_block(const RowsShape& s, int lo, int hi, const Ranked& r, int live, int* rowOf, int* slotOf) {
  const int E = s.experts;
  int from, to;
  warp_range(lo, hi, from, to);
  const int* hist = r.hist + (threadIdx.x >> 5) * E;
  for (int i = from - lo + (threadIdx.x & 31); i < to - lo; i += 32) {
    const unsigned p = r.packed[i];
    const int e = p >> kRankBits;
    int row = -1;
    if (e < E) {
      const int place = r.total[e] + hist[e] + (int)(p & ((1u << kRankBits) - 1));
      row = r.shift[e] + place;
      if (row >= s.capacity) row = -1;
      r.sorted[place] = ((unsigned)e << kRankBits) | (unsigned)i;
    }
    rowOf[lo + i] = row;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < live; k += blockDim.x) {
    const unsigned p = r.sorted[k];
    const int row = r.shift[p >> kRankBits] + k;
    if (row < s.capacity) slotOf[row] = lo + (int)(p & ((1u << kRankBits) - 1));
  }
}

// The map in one cluster of 1 to kMostClusterBlocks blocks: the blocks read one another's counts through
// distributed shared memory, so there is one launch and no workspace.
template <typename I>
__global__ void __launch_bounds__(1024)
sort_cluster(RowsShape s, const I* ids, int slots, int* count, int* offset, int* rowOf, int* slotOf) {
  extern __shared__ int smem[];
  __shared__ int2 scratch[32];
  begin_row_kernel();
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = gridDim.x, me = blockIdx.x, E = s.experts;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int n = s.tokens * s.choices;
  const int lo = min(n, me * slots), hi = min(n, lo + slots);
  const Ranked r = carve(smem, slots, nw, E);
  int* mine = r.shift + E;           // this block's counts, as the other blocks read them
  int* gapFrom = mine + E;           // rows of each segment that no slot owns
  int* gapTo = gapFrom + E;
  rank_block(s, ids, lo, hi, r);
  for (int e = threadIdx.x; e < E; e += blockDim.x) mine[e] = r.total[e];
  cluster.sync();
  int2 carry = make_int2(0, 0);
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int n_e = 0, before = 0, own = 0;
    if (e < E) {
      own = mine[e];
      int c[kMostClusterBlocks];         // all reads at once: one after the other each waits for its round trip
#pragma unroll
      for (int b = 0; b < kMostClusterBlocks; b++) c[b] = b < blocks ? cluster.map_shared_rank(mine, b)[e] : 0;
#pragma unroll
      for (int b = 0; b < kMostClusterBlocks; b++) {
        if (b < me) before += c[b];
        n_e += c[b];
      }
    }
    int2 total;
    const int2 at = block_scan(make_int2(align_rows(n_e, s.align), own), scratch, total);
    const int o = carry.x + at.x, place = carry.y + at.y;
    carry.x += total.x;
    carry.y += total.y;
    if (e < E) {
      r.total[e] = place;
      r.shift[e] = o + before - place;
      if (me == 0) {
        count[e] = held_rows(o, n_e, s.capacity);
        offset[e] = clip_row(o, s.capacity);
      }
      gapFrom[e] = clip_row(o + n_e, s.capacity);
      gapTo[e] = clip_row(o + align_rows(n_e, s.align), s.capacity);
    }
  }
  const int end = clip_row(carry.x, s.capacity);
  if (me == 0 && threadIdx.x == 0) offset[E] = end;
  __syncthreads();
  write_block(s, lo, hi, r, carry.y, rowOf, slotOf);
  if (s.align > 1)
    for (int e = me * nw + w; e < E; e += blocks * nw)
      for (int k = gapFrom[e] + lane; k < gapTo[e]; k += 32) slotOf[k] = -1;
  for (int k = end + me * blockDim.x + threadIdx.x; k < s.capacity; k += blocks * blockDim.x) slotOf[k] = -1;
  cluster.sync();                    // no block leaves while another reads its counts
}

// The map in three kernels over chunks of slots: counts of each chunk, starts of each (chunk,
// expert), rows.  The counts and starts of chunk b lie in the first `experts` words of the part of
// rowOf that chunk b's slots own (a chunk has at least that many): the last kernel reads them
// before it writes its rows there, so the map needs no workspace.
constexpr int kChunkThreads = 512;

__device__ __forceinline__ void chunk_range(int n, int chunk, int chunks, int b, int& lo, int& hi) {
  lo = b * chunk;
  hi = b == chunks - 1 ? n : lo + chunk;
}

template <typename I>
__global__ void __launch_bounds__(kChunkThreads)
sort_count(RowsShape s, const I* ids, int* rowOf, int chunk, int chunks) {
  extern __shared__ int hist[];
  begin_row_kernel();
  const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int lo, hi;
  chunk_range(s.tokens * s.choices, chunk, chunks, blockIdx.x, lo, hi);
  for (int e = threadIdx.x; e < s.experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  // counts do not depend on the order of these additions
  for (int base = lo + w * 32 * kAhead; base < hi; base += nw * 32 * kAhead) {
    int e[kAhead];
    load_experts(ids, base, hi, s.first, s.experts, e);
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (e[k] < s.experts) atomicAdd(&hist[e[k]], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < s.experts; e += blockDim.x) rowOf[lo + e] = hist[e];
}

// A cluster of kStartBlocks blocks.  Each takes a part of the experts; its threads form groups with
// a part of the chunks each and a thread for every expert of the block's.  One block would read
// and write the whole table by itself (256 chunks x 256 experts: 0.25 MB twice, about 8 us).
constexpr int kStartBlocks = 8;
constexpr int kBatch = 16;               // loads of a thread in flight at once
__device__ __forceinline__ void load_batch(const int* p, int b, int end, int chunk, int (&n)[kBatch]) {
#pragma unroll
  for (int k = 0; k < kBatch; k++) n[k] = b + k < end ? p[(long long)(b + k) * chunk] : 0;
}
constexpr int kMostPart = (kRowsMaxExperts + kStartBlocks - 1) / kStartBlocks;

__global__ void __cluster_dims__(kStartBlocks, 1, 1) __launch_bounds__(kChunkThreads)
sort_starts(RowsShape s, int* count, int* offset, int* rowOf, int chunk, int chunks) {
  __shared__ int part[kChunkThreads];
  __shared__ int total[kMostPart];       // of this block's experts
  __shared__ int start[kMostPart];
  __shared__ int2 scratch[32];
  cg::cluster_group cluster = cg::this_cluster();
  // the last kernel may start its ranks: the inputs are complete, sort_count saw to that (load_index)
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  const int E = s.experts, own = (E + kStartBlocks - 1) / kStartBlocks;
  const int e0 = blockIdx.x * own, e1 = min(E, e0 + own);
  int wide = 1;                          // threads of a group: experts of this block, at most the block
  while (wide < own && wide < kChunkThreads) wide <<= 1;
  const int groups = kChunkThreads / wide, g = threadIdx.x / wide, col = threadIdx.x % wide;
  const int per = (chunks + groups - 1) / groups;
  const int b0 = min(chunks, g * per), b1 = min(chunks, b0 + per);
  const int e = e0 + col;                // own <= kMostPart = kChunkThreads: one pass
  int sum = 0, n[kBatch];
  if (e < e1)
    for (int b = b0; b < b1; b += kBatch) {
      load_batch(rowOf + e, b, b1, chunk, n);
#pragma unroll
      for (int k = 0; k < kBatch; k++) sum += n[k];
    }
  part[threadIdx.x] = sum;
  __syncthreads();
  int before = 0;
  if (e < e1) {
    int all = 0;
#pragma unroll 8
    for (int k = 0; k < groups; k++) {
      const int p = part[k * wide + col];
      if (k < g) before += p;
      all += p;
    }
    if (g == 0) total[col] = all;
  }
  cluster.sync();
  int carry = 0;
  for (int f0 = 0; f0 < E; f0 += kChunkThreads) {
    const int f = f0 + threadIdx.x;
    const int n_f = f < E ? cluster.map_shared_rank(total, f / own)[f % own] : 0;
    int2 sum2;
    const int o = carry + block_scan(make_int2(align_rows(n_f, s.align), 0), scratch, sum2).x;
    carry += sum2.x;
    if (f >= e0 && f < e1) {
      start[f - e0] = o;
      count[f] = held_rows(o, n_f, s.capacity);
      offset[f] = clip_row(o, s.capacity);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offset[E] = clip_row(carry, s.capacity);
  __syncthreads();
  if (e < e1) {
    int at = start[col] + before;
    for (int b = b0; b < b1; b += kBatch) {
      if (b1 - b0 > kBatch) load_batch(rowOf + e, b, b1, chunk, n);     // else they are still there
#pragma unroll
      for (int k = 0; k < kBatch; k++) {
        if (b + k < b1) rowOf[(long long)(b + k) * chunk + e] = at;
        at += n[k];
      }
    }
  }
  cluster.sync();                        // no block leaves while another reads its counts
}

template <typename I>
__global__ void __launch_bounds__(1024)
sort_rows(RowsShape s, const I* ids, const int* count, const int* offset, int* rowOf, int* slotOf, int chunk,
          int chunks, int slots) {
  extern __shared__ int smem[];
  __shared__ int2 scratch[32];
  const int nw = blockDim.x >> 5, E = s.experts;
  int lo, hi;
  chunk_range(s.tokens * s.choices, chunk, chunks, blockIdx.x, lo, hi);
  const Ranked r = carve(smem, slots, nw, E);
  rank_block(s, ids, lo, hi, r);         // of the kernels' outputs none is needed yet; inputs: load_index
  begin_row_kernel();
  int carry = 0;
  for (int e0 = 0; e0 < E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int2 total;
    const int place = carry + block_scan(make_int2(e < E ? r.total[e] : 0, 0), scratch, total).x;
    carry += total.x;
    if (e < E) {
      r.total[e] = place;
      r.shift[e] = rowOf[lo + e] - place;
    }
  }
  __syncthreads();
  write_block(s, lo, hi, r, carry, rowOf, slotOf);
  fill_gaps(E, s.capacity, count, offset, slotOf, blockIdx.x, gridDim.x);
}

static_assert(kMostSortWords * 4 <= kRowSharedLimit, "every call's shared memory is within the limit that all calls set");

template <typename I>
cudaError_t sort_typed(const RowsShape& s, const I* ids, int* count, int* offset, int* rowOf, int* slotOf, int numSM,
                       int cluster, cudaStream_t stream) {
  const int n = s.tokens * s.choices, E = s.experts;
  const SortShape c = sort_shape(n, E, cluster);
  if (c.blocks)
    return launch_row_kernel(sort_cluster<I>, dim3(c.blocks), c.warps * 32, c.words * 4, c.blocks, stream, s, ids, c.slots, count, offset,
                             rowOf, slotOf);
  // one chunk for an SM: more of them are more rows of the table of counts (524288 slots: 148 chunks
  // 12.4 us, 296 chunks 16.6)
  int chunk = (n + numSM - 1) / numSM;
  if (chunk < E) chunk = E;
  if (chunk > 8192) chunk = 8192;
  chunk = (chunk + 31) & ~31;
  int chunks = n / chunk;
  if (chunks == 0 || n - chunks * chunk >= E) chunks++;    // else the last one takes the rest
  const int slots = (chunk + E + 31) & ~31;
  cudaError_t e = launch_row_kernel(sort_count<I>, dim3(chunks), kChunkThreads, E * 4, 0, stream, s, ids, rowOf, chunk, chunks);
  if (e != cudaSuccess) return e;
  e = launch_row_kernel(sort_starts, dim3(kStartBlocks), kChunkThreads, 0, 0, stream, s, count, offset, rowOf, chunk, chunks);
  if (e != cudaSuccess) return e;
  const int warps = warps_for(slots, E, kSortWarps);
  return launch_row_kernel(sort_rows<I>, dim3(chunks), warps * 32, ranked_words(slots, warps, E) * 4, 0, stream, s, ids, count,
                           offset, rowOf, slotOf, chunk, chunks, slots);
}

}  // namespace

int rows_sort_clusters(const RowsShape& s, cudaStream_t stream) {
  const SortShape c = sort_shape(s.tokens * s.choices, s.experts, kMostClusterBlocks);
  if (c.blocks <= kPortableBlocks) return kMostClusterBlocks;
  return cluster_fits(sort_cluster<int>, c.blocks, c.warps * 32, c.words * 4, stream) &&
                 cluster_fits(sort_cluster<long long>, c.blocks, c.warps * 32, c.words * 4, stream)
             ? kMostClusterBlocks
             : kPortableBlocks;
}

cudaError_t launch_rows_sort(const RowsShape& s, const void* expertOf, int indexBytes, int* count, int* offset,
                             int* rowOf, int* slotOf, int numSM, int cluster, cudaStream_t stream) {
  if (indexBytes == 4) return sort_typed(s, (const int*)expertOf, count, offset, rowOf, slotOf, numSM, cluster, stream);
  return sort_typed(s, (const long long*)expertOf, count, offset, rowOf, slotOf, numSM, cluster, stream);
}

}  // namespace cuttb
