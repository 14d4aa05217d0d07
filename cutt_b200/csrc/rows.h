// Launch interface of the row operators (rows_map.cu, rows_move.cu, pages.cu).
#pragma once
#include <cuda_runtime.h>

#include "kernels.h"
#include "rows_plan.h"

namespace cuttb {

// Launch of a row operator's kernel.  The kernels of a step follow one another in microseconds, so each
// is launched while the one before it still runs (programmatic dependent launch) and waits, as its first
// statement, for that one's end: begin_row_kernel.  It lets the next kernel start in turn only then, so
// whatever precedes this kernel in the stream is done before the next one begins.  Within the map of three
// kernels (rows_map.cu) two differ: sort_starts lets sort_rows start before its own wait, and sort_rows
// ranks the map's inputs before its wait, with loads that allow that (load_index there).  Inputs are read
// with coherent loads (no __restrict__): a line may have come into the cache before the kernel that writes
// it ended.
// `cluster`: blocks of a cluster, 0 for none.
// The limit of a kernel's shared memory belongs to the process, and calls of several threads need different
// sizes of one kernel: every call sets the same limit, which is enough for all of them.
constexpr int kRowSharedLimit = 220 * 1024;   // an SM's 227 KB less what the kernels declare statically
template <typename... P, typename... A>
cudaError_t launch_row_kernel(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, A... args) {
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSharedLimit);
    if (e != cudaSuccess) return e;
  }
  if (cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute attr[2] = {};
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  c.attrs = attr;
  attr[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[c.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  if (cluster > 1) {
    attr[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[c.numAttrs].val.clusterDim.x = cluster;
    attr[c.numAttrs].val.clusterDim.y = 1;
    attr[c.numAttrs++].val.clusterDim.z = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, P(args)...);
  if (e == cudaSuccess) count_launch();
  return e;
}

// Whether the device, or the part of it that the stream's context has (a green context), can hold a cluster of
// this launch.  Clusters of up to kPortableBlocks blocks fit everywhere; larger ones are asked for when the plan
// is made.
template <typename... P>
bool cluster_fits(void (*kernel)(P...), int blocks, int threads, size_t smem, cudaStream_t stream) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(blocks);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  c.attrs = &attr;
  c.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSharedLimit) == cudaSuccess &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
      cudaOccupancyMaxActiveClusters(&n, kernel, &c) == cudaSuccess)
    return n > 0;
  cudaGetLastError();
  return false;
}

#ifdef __CUDACC__
__device__ __forceinline__ void begin_row_kernel() {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
}
#endif

// `cluster`: most blocks of a cluster, as rows_sort_clusters (pages_build_clusters) says for the plan's stream.
int rows_sort_clusters(const RowsShape& s, cudaStream_t stream);
int pages_build_clusters(const PagesShape& s, cudaStream_t stream);
cudaError_t launch_rows_sort(const RowsShape& s, const void* expertOf, int indexBytes, int* count, int* offset,
                             int* rowOf, int* slotOf, int numSM, int cluster, cudaStream_t stream);

// One row to its slots' rows (dispatch, combine_grad) and the sum of its slots' rows (combine,
// dispatch_grad).  token / row: the tensors of the two sides, whichever is written.
struct RowsMove {
  const unsigned char* token;
  const unsigned char* row;
  const unsigned char* other;
  long long tokenStride, rowStride, otherStride;   // bytes
  const int* rowOf;
  const int* count;
  const int* offset;
  const float* weight;
  float* dweight;
  int tokens, choices, experts, capacity, width, type;
};
cudaError_t launch_rows_scatter(const RowsMove& m, int align, int numSM, cudaStream_t stream);
cudaError_t launch_rows_gather(const RowsMove& m, int numSM, cudaStream_t stream);

cudaError_t launch_pages_build(const PagesBuild& b, const int* poolIn, int* poolOut, int* tokenOffset, int* pageOffset,
                               int numSM, int cluster, cudaStream_t stream);

struct PagedMove {
  const unsigned char* src[2];
  unsigned char* dst[2];
  long long tokenStride, headStride;   // of the rows, bytes
  const long long* slot;
  int tensors;                         // 1 or 2
  int store;                           // rows to cache, else cache to rows
};
cudaError_t launch_paged(const PagedShape& s, const PagedMove& m, int numSM, cudaStream_t stream);

// Row plans of the public handle space (rows_api.cu).  Their numbers have the top bit set, which
// cuttPlan's never reach.
constexpr unsigned int kRowsHandleBit = 0x80000000u;
bool rows_destroy(unsigned int handle);
bool rows_describe(unsigned int handle, char* buf, size_t len);

}  // namespace cuttb
