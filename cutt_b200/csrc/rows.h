// Launch interface of the row operators (rows_map.cu, rows_move.cu, pages.cu).
#pragma once
#include <cuda_runtime.h>

#include "rows_plan.h"

namespace cuttb {

cudaError_t launch_rows_sort(const RowsShape& s, const void* expertOf, int indexBytes, int* count, int* offset,
                             int* rowOf, int* slotOf, int numSM, cudaStream_t stream);

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
                               int numSM, cudaStream_t stream);

struct PagedMove {
  const unsigned char* src[2];
  unsigned char* dst[2];
  long long tokenStride, headStride;   // of the rows, bytes
  const long long* slot;
  int tensors;                         // 1 or 2
  int store;                           // rows to cache, else cache to rows
};
cudaError_t launch_paged(const PagedShape& s, const PagedMove& m, cudaStream_t stream);

// Row plans of the public handle space (rows_api.cu).  Their numbers have the top bit set, which
// cuttPlan's never reach.
constexpr unsigned int kRowsHandleBit = 0x80000000u;
bool rows_destroy(unsigned int handle);
bool rows_describe(unsigned int handle, char* buf, size_t len);

}  // namespace cuttb
