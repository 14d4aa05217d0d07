// C entry points of the row operators (include/cutt_rows.h): plan table, checks, launches.
//
// Order of the checks in every call: handle, arguments, device.  The arguments are checked without
// touching the device, so a refusal costs nothing and leaves no CUDA error behind.
#include "../../include/cutt_rows.h"

#include <cstdio>
#include <memory>
#include <mutex>
#include <new>
#include <unordered_map>

#include "../../include/cutt.h"
#include "kernels.h"
#include "rows.h"

namespace cuttb {

namespace {

enum Kind { kRows, kPages, kPaged };

struct Plan {
  Kind kind;
  int device = 0;
  int numSM = 0;
  int cluster = 0;         // blocks of the largest cluster that its calls may use
  cudaStream_t stream = 0;
  RowsShape rows{};
  PagesShape pages{};
  PagedShape paged{};
};

std::mutex g_lock;
// shared: a call keeps its plan alive while it launches, whoever destroys the handle meanwhile
std::unordered_map<unsigned int, std::shared_ptr<const Plan>> g_table;
unsigned int g_next = 0;

int add_plan(unsigned int* handle, Plan& p, void* stream) {
  p.stream = (cudaStream_t)stream;
  if (cudaGetDevice(&p.device) != cudaSuccess ||
      cudaDeviceGetAttribute(&p.numSM, cudaDevAttrMultiProcessorCount, p.device) != cudaSuccess) {
    cudaGetLastError();
    return CUTT_INTERNAL_ERROR;
  }
  if (p.kind == kRows) p.cluster = rows_sort_clusters(p.rows, p.stream);
  if (p.kind == kPages) p.cluster = pages_build_clusters(p.pages, p.stream);
  try {
    std::shared_ptr<const Plan> q = std::make_shared<Plan>(p);
    std::lock_guard<std::mutex> lk(g_lock);
    if (g_next >= kRowsHandleBit - 1) return CUTT_INTERNAL_ERROR;      // 0xffffffff stays free
    const unsigned int h = g_next | kRowsHandleBit;
    g_table[h] = std::move(q);
    g_next++;
    *handle = h;
  } catch (...) {
    return CUTT_INTERNAL_ERROR;
  }
  return CUTT_SUCCESS;
}

std::shared_ptr<const Plan> find_plan(unsigned int handle, Kind kind) {
  std::lock_guard<std::mutex> lk(g_lock);
  auto it = g_table.find(handle);
  if (it == g_table.end() || it->second->kind != kind) return nullptr;
  return it->second;
}

int check_device(const Plan& p) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return CUTT_INTERNAL_ERROR; }
  return dev == p.device ? CUTT_SUCCESS : CUTT_INVALID_DEVICE;
}

int result(cudaError_t e) {
  if (e == cudaSuccess) return CUTT_SUCCESS;
  cudaGetLastError();        // reported here, not by the caller's next CUDA call
  return CUTT_INTERNAL_ERROR;
}

int move_rows(unsigned int handle, const RowsMoveArgs& a) {
  const std::shared_ptr<const Plan> p = find_plan(handle, kRows);
  if (!p) return CUTT_INVALID_PLAN;
  const RowsShape& s = p->rows;
  if (check_rows_move(s, a)) return CUTT_INVALID_PARAMETER;
  const int rc = check_device(*p);
  if (rc != CUTT_SUCCESS) return rc;
  const long long elt = rows_element_bytes(s.type);
  RowsMove m{};
  m.token = (const unsigned char*)a.token;
  m.row = (const unsigned char*)a.row;
  m.other = (const unsigned char*)a.other;
  m.tokenStride = a.tokenStride * elt;
  m.rowStride = a.rowStride * elt;
  m.otherStride = a.other ? a.otherStride * elt : 0;
  m.rowOf = a.rowOf;
  m.count = a.count;
  m.offset = a.offset;
  m.weight = a.weight;
  m.dweight = const_cast<float*>(a.dweight);
  m.tokens = s.tokens;
  m.choices = s.choices;
  m.experts = s.experts;
  m.capacity = s.capacity;
  m.width = s.width;
  m.type = s.type;
  return result(a.rowsOut ? launch_rows_scatter(m, s.align, p->numSM, p->stream) : launch_rows_gather(m, p->numSM, p->stream));
}

}  // namespace

bool rows_destroy(unsigned int handle) {
  std::shared_ptr<const Plan> last;    // freed outside the lock
  std::lock_guard<std::mutex> lk(g_lock);
  auto it = g_table.find(handle);
  if (it == g_table.end()) return false;
  last = it->second;
  g_table.erase(it);
  return true;
}

bool rows_describe(unsigned int handle, char* buf, size_t len) {
  std::shared_ptr<const Plan> p;
  {
    std::lock_guard<std::mutex> lk(g_lock);
    auto it = g_table.find(handle);
    if (it == g_table.end()) return false;
    p = it->second;
  }
  static const char* const types[] = {"bytes", "f16", "bf16", "f32"};
  if (p->kind == kRows)
    snprintf(buf, len, "{\"method\": \"rows\", \"tokens\": %d, \"choices\": %d, \"experts\": %d, \"first\": %d, \"align\": %d, "
             "\"capacity\": %d, \"width\": %d, \"type\": \"%s\", \"cluster\": %d}", p->rows.tokens, p->rows.choices, p->rows.experts,
             p->rows.first, p->rows.align, p->rows.capacity, p->rows.width, types[p->rows.type], p->cluster);
  else if (p->kind == kPages)
    snprintf(buf, len, "{\"method\": \"pages\", \"requests\": %d, \"page_size\": %d, \"table_width\": %d, \"max_tokens\": %d, "
             "\"cluster\": %d}", p->pages.requests, p->pages.pageSize, p->pages.tableWidth, p->pages.maxTokens, p->cluster);
  else
    snprintf(buf, len, "{\"method\": \"paged rows\", \"tokens\": %d, \"heads\": %d, \"head_size\": %d, \"element\": %d, "
             "\"pages\": %d, \"page_size\": %d}", p->paged.tokens, p->paged.heads, p->paged.headSize, p->paged.elt,
             p->paged.pages, p->paged.pageSize);
  return true;
}

}  // namespace cuttb

using namespace cuttb;

extern "C" {

int cutt_rows_plan(unsigned int* handle, int tokens, int choices, int experts, int firstExpert, int align, int capacity,
                   int width, int type, void* stream) {
  Plan p;
  p.kind = kRows;
  p.rows = RowsShape{tokens, choices, experts, firstExpert, align, capacity, width, type};
  if (!handle || check_rows_shape(p.rows)) return CUTT_INVALID_PARAMETER;
  return add_plan(handle, p, stream);
}

int cutt_rows_sort(unsigned int handle, const void* expertOf, size_t sizeofIndex, int* count, int* offset, int* rowOf,
                   int* slotOf) {
  const std::shared_ptr<const Plan> p = find_plan(handle, kRows);
  if (!p) return CUTT_INVALID_PLAN;
  if (check_rows_sort(p->rows, expertOf, sizeofIndex, count, offset, rowOf, slotOf)) return CUTT_INVALID_PARAMETER;
  const int rc = check_device(*p);
  if (rc != CUTT_SUCCESS) return rc;
  return result(launch_rows_sort(p->rows, expertOf, (int)sizeofIndex, count, offset, rowOf, slotOf, p->numSM, p->cluster, p->stream));
}

int cutt_rows_dispatch(unsigned int handle, const void* x, long long xStride, const int* rowOf, const int* count,
                       const int* offset, const float* weight, void* y, long long yStride) {
  return move_rows(handle, RowsMoveArgs{x, xStride, y, yStride, rowOf, count, offset, weight, nullptr, 0, nullptr, true, true});
}

int cutt_rows_combine(unsigned int handle, const void* y, long long yStride, const int* rowOf, const float* weight,
                      void* out, long long outStride) {
  return move_rows(handle, RowsMoveArgs{out, outStride, y, yStride, rowOf, nullptr, nullptr, weight, nullptr, 0, nullptr, false, false});
}

int cutt_rows_dispatch_grad(unsigned int handle, const void* dy, long long dyStride, const int* rowOf, const float* weight,
                            const void* x, long long xStride, void* dx, long long dxStride, float* dweight) {
  return move_rows(handle, RowsMoveArgs{dx, dxStride, dy, dyStride, rowOf, nullptr, nullptr, weight, x, xStride, dweight, false, false});
}

int cutt_rows_combine_grad(unsigned int handle, const void* dout, long long doutStride, const int* rowOf, const int* count,
                           const int* offset, const float* weight, const void* y, long long yStride, void* dy,
                           long long dyStride, float* dweight) {
  return move_rows(handle, RowsMoveArgs{dout, doutStride, dy, dyStride, rowOf, count, offset, weight, y, yStride, dweight, true, true});
}

int cutt_pages_plan(unsigned int* handle, int requests, int pageSize, int tableWidth, int maxTokens, void* stream) {
  Plan p;
  p.kind = kPages;
  p.pages = PagesShape{requests, pageSize, tableWidth, maxTokens, FastDiv()};
  if (!handle || check_pages_shape(p.pages)) return CUTT_INVALID_PARAMETER;
  p.pages.divPage = make_fastdiv(pageSize);
  return add_plan(handle, p, stream);
}

int cutt_pages_build(unsigned int handle, const int* held, const int* added, const int* freeList, const int* poolIn,
                     int* poolOut, int* table, long long tableStride, int* tokenOffset, int* pageOffset, long long* slot) {
  const std::shared_ptr<const Plan> p = find_plan(handle, kPages);
  if (!p) return CUTT_INVALID_PLAN;
  if (check_pages_build(p->pages, held, added, freeList, poolIn, poolOut, table, tableStride, tokenOffset, pageOffset, slot))
    return CUTT_INVALID_PARAMETER;
  const int rc = check_device(*p);
  if (rc != CUTT_SUCCESS) return rc;
  const PagesBuild b{p->pages, held, added, freeList, poolOut, table, tableStride, tokenOffset, pageOffset, slot};
  return result(launch_pages_build(b, poolIn, poolOut, tokenOffset, pageOffset, p->numSM, p->cluster, p->stream));
}

int cutt_pages_plan_rows(unsigned int* handle, int tokens, int heads, int headSize, size_t sizeofType, int pages,
                         int pageSize, long long pageStride, long long slotStride, long long headStride, void* stream) {
  Plan p;
  p.kind = kPaged;
  p.paged = PagedShape{tokens, heads, headSize, sizeofType <= 8 ? (int)sizeofType : 0, pages, pageSize, pageStride, slotStride, headStride};
  if (!handle || check_paged_shape(p.paged)) return CUTT_INVALID_PARAMETER;
  return add_plan(handle, p, stream);
}

static int move_paged(unsigned int handle, const void* k, const void* v, long long tokenStride, long long headStride,
                      const long long* slot, const void* kCache, const void* vCache, bool store) {
  const std::shared_ptr<const Plan> p = find_plan(handle, kPaged);
  if (!p) return CUTT_INVALID_PLAN;
  const PagedShape& s = p->paged;
  if (check_paged_move(s, k, v, tokenStride, headStride, slot, kCache, vCache, !store)) return CUTT_INVALID_PARAMETER;
  const int rc = check_device(*p);
  if (rc != CUTT_SUCCESS) return rc;
  PagedMove m{};
  const void* rows[2] = {k, v};
  const void* caches[2] = {kCache, vCache};
  m.tensors = v ? 2 : 1;
  for (int i = 0; i < m.tensors; i++) {
    m.src[i] = (const unsigned char*)(store ? rows[i] : caches[i]);
    m.dst[i] = (unsigned char*)const_cast<void*>(store ? caches[i] : rows[i]);
  }
  m.tokenStride = tokenStride * s.elt;
  m.headStride = headStride * s.elt;
  m.slot = slot;
  m.store = store ? 1 : 0;
  return result(launch_paged(s, m, p->numSM, p->stream));
}

int cutt_pages_store(unsigned int handle, const void* k, const void* v, long long tokenStride, long long headStride,
                     const long long* slot, void* kCache, void* vCache) {
  return move_paged(handle, k, v, tokenStride, headStride, slot, kCache, vCache, true);
}

int cutt_pages_load(unsigned int handle, const void* kCache, const void* vCache, const long long* slot, void* k, void* v,
                    long long tokenStride, long long headStride) {
  return move_paged(handle, k, v, tokenStride, headStride, slot, kCache, vCache, false);
}

}  // extern "C"
