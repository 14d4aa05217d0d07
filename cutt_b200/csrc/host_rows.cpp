// Test-only: the argument checks and the index arithmetic of the row operators on the host.
#include <string.h>

#include "rows_plan.h"

using namespace cuttb;

extern "C" {

int cutt_hostcheck_rows_shape(int tokens, int choices, int experts, int first, int align, int capacity, int width, int type) {
  return check_rows_shape(RowsShape{tokens, choices, experts, first, align, capacity, width, type});
}

int cutt_hostcheck_pages_shape(int requests, int pageSize, int tableWidth, int maxTokens) {
  return check_pages_shape(PagesShape{requests, pageSize, tableWidth, maxTokens, FastDiv()});
}

int cutt_hostcheck_paged_shape(int tokens, int heads, int headSize, int elt, int pages, int pageSize, long long pageStride,
                               long long slotStride, long long headStride) {
  return check_paged_shape(PagedShape{tokens, heads, headSize, elt, pages, pageSize, pageStride, slotStride, headStride});
}

// The checks of a call on addresses that are never read.
int cutt_hostcheck_rows_sort(const int* shape, const void* expertOf, size_t sizeofIndex, const void* count, const void* offset,
                             const void* rowOf, const void* slotOf) {
  const RowsShape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6], shape[7]};
  return check_rows_sort(s, expertOf, sizeofIndex, count, offset, rowOf, slotOf);
}

int cutt_hostcheck_rows_move(const int* shape, const void* token, long long tokenStride, const void* row, long long rowStride,
                             const void* rowOf, const void* count, const void* offset, const void* weight, const void* other,
                             long long otherStride, const void* dweight, int rowsOut) {
  const RowsShape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6], shape[7]};
  return check_rows_move(s, RowsMoveArgs{token, tokenStride, row, rowStride, (const int*)rowOf, (const int*)count, (const int*)offset,
                                         (const float*)weight, other, otherStride, (const float*)dweight, rowsOut != 0, rowsOut != 0});
}

int cutt_hostcheck_pages_build(const int* shape, const void* held, const void* added, const void* freeList, const void* poolIn,
                               const void* poolOut, const void* table, long long tableStride, const void* tokenOffset,
                               const void* pageOffset, const void* slot) {
  const PagesShape s{shape[0], shape[1], shape[2], shape[3], FastDiv()};
  return check_pages_build(s, held, added, freeList, poolIn, poolOut, table, tableStride, tokenOffset, pageOffset, slot);
}

int cutt_hostcheck_paged_move(const int* shape, const long long* strides, const void* k, const void* v, long long tokenStride,
                              long long headStride, const void* slot, const void* kCache, const void* vCache, int rowsOut) {
  const PagedShape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], strides[0], strides[1], strides[2]};
  return check_paged_move(s, k, v, tokenStride, headStride, slot, kCache, vCache, rowsOut != 0);
}

// Exclusive prefix sums of a block's (tokens, pages) in the steps of the kernel's scan: within warps of 32, over the
// warps' sums, then both together.
struct Pair {
  uint32_t tokens, pages;
};
static Pair operator+(Pair a, Pair b) { return Pair{add_up_to_int(a.tokens, b.tokens), a.pages + b.pages}; }
static void warp_scan(Pair* x) {         // inclusive
  for (int d = 1; d < 32; d <<= 1)
    for (int lane = 31; lane >= d; lane--) x[lane] = x[lane] + x[lane - d];
}
static Pair block_scan(Pair* x, int threads) {
  Pair sums[32] = {};
  for (int w = 0; w < threads / 32; w++) {
    warp_scan(x + w * 32);
    sums[w] = x[w * 32 + 31];
  }
  warp_scan(sums);
  for (int t = threads - 1; t >= 0; t--) {
    const Pair inWarp = t % 32 ? x[t - 1] : Pair{0, 0};
    x[t] = t / 32 ? inWarp + sums[t / 32 - 1] : inWarp;
  }
  return sums[threads / 32 - 1];
}

// cutt_pages_build on host arrays: the scan in blocks of `threads` requests, then the kernel's expressions per token
// and per page.  Returns the number of accesses outside the arrays (table: requests * tableStride
// entries, freeList: freeEntries), which are skipped.
static long long pages_run(int requests, int pageSize, int tableWidth, int maxTokens, const int* held, const int* added,
                           const int* freeList, int freeEntries, const int* poolIn, int* poolOut, int* table,
                           long long tableStride, int* tokenOffset, int* pageOffset, long long* slot, int threads) {
  PagesBuild p{PagesShape{requests, pageSize, tableWidth, maxTokens, make_fastdiv(pageSize)}, held, added, freeList, poolOut,
               table, tableStride, tokenOffset, pageOffset, slot};
  long long bad = 0;
  int first = 0, limit = 0;
  if (freeList) {
    first = clamp_pool(poolIn[0]);
    limit = clamp_pool(poolIn[1]);
  }
  Pair at{0, (uint32_t)first}, x[1024];
  for (int b0 = 0; b0 < requests; b0 += threads) {
    for (int t = 0; t < threads; t++) {
      const int b = b0 + t;
      const int n = b < requests && added[b] > 0 ? added[b] : 0;
      x[t] = Pair{(uint32_t)n, b < requests && freeList ? (uint32_t)pages_taken(held[b], n, p.s.divPage, tableWidth) : 0u};
    }
    const Pair total = block_scan(x, threads);
    for (int t = 0; t < threads && b0 + t < requests; t++) {
      const Pair q = at + x[t];
      tokenOffset[b0 + t] = (int)q.tokens;
      if (freeList) pageOffset[b0 + t] = (int)q.pages;
    }
    at = at + total;
  }
  tokenOffset[requests] = (int)at.tokens;
  if (freeList) {
    if (at.pages > 0x7fffffffu) bad++;
    pageOffset[requests] = (int)at.pages;
    poolOut[0] = (int)at.pages < (first > limit ? first : limit) ? (int)at.pages : (first > limit ? first : limit);
    poolOut[1] = poolIn[1];
    if (limit > freeEntries) return -1;
  }
  for (int q = 0; q < maxTokens; q++) {
    slot[q] = -1;
    if (q >= tokenOffset[requests]) continue;
    const int b = last_at_or_before(tokenOffset, requests + 1, q);
    if (b < 0 || b >= requests) { bad++; continue; }
    slot[q] = slot_of_token(p, b, q, limit);
  }
  if (freeList)
    for (int f = pageOffset[0]; f < pageOffset[requests]; f++) {
      const int b = last_at_or_before(pageOffset, requests + 1, f);
      if (b < 0 || b >= requests) { bad++; continue; }
      const long long idx = pages_of(held[b] > 0 ? held[b] : 0, p.s.divPage) + (long long)(f - pageOffset[b]);
      if (idx >= tableWidth) { bad++; continue; }
      take_page(p, b, f, limit);
    }
  return bad;
}

long long cutt_hostcheck_pages_run(int requests, int pageSize, int tableWidth, int maxTokens, const int* held, const int* added,
                                   const int* freeList, int freeEntries, const int* poolIn, int* poolOut, int* table,
                                   long long tableStride, int* tokenOffset, int* pageOffset, long long* slot) {
  return pages_run(requests, pageSize, tableWidth, maxTokens, held, added, freeList, freeEntries, poolIn, poolOut, table,
                   tableStride, tokenOffset, pageOffset, slot, requests > 512 || maxTokens > 512 ? 1024 : 512);
}

// Element offset of a slot in a cache, -1 where it is not one of the cache's.
long long cutt_hostcheck_cache_offset(int pages, int pageSize, long long pageStride, long long slotStride, long long slot) {
  const PagedShape s{1, 1, 1, 1, pages, pageSize, pageStride, slotStride, 1};
  return cache_offset(s, slot, make_fastdiv(pageSize));
}

// cutt_pages_store / cutt_pages_load of one tensor on host arrays, access by access as the blocks do
// it.  Returns the accesses outside the arrays (rowBytes, cacheBytes) or off their alignment, which
// are skipped.
long long cutt_hostcheck_paged_run(const int* shape, const long long* strides, long long tokenStride, long long headStride,
                                   const long long* slot, unsigned char* rows, long long rowBytes, unsigned char* cache,
                                   long long cacheBytes, int store) {
  const PagedShape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], strides[0], strides[1], strides[2]};
  const PagedItems p = paged_items(s, tokenStride * s.elt, headStride * s.elt, (uintptr_t)rows | (uintptr_t)cache);
  long long bad = 0;
  for (int q0 = 0; q0 < s.tokens; q0 += p.perBlock) {
    const int nq = p.perBlock < s.tokens - q0 ? p.perBlock : s.tokens - q0;
    for (uint32_t i = 0; i < (uint32_t)nq * p.vecs; i++) {
      const PagedPlace a = paged_place(p, q0, i);
      long long r, c;
      if (!paged_access(p, a, slot[a.token], r, c)) continue;
      if (c < 0 || r < 0 || c + p.access > cacheBytes || r + p.access > rowBytes || (uintptr_t)(cache + c) % p.access ||
          (uintptr_t)(rows + r) % p.access) {
        bad++;
        continue;
      }
      if (store) memcpy(cache + c, rows + r, p.access);
      else memcpy(rows + r, cache + c, p.access);
    }
  }
  return bad;
}

// {blocks, slots, warps, words} of the map's launch.
void cutt_hostcheck_sort_shape(int n, int experts, int most, int* out) {
  const SortShape c = sort_shape(n, experts, most);
  out[0] = c.blocks;
  out[1] = c.slots;
  out[2] = c.warps;
  out[3] = c.words;
}

int cutt_hostcheck_local_expert(long long e, int first, int experts) { return local_expert(e, first, experts); }

}  // extern "C"
