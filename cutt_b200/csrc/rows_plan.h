// Plans of the row operators (include/cutt_rows.h): shapes, limits and argument checks that need
// no device, and the index arithmetic that the kernels and the host interpreter share.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "permute_desc.h"

namespace cuttb {

constexpr int kRowsMaxExperts = 4096;
constexpr int kRowsMaxAlign = 4096;
constexpr int kRowsMaxCount = 1 << 30;    // slots, capacity, table entries, tokens of a slot map
constexpr int kRowsMaxWidth = 1 << 24;

struct RowsShape {
  int tokens, choices, experts, first, align, capacity, width, type;
};

struct PagesShape {
  int requests, pageSize, tableWidth, maxTokens;
  FastDiv divPage;
};

struct PagedShape {
  int tokens, heads, headSize, elt, pages, pageSize;
  long long pageStride, slotStride, headStride;   // of the cache, in elements
};

// 0 or CUTT_INVALID_PARAMETER (2).
int check_rows_shape(const RowsShape& s);
int check_pages_shape(const PagesShape& s);
int check_paged_shape(const PagedShape& s);
int rows_element_bytes(int type);   // 0: no such type

// Arguments of one move, as the C entry points get them.
struct RowsMoveArgs {
  const void* token;         // token-side tensor (input of dispatch, output of combine)
  long long tokenStride;
  const void* row;           // row-side tensor
  long long rowStride;
  const int* rowOf;
  const int* count;          // null where no padding rows are written
  const int* offset;
  const float* weight;
  const void* other;         // second factor of the weights' gradient
  long long otherStride;
  const float* dweight;
  bool rowsOut;              // dispatch, combine_grad: rows are written
  bool needMap;              // count and offset are required
};
int check_rows_sort(const RowsShape& s, const void* expertOf, size_t sizeofIndex, const void* count,
                    const void* offset, const void* rowOf, const void* slotOf);
int check_rows_move(const RowsShape& s, const RowsMoveArgs& a);
int check_pages_build(const PagesShape& s, const void* held, const void* added, const void* freeList,
                      const void* poolIn, const void* poolOut, const void* table, long long tableStride,
                      const void* tokenOffset, const void* pageOffset, const void* slot);
int check_paged_move(const PagedShape& s, const void* k, const void* v, long long tokenStride,
                     long long headStride, const void* slot, const void* kCache, const void* vCache,
                     bool rowsOut);

// Widest access (16, 8, 4, 2 or 1 bytes, at least the element) that divides all of the given
// addresses and byte distances, or-ed together.
int access_bytes(unsigned long long bits, int elt);

// Launch of the map of n slots.  Up to kClusterSlots slots one cluster, above three kernels (blocks = 0).
// `most`: blocks of the largest cluster that the device can hold, kPortableBlocks at least.
constexpr int kClusterSlots = 65536;
constexpr int kMostClusterBlocks = 16;
constexpr int kPortableBlocks = 8;            // of a cluster that every device can hold
constexpr int kMostSortWords = 216 * 1024 / 4;   // of a block's shared memory
// Warps of a block: one for 32 slots, at most 16 (every further one is a histogram to clear and to scan).
// 8, 16, 32 of them: 65536 slots of 128 experts 8.8, 6.9, 8.4 us; 524288 slots of 256 experts 13.4, 12.4, 14.7.
constexpr int kSortWarps = 16;
struct SortShape {
  int blocks, slots, warps;   // of the cluster, of a block, of a block
  int words;                  // of a block's shared memory
};
int ranked_words(int slots, int warps, int experts);
int warps_for(int slots, int experts, int most);
SortShape sort_shape(int n, int experts, int most);

// --- index arithmetic ---

// Expert of a slot counted from the first one held here; -1: not held here.
CUTT_HD int local_expert(long long e, int first, int experts) {
  return e >= first && e < (long long)first + experts ? (int)(e - first) : -1;
}
CUTT_HD int local_expert(int e, int first, int experts) {
  return e >= first && e < first + experts ? e - first : -1;     // first + experts fits: check_rows_shape
}

// Segment of an expert with n rows that starts at row o (not clipped): what fits into `capacity`.
CUTT_HD int clip_row(int o, int capacity) { return o < capacity ? o : capacity; }
CUTT_HD int held_rows(int o, int n, int capacity) { return clip_row(o + n, capacity) - clip_row(o, capacity); }
CUTT_HD int align_rows(int n, int align) { return (n + align - 1) / align * align; }

// Pages of a request: held by its tokens, taken for the new ones.  Lengths are at most 2^31 - 1 each, so
// their sum has 32 bits (a 64-bit division would take longer than everything else on a request).
CUTT_HD uint32_t pages_of(uint32_t tokens, const FastDiv& divPage) { return tokens ? fdiv(tokens - 1, divPage) + 1 : 0; }
CUTT_HD int pages_taken(int held, int added, const FastDiv& divPage, int tableWidth) {
  const uint32_t c = held > 0 ? held : 0, n = added > 0 ? added : 0;
  const uint32_t have = pages_of(c, divPage), all = pages_of(c + n, divPage);
  const uint32_t want = all < (uint32_t)tableWidth ? all : tableWidth;
  return want > have ? (int)(want - have) : 0;
}

// Sum of two counts that stops at 2^31 - 1.  Associative, so a scan with it is the saturated scan.
CUTT_HD uint32_t add_up_to_int(uint32_t a, uint32_t b) {
  const uint32_t c = a + b;              // counts are at most 2^31 - 1 each
  return c < 0x7fffffffu ? c : 0x7fffffffu;
}
CUTT_HD int clamp_pool(int v) { return v < 0 ? 0 : v > kRowsMaxCount ? kRowsMaxCount : v; }

// First entry greater than q of an ascending array of n entries, less one: the last request that
// starts at or before q (requests without tokens start where the next one does and are passed).
CUTT_HD int last_at_or_before(const int* start, int n, int q) {
  int lo = 0, hi = n;            // start[0] <= q is given
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] > q) hi = mid; else lo = mid + 1;
  }
  return lo - 1;
}

struct PagesBuild {
  PagesShape s;
  const int* held;
  const int* added;
  const int* freeList;
  const int* pool;            // {.., entries} (poolOut: its second word is not changed by a call)
  int* table;
  long long tableStride;
  const int* tokenOffset;
  const int* pageOffset;
  long long* slot;
};

// Slot of token q (q < tokenOffset[requests]) of request b.
CUTT_HD long long slot_of_token(const PagesBuild& p, int b, int q, int limit) {
  const unsigned c = p.held[b] > 0 ? p.held[b] : 0;
  const unsigned pos = c + (unsigned)(q - p.tokenOffset[b]);   // at most 2^31 - 1 + 2^30
  const unsigned idx = fdiv(pos, p.s.divPage);
  if (idx >= (unsigned)p.s.tableWidth) return -1;
  int page;
  const unsigned have = p.freeList ? pages_of(c, p.s.divPage) : 0xffffffffu;
  if (idx < have) {
    page = p.table[(long long)b * p.tableStride + idx];
  } else {
    const int f = p.pageOffset[b] + (int)(idx - have);
    page = f < limit ? p.freeList[f] : -1;
  }
  return page < 0 ? -1 : (long long)page * p.s.pageSize + (pos - idx * (unsigned)p.s.pageSize);
}

// Writes the table entry of position f of the free list (pageOffset[0] <= f < pageOffset[requests]).
CUTT_HD void take_page(const PagesBuild& p, int b, int f, int limit) {
  const unsigned c = p.held[b] > 0 ? p.held[b] : 0;
  const unsigned idx = pages_of(c, p.s.divPage) + (unsigned)(f - p.pageOffset[b]);
  p.table[(long long)b * p.tableStride + idx] = f < limit ? p.freeList[f] : -1;
}

// Element offset of a slot's row in a cache; -1: not a slot of this cache.
CUTT_HD long long cache_offset(const PagedShape& s, long long slot, const FastDiv& divPage) {
  if (slot < 0 || slot >= (long long)s.pages * s.pageSize) return -1;
  if (slot >> 32) {          // more than 2^32 slots: plain division
    const long long page = slot / s.pageSize;
    return page * s.pageStride + (slot - page * s.pageSize) * s.slotStride;
  }
  const uint32_t page = fdiv((uint32_t)slot, divPage);
  return page * s.pageStride + ((uint32_t)slot - page * (uint32_t)s.pageSize) * s.slotStride;
}

// Rows stored into or loaded from pages, as accesses of `access` bytes.
struct PagedItems {
  PagedShape s;                        // heads that lie one behind the other on both sides are one
  long long tokenStride, headStride;   // of the rows, bytes
  int access;
  int vecs;                            // accesses of a token
  int perBlock;                        // tokens of a block
  FastDiv divPage, divRow, divHead;    // by pageSize, by accesses of a token, by accesses of a head
};
constexpr int kPagedThreads = 128;
constexpr int kPagedItems = 4;         // accesses of a thread in flight at once

// strides in bytes; addresses: those of all rows and caches, or-ed together.
PagedItems paged_items(const PagedShape& s, long long tokenStride, long long headStride, unsigned long long addresses);

// Access i of a block whose first token is q0: its token, head and place in the head's elements.
struct PagedPlace {
  int token;
  uint32_t head, piece;
};
CUTT_HD PagedPlace paged_place(const PagedItems& p, int q0, uint32_t i) {
  const uint32_t q = fdiv(i, p.divRow), r = i - q * (uint32_t)p.vecs;
  const uint32_t h = fdiv(r, p.divHead);
  return PagedPlace{q0 + (int)q, h, r - h * p.divHead.d};
}
// Its byte offsets in the rows and in the cache.  False where the token's slot is not one of the cache's:
// neither side is read or written then (the rows may end before such a token).
CUTT_HD bool paged_access(const PagedItems& p, const PagedPlace& a, long long slot, long long& row, long long& cache) {
  const long long at = cache_offset(p.s, slot, p.divPage);
  if (at < 0) return false;
  row = (long long)a.token * p.tokenStride + a.head * p.headStride + (long long)a.piece * p.access;
  cache = (at + a.head * p.s.headStride) * p.s.elt + (long long)a.piece * p.access;
  return true;
}

}  // namespace cuttb
