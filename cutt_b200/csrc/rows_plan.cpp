// Argument checks of the row operators (no CUDA calls).
#include "rows_plan.h"

namespace cuttb {

namespace {
constexpr int kBad = 2;   // CUTT_INVALID_PARAMETER

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Whether an output is given twice, or as an input too.  Null pointers are no addresses.
bool shares(const void* const* out, int outs, const void* const* in, int ins) {
  for (int i = 0; i < outs; i++) {
    if (!out[i]) continue;
    for (int j = 0; j < i; j++)
      if (out[i] == out[j]) return true;
    for (int j = 0; j < ins; j++)
      if (out[i] == in[j]) return true;
  }
  return false;
}
}  // namespace

int rows_element_bytes(int type) {
  switch (type) {
    case 0: return 1;
    case 1: case 2: return 2;
    case 3: return 4;
  }
  return 0;
}

int check_rows_shape(const RowsShape& s) {
  if (!rows_element_bytes(s.type)) return kBad;
  if (s.tokens < 0 || s.choices < 1 || (long long)s.tokens * s.choices > kRowsMaxCount) return kBad;
  if (s.experts < 1 || s.experts > kRowsMaxExperts) return kBad;
  if (s.first < 0 || (long long)s.first + s.experts > 0x7fffffffLL) return kBad;
  if (s.align < 1 || s.align > kRowsMaxAlign) return kBad;
  if (s.capacity < 1 || s.capacity > kRowsMaxCount) return kBad;
  if (s.width < 1 || s.width > kRowsMaxWidth) return kBad;
  return 0;
}

// Up to kClusterSlots slots a cluster, above three kernels.  Measured, 128 experts: 32768 slots 5.5
// against 7.8 us, 65536 slots 6.9 against 7.8 us, and one launch against three; 524288 slots of 256
// experts and 64-bit indices take 12.5 us in three kernels.
// A block takes this many slots where one is enough, else half of them, and more once the cluster is
// full: 288 slots 3.3 us in one block and in four, 512 slots 3.7 and 3.5; 1024 slots 3.5 in four, 4.1
// in one.
constexpr int kBlockSlots = 512;

int ranked_words(int slots, int warps, int experts) { return 2 * slots + (2 * warps + 2) * experts; }

// Warps of a block whose histograms leave room for `slots` slots.
int warps_for(int slots, int experts, int most) {
  int w = most;
  while (w > 1 && ranked_words(slots, w, experts) + 3 * experts > kMostSortWords) w >>= 1;
  return w;
}

SortShape sort_shape(int n, int experts, int most) {
  if (n > kClusterSlots) return SortShape{0, 0, 0, 0};     // (experts are fewer)
  int blocks = 1;
  if (n > kBlockSlots)
    while (blocks < most && n > blocks * (kBlockSlots / 2)) blocks <<= 1;
  SortShape c;
  c.blocks = blocks;
  c.slots = ((n + blocks - 1) / blocks + 31) & ~31;
  c.warps = warps_for(c.slots, experts, kSortWarps);
  while (c.warps > 4 && c.warps * 32 > c.slots) c.warps >>= 1;
  c.words = ranked_words(c.slots, c.warps, experts) + 3 * experts;
  return c;
}

int check_pages_shape(const PagesShape& s) {
  if (s.requests < 1 || s.pageSize < 1 || s.tableWidth < 1) return kBad;
  if (s.pageSize > kRowsMaxCount || (long long)s.requests * s.tableWidth >= kRowsMaxCount) return kBad;
  if (s.maxTokens < 0 || s.maxTokens > kRowsMaxCount) return kBad;
  return 0;
}

int check_paged_shape(const PagedShape& s) {
  if (s.elt != 1 && s.elt != 2 && s.elt != 4 && s.elt != 8) return kBad;
  if (s.tokens < 0 || s.tokens > kRowsMaxCount || s.pages < 1 || s.pageSize < 1) return kBad;
  if (s.heads < 1 || s.heads > (1 << 16) || s.headSize < 1 || s.headSize > (1 << 16)) return kBad;
  if ((long long)s.heads * s.headSize > kRowsMaxWidth) return kBad;
  const long long top = 1LL << 58;   // bytes that a stride may span in all
  if (s.slotStride < s.headSize || s.slotStride > top / s.elt / s.pageSize) return kBad;
  if (s.headStride < s.headSize || s.headStride > top / s.elt / s.heads) return kBad;
  if (s.pageStride < s.headSize || s.pageStride > top / s.elt / s.pages) return kBad;
  return 0;
}

int check_rows_sort(const RowsShape& s, const void* expertOf, size_t sizeofIndex, const void* count,
                    const void* offset, const void* rowOf, const void* slotOf) {
  const bool any = (long long)s.tokens * s.choices > 0;
  if (sizeofIndex != 4 && sizeofIndex != 8) return kBad;
  if (!count || !offset || !slotOf || (any && (!expertOf || !rowOf))) return kBad;
  const void* p[] = {expertOf, count, offset, rowOf, slotOf};
  for (int i = 0; i < 5; i++)
    for (int j = 0; j < i; j++)
      if (p[i] && p[i] == p[j]) return kBad;
  if (!aligned(expertOf, sizeofIndex)) return kBad;
  for (const void* q : p)
    if (!aligned(q, 4)) return kBad;
  return 0;
}

int check_rows_move(const RowsShape& s, const RowsMoveArgs& a) {
  const int elt = rows_element_bytes(s.type);
  const long long top = (1LL << 58) / elt;
  const long long slots = (long long)s.tokens * s.choices;
  // A plan of no tokens: its token-side tensors are empty, their addresses null or any.
  if (!a.row || (slots && (!a.token || !a.rowOf || a.token == a.row))) return kBad;
  if (a.needMap && (!a.count || !a.offset)) return kBad;
  if (s.type == 0 && (a.weight || a.dweight || !a.rowsOut)) return kBad;
  if (slots && (a.dweight != nullptr) != (a.other != nullptr)) return kBad;
  const void* out[] = {a.rowsOut ? a.row : slots ? a.token : nullptr, slots ? a.dweight : nullptr};
  const void* in[] = {a.rowsOut ? slots ? a.token : nullptr : a.row, slots ? a.rowOf : nullptr, a.count, a.offset,
                      slots ? a.weight : nullptr, slots || a.rowsOut ? a.other : nullptr};
  if (shares(out, 2, in, 6)) return kBad;
  if (!aligned(a.token, elt) || !aligned(a.row, elt) || !aligned(a.other, elt)) return kBad;
  if (!aligned(a.rowOf, 4) || !aligned(a.count, 4) || !aligned(a.offset, 4) || !aligned(a.weight, 4) ||
      !aligned(a.dweight, 4))
    return kBad;
  if (a.tokenStride < 0 || a.rowStride < 0 || a.otherStride < 0) return kBad;
  if ((a.rowsOut ? a.rowStride : a.tokenStride) < s.width) return kBad;
  if (a.tokenStride > top / (s.tokens + 1) || a.rowStride > top / s.capacity) return kBad;
  // the other factor lies on the side that is written
  if (a.other && a.otherStride > top / ((a.rowsOut ? s.capacity : s.tokens) + 1)) return kBad;
  return 0;
}

int check_pages_build(const PagesShape& s, const void* held, const void* added, const void* freeList,
                      const void* poolIn, const void* poolOut, const void* table, long long tableStride,
                      const void* tokenOffset, const void* pageOffset, const void* slot) {
  if (!held || !added || !table || !tokenOffset || (!slot && s.maxTokens)) return kBad;
  const bool take = freeList != nullptr;
  if (take != (poolIn != nullptr) || take != (poolOut != nullptr) || take != (pageOffset != nullptr)) return kBad;
  if (tableStride < s.tableWidth || tableStride > (1LL << 56) / s.requests) return kBad;
  if (poolIn != poolOut && (uintptr_t)poolIn < (uintptr_t)poolOut + 8 && (uintptr_t)poolOut < (uintptr_t)poolIn + 8) return kBad;
  const void* in[] = {held, added, freeList, poolIn};
  const void* out[] = {table, tokenOffset, pageOffset, slot, poolOut};
  for (const void* o : out) {
    if (!o) continue;
    for (const void* i : in)
      if (i == o && !(o == poolOut && i == poolIn)) return kBad;
  }
  for (int i = 0; i < 5; i++)
    for (int j = 0; j < i; j++)
      if (out[i] && out[i] == out[j]) return kBad;
  for (const void* p : in)
    if (!aligned(p, 4)) return kBad;
  for (const void* p : out)
    if (!aligned(p, p == slot ? 8 : 4)) return kBad;
  return 0;
}

int check_paged_move(const PagedShape& s, const void* k, const void* v, long long tokenStride,
                     long long headStride, const void* slot, const void* kCache, const void* vCache,
                     bool rowsOut) {
  if (!kCache) return kBad;
  // (rows and slots of no tokens are empty: their addresses are null or any)
  if (s.tokens && (!k || !slot || (v != nullptr) != (vCache != nullptr))) return kBad;
  const void* rows[] = {k, v, slot};
  const void* caches[] = {kCache, vCache, slot};
  if (s.tokens && (rowsOut ? shares(rows, 2, caches, 3) : shares(caches, 2, rows, 3))) return kBad;
  const void* p[] = {k, v, kCache, vCache};
  for (const void* q : p)
    if (!aligned(q, s.elt)) return kBad;
  if (!aligned(slot, 8)) return kBad;
  const long long low = rowsOut ? s.headSize : 0, top = (1LL << 58) / s.elt;
  if (tokenStride < low || tokenStride > top / (s.tokens + 1)) return kBad;
  if (headStride < low || headStride > top / s.heads) return kBad;
  return 0;
}

int access_bytes(unsigned long long bits, int elt) {
  int vb = 16;
  while (vb > elt && bits % vb) vb >>= 1;
  return vb;
}

PagedItems paged_items(const PagedShape& s, long long tokenStride, long long headStride, unsigned long long addresses) {
  PagedItems p;
  p.s = s;
  p.tokenStride = tokenStride;
  p.headStride = headStride;
  // longer pieces, and wider accesses where the head size is odd
  if (s.headStride == s.headSize && headStride == (long long)s.headSize * s.elt) {
    p.s.headSize = s.headSize * s.heads;
    p.s.heads = 1;
  }
  unsigned long long bits = addresses | (unsigned long long)p.s.headSize * s.elt | (unsigned long long)tokenStride |
                            (unsigned long long)(s.pageStride * s.elt) | (unsigned long long)(s.slotStride * s.elt);
  if (p.s.heads > 1) bits |= (unsigned long long)headStride | (unsigned long long)(s.headStride * s.elt);
  p.access = access_bytes(bits, s.elt);
  const int perHead = p.s.headSize * s.elt / p.access;
  p.vecs = perHead * p.s.heads;
  p.divPage = make_fastdiv(s.pageSize);
  p.divHead = make_fastdiv(perHead);
  p.divRow = make_fastdiv(p.vecs);
  p.perBlock = p.vecs >= kPagedThreads * kPagedItems ? 1 : kPagedThreads * kPagedItems / p.vecs;
  return p;
}

}  // namespace cuttb
