/*
 * cutt_rows.h - rows moved by an index map that the GPU builds (expert order, paged caches).
 *
 * NOTHING in this header has a counterpart in the original cuTT.  A cuttPlan's order of elements
 * is known on the host when the plan is made; here the order is data on the device:
 *   - rows of tokens sorted by expert, moved into that order and back with weights, and the
 *     gradients of both moves (cutt_rows_*);
 *   - block tables and slot maps of a paged cache built from request lengths, and rows stored
 *     into and loaded from its pages (cutt_pages_*).
 *
 * Conventions are those of cutt_c.h: result codes are cuttResult values as ints, streams are
 * passed as void*, all data pointers are DEVICE pointers, a plan is bound to the device and
 * stream it was made with, plans own no device memory and every call is asynchronous on the
 * plan's stream.  Handles are destroyed with cuttDestroy / cutt_c_destroy and described by
 * cutt_c_plan_describe; they are not valid for cuttExecute.  No call synchronises, allocates
 * or keeps anything between calls, so every call may be captured into a CUDA graph (a replay
 * reads the maps and lengths that are in the buffers then).
 *
 * Clusters of 16 blocks are used where the stream's context can hold them, else of 8; a context
 * must be able to hold those (eight SMs of one group, as the driver splits them for green contexts).
 *
 * Argument errors return CUTT_INVALID_PARAMETER before anything is launched; a call on another
 * device than the plan's returns CUTT_INVALID_DEVICE; a handle of another kind or none
 * CUTT_INVALID_PLAN.  Inputs and outputs must not overlap (equal addresses are refused).
 */
#ifndef CUTT_ROWS_H
#define CUTT_ROWS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the rows.  CUTT_ROWS_BYTES: 1-byte elements moved as they are (no weights, no
 * sums).  The others are summed and multiplied in 32 bits and rounded once. */
#define CUTT_ROWS_BYTES 0
#define CUTT_ROWS_F16 1
#define CUTT_ROWS_BF16 2
#define CUTT_ROWS_F32 3

/* Plan for `tokens` rows (>= 0) of `width` elements, each with `choices` experts.  A slot s =
 * token * choices + j names one choice.  This process holds experts firstExpert ..
 * firstExpert + experts - 1 (1 <= experts <= 4096); slots that name any other number are dropped.
 * `capacity` rows hold the sorted rows; each expert's segment starts at a multiple of `align`
 * (1 .. 4096).  tokens * choices and capacity are at most 2^30, width at most 2^24.  With no tokens the
 * tensors of tokens and slots are empty and may be NULL. */
int cutt_rows_plan(unsigned int* handle, int tokens, int choices, int experts, int firstExpert,
                   int align, int capacity, int width, int type, void* stream);

/* The map.  expertOf[tokens * choices]: sizeofIndex 4 (int32) or 8 (int64) bytes each.
 *   count[experts]        rows of each expert
 *   offset[experts + 1]   first row of each expert's segment; offset[experts] = rows in use
 *   rowOf[slots]          row of each slot, -1 where the slot is dropped
 *   slotOf[capacity]      slot of each row, -1 where the row is padding or not in use
 * Slots of one expert keep their order.  Rows that would lie at or beyond `capacity` are dropped
 * (the last experts lose theirs; count and offset say what is held): with capacity >= slots +
 * min(experts, slots) * (align - 1) none is. */
int cutt_rows_sort(unsigned int handle, const void* expertOf, size_t sizeofIndex, int* count,
                   int* offset, int* rowOf, int* slotOf);

/* Row strides below are in elements.  An input's may be anything from 0 (one row for all) up, an
 * output's is at least `width`.  Token-side inputs have `tokens` rows, row-side ones `capacity`; all of
 * them, and what lies between them, may be read.  weight[slots] may be NULL (1 everywhere).  Entries of
 * rowOf outside 0 .. capacity-1 are taken as dropped.  Sums over slots are in the order of the slots;
 * the last bits of dweight depend on the shapes, the strides' alignment and the device, not on the run. */

/* y[rowOf[s]] = weight[s] * x[s / choices]; padding rows inside the segments (between
 * offset[e] + count[e] and offset[e+1]) become zero; rows from offset[experts] on are left alone. */
int cutt_rows_dispatch(unsigned int handle, const void* x, long long xStride, const int* rowOf,
                       const int* count, const int* offset, const float* weight, void* y,
                       long long yStride);

/* out[t] = sum over j of weight[s] * y[rowOf[s]], s = t * choices + j, in the order of j; dropped
 * slots add nothing, a token without any becomes zero. */
int cutt_rows_combine(unsigned int handle, const void* y, long long yStride, const int* rowOf,
                      const float* weight, void* out, long long outStride);

/* Gradient of cutt_rows_dispatch: dx[t] = sum over j of weight[s] * dy[rowOf[s]]; with dweight
 * (then x is needed too, otherwise both are NULL) dweight[s] = <dy[rowOf[s]], x[t]>, 0 where
 * dropped. */
int cutt_rows_dispatch_grad(unsigned int handle, const void* dy, long long dyStride, const int* rowOf,
                            const float* weight, const void* x, long long xStride, void* dx,
                            long long dxStride, float* dweight);

/* Gradient of cutt_rows_combine: dy[rowOf[s]] = weight[s] * dout[t], padding rows inside the
 * segments zero; with dweight (then y is needed too) dweight[s] = <y[rowOf[s]], dout[t]>, 0
 * where dropped. */
int cutt_rows_combine_grad(unsigned int handle, const void* dout, long long doutStride, const int* rowOf,
                           const int* count, const int* offset, const float* weight, const void* y,
                           long long yStride, void* dy, long long dyStride, float* dweight);

/* Plan for block tables of `requests` rows (1 at least) of `tableWidth` pages each (requests *
 * tableWidth < 2^30) and slot maps of `maxTokens` entries (<= 2^30).  A page holds `pageSize` tokens. */
int cutt_pages_plan(unsigned int* handle, int requests, int pageSize, int tableWidth, int maxTokens,
                    void* stream);

/* Request b has held[b] tokens in its pages and added[b] new ones (negative counts as 0).
 *   need_b = pages that the new tokens take beyond those of the held ones (never beyond tableWidth)
 *   tokenOffset[requests + 1]  prefix sums of added
 *   pageOffset[requests + 1]   pool[0] + prefix sums of need: where in freeList each request's start
 *   table[b][pages held + i]   freeList[pageOffset[b] + i], or -1 at or beyond pool[1]; the other
 *                              entries are left alone.  Rows are tableStride entries apart.
 *   slot[maxTokens]            of new token i of request b, at tokenOffset[b] + i: page * pageSize +
 *                              place in the page, from the table; -1 where there is no page and
 *                              behind the last token.  Tokens at or beyond maxTokens get no entry.
 *   pool                       {next free entry, entries} of freeList (at most 2^30); poolOut = {min(pageOffset[
 *                              requests], max(pool[0], pool[1])), pool[1]} and may be the same address.
 * pageOffset[requests] > pool[1] says that pages ran short, and by how many.
 * With freeList NULL (then poolIn, poolOut and pageOffset are NULL too) no page is taken and the
 * table is only read: slots of tokens whose pages the table has already. */
int cutt_pages_build(unsigned int handle, const int* held, const int* added, const int* freeList,
                     const int* poolIn, int* poolOut, int* table, long long tableStride,
                     int* tokenOffset, int* pageOffset, long long* slot);

/* Plan for rows of `tokens` tokens x `heads` x `headSize` elements of sizeofType (1, 2, 4 or 8)
 * bytes in caches of `pages` pages of `pageSize` tokens: element d of head h of slot s lies at
 * (s / pageSize) * pageStride + (s % pageSize) * slotStride + h * headStride + d (strides in
 * elements, slotStride and headStride at least headSize).  With no tokens k, v and slot are empty and
 * may be NULL. */
int cutt_pages_plan_rows(unsigned int* handle, int tokens, int heads, int headSize, size_t sizeofType,
                         int pages, int pageSize, long long pageStride, long long slotStride,
                         long long headStride, void* stream);

/* Stores rows into / loads rows from the slots slot[tokens].  Row q, head h starts at q *
 * tokenStride + h * headStride (elements; for loads both at least headSize).  v and vCache may
 * both be NULL.  Rows whose slot is not in 0 .. pages * pageSize - 1 are skipped: neither the cache
 * nor the row is read or written (k and v may end before such rows).  Two rows stored to one slot leave either's elements there. */
int cutt_pages_store(unsigned int handle, const void* k, const void* v, long long tokenStride,
                     long long headStride, const long long* slot, void* kCache, void* vCache);
int cutt_pages_load(unsigned int handle, const void* kCache, const void* vCache, const long long* slot,
                    void* k, void* v, long long tokenStride, long long headStride);

#ifdef __cplusplus
}
#endif
#endif /* CUTT_ROWS_H */
