"""Rows moved by an index map that the GPU builds (``include/cutt_rows.h``): rows sorted by expert,
moved into that order and back with weights, the gradients of both moves; block tables and slot
maps of a paged cache, rows stored into and loaded from its pages.

Like the rest of the package this is a thin ctypes mirror of the C ABI: data pointers are raw device
addresses (``tensor.data_ptr()``; 0 where the C call takes NULL), strides count elements, streams are
raw ``cudaStream_t`` values, and every call is asynchronous on its plan's stream.  The classes raise
``CuttError`` where the C call returns a code other than ``CUTT_SUCCESS``.

A layer whose tokens go to experts, forward and backward::

    p = RowPlan(tokens, choices, experts, width, CUTT_ROWS_BF16, align=128, stream=s)
    p.sort(expert_of, 8, count, offset, row_of, slot_of)
    p.dispatch(x, row_of, count, offset, rows)
    ...                                        # the experts' products: rows -> y, segment by segment
    p.combine(y, row_of, out, weight=w)
    p.combine_grad(dout, row_of, count, offset, dy, weight=w, y=y, dweight=dw)
    ...                                        # the products' gradients: dy -> drows
    p.dispatch_grad(drows, row_of, dx)

A step of a server with a paged cache::

    pages = PagePlan(requests, page_size, table_width, max_tokens, stream=s)
    pages.build(held, added, free_list, pool, pool, table, token_offset, page_offset, slot)
    rows = PagedRows(max_tokens, heads, head_size, 2, num_pages, page_size, *strides, stream=s)
    rows.store(k, v, slot, k_cache, v_cache)   # for every layer with the same slot map
"""
from __future__ import annotations

import ctypes

CUTT_ROWS_BYTES = 0
CUTT_ROWS_F16 = 1
CUTT_ROWS_BF16 = 2
CUTT_ROWS_F32 = 3


def bind(L: ctypes.CDLL) -> None:
    """Declares the argument types of the row operators."""
    up = ctypes.POINTER(ctypes.c_uint)
    i, u, vp, ll, sz = ctypes.c_int, ctypes.c_uint, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_size_t
    for name, args in (
            ("cutt_rows_plan", [up] + [i] * 8 + [vp]),
            ("cutt_rows_sort", [u, vp, sz, vp, vp, vp, vp]),
            ("cutt_rows_dispatch", [u, vp, ll, vp, vp, vp, vp, vp, ll]),
            ("cutt_rows_combine", [u, vp, ll, vp, vp, vp, ll]),
            ("cutt_rows_dispatch_grad", [u, vp, ll, vp, vp, vp, ll, vp, ll, vp]),
            ("cutt_rows_combine_grad", [u, vp, ll, vp, vp, vp, vp, vp, ll, vp, ll, vp]),
            ("cutt_pages_plan", [up, i, i, i, i, vp]),
            ("cutt_pages_build", [u] + [vp] * 6 + [ll] + [vp] * 3),
            ("cutt_pages_plan_rows", [up, i, i, i, sz, i, i, ll, ll, ll, vp]),
            ("cutt_pages_store", [u, vp, vp, ll, ll, vp, vp, vp]),
            ("cutt_pages_load", [u, vp, vp, vp, vp, vp, ll, ll])):
        f = getattr(L, name)
        f.argtypes = args
        f.restype = i


def _package():
    import cutt_b200
    return cutt_b200


def _c_ints(what: str, *values: int) -> None:
    """ctypes would cut larger numbers down to 32 bits."""
    if not all(-2**31 <= v < 2**31 for v in values):
        C = _package()
        raise C.CuttError(C.CUTT_INVALID_PARAMETER, what)


# Never a plan's number: calls after destroy() are refused as those of any unknown handle.
_NONE = 0xffffffff


class _Handle:
    """A plan.  Calls are a few microseconds in all, so the methods below go to the C functions directly."""
    handle = None
    _h = _NONE

    def _made(self, rc: int, handle: ctypes.c_uint) -> None:
        C = _package()
        if rc != C.CUTT_SUCCESS:
            raise C.CuttError(rc, type(self).__name__)
        self.handle = self._h = handle.value
        self._lib = C.lib()

    def _failed(self, rc: int, what: str):
        return _package().CuttError(rc, what)

    def describe(self) -> str:
        return _package().plan_describe(self._h)

    def destroy(self) -> None:
        if self.handle is not None:
            _package().cuttDestroy(self.handle)
            self.handle, self._h = None, _NONE

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class RowPlan(_Handle):
    """Rows of ``tokens`` x ``width`` sorted by ``choices`` experts each (cutt_rows_plan).  ``capacity``
    defaults to the rows that the map can need at most."""

    def __init__(self, tokens: int, choices: int, experts: int, width: int, type: int, first: int = 0,
                 align: int = 1, capacity: int | None = None, stream: int = 0):
        if capacity is None:
            slots = tokens * choices
            capacity = max(1, slots + min(experts, slots) * (align - 1))
        _c_ints("RowPlan", tokens, choices, experts, first, align, capacity, width, type)
        self.capacity, self.width = capacity, width
        h = ctypes.c_uint(0)
        rc = _package().lib().cutt_rows_plan(ctypes.byref(h), tokens, choices, experts, first, align, capacity,
                                             width, type, stream)
        self._made(rc, h)

    def sort(self, expert_of: int, index_bytes: int, count: int, offset: int, row_of: int, slot_of: int) -> None:
        rc = self._lib.cutt_rows_sort(self._h, expert_of, index_bytes, count, offset, row_of, slot_of)
        if rc:
            raise self._failed(rc, "sort")

    def dispatch(self, x: int, row_of: int, count: int, offset: int, y: int, weight: int = 0,
                 x_stride: int | None = None, y_stride: int | None = None) -> None:
        w = self.width
        rc = self._lib.cutt_rows_dispatch(self._h, x, w if x_stride is None else x_stride, row_of, count, offset,
                                          weight, y, w if y_stride is None else y_stride)
        if rc:
            raise self._failed(rc, "dispatch")

    def combine(self, y: int, row_of: int, out: int, weight: int = 0, y_stride: int | None = None,
                out_stride: int | None = None) -> None:
        w = self.width
        rc = self._lib.cutt_rows_combine(self._h, y, w if y_stride is None else y_stride, row_of, weight, out,
                                         w if out_stride is None else out_stride)
        if rc:
            raise self._failed(rc, "combine")

    def dispatch_grad(self, dy: int, row_of: int, dx: int, weight: int = 0, x: int = 0, dweight: int = 0,
                      dy_stride: int | None = None, x_stride: int | None = None, dx_stride: int | None = None) -> None:
        w = self.width
        rc = self._lib.cutt_rows_dispatch_grad(self._h, dy, w if dy_stride is None else dy_stride, row_of, weight,
                                               x, w if x_stride is None else x_stride, dx,
                                               w if dx_stride is None else dx_stride, dweight)
        if rc:
            raise self._failed(rc, "dispatch_grad")

    def combine_grad(self, dout: int, row_of: int, count: int, offset: int, dy: int, weight: int = 0, y: int = 0,
                     dweight: int = 0, dout_stride: int | None = None, y_stride: int | None = None,
                     dy_stride: int | None = None) -> None:
        w = self.width
        rc = self._lib.cutt_rows_combine_grad(self._h, dout, w if dout_stride is None else dout_stride, row_of,
                                              count, offset, weight, y, w if y_stride is None else y_stride, dy,
                                              w if dy_stride is None else dy_stride, dweight)
        if rc:
            raise self._failed(rc, "combine_grad")


class PagePlan(_Handle):
    """Block tables and slot maps of ``requests`` requests (cutt_pages_plan)."""

    def __init__(self, requests: int, page_size: int, table_width: int, max_tokens: int, stream: int = 0):
        _c_ints("PagePlan", requests, page_size, table_width, max_tokens)
        self.table_width = table_width
        h = ctypes.c_uint(0)
        rc = _package().lib().cutt_pages_plan(ctypes.byref(h), requests, page_size, table_width, max_tokens, stream)
        self._made(rc, h)

    def build(self, held: int, added: int, free_list: int, pool_in: int, pool_out: int, table: int, token_offset: int,
              page_offset: int, slot: int, table_stride: int | None = None) -> None:
        rc = self._lib.cutt_pages_build(self._h, held, added, free_list, pool_in, pool_out, table,
                                        self.table_width if table_stride is None else table_stride, token_offset,
                                        page_offset, slot)
        if rc:
            raise self._failed(rc, "build")

    def slots(self, held: int, added: int, table: int, token_offset: int, slot: int, table_stride: int | None = None) -> None:
        """Slots of tokens whose pages the table has already: no page is taken, the table is only read."""
        self.build(held, added, 0, 0, 0, table, token_offset, 0, slot, table_stride)


class PagedRows(_Handle):
    """Rows of ``tokens`` x ``heads`` x ``head_size`` elements in pages (cutt_pages_plan_rows)."""

    def __init__(self, tokens: int, heads: int, head_size: int, element_bytes: int, pages: int, page_size: int,
                 page_stride: int, slot_stride: int, head_stride: int, stream: int = 0):
        _c_ints("PagedRows", tokens, heads, head_size, element_bytes, pages, page_size)
        self.token_stride, self.head_stride = heads * head_size, head_size
        h = ctypes.c_uint(0)
        rc = _package().lib().cutt_pages_plan_rows(ctypes.byref(h), tokens, heads, head_size, element_bytes, pages,
                                                   page_size, page_stride, slot_stride, head_stride, stream)
        self._made(rc, h)

    def store(self, k: int, v: int, slot: int, k_cache: int, v_cache: int, token_stride: int | None = None,
              head_stride: int | None = None) -> None:
        rc = self._lib.cutt_pages_store(self._h, k, v, self.token_stride if token_stride is None else token_stride,
                                        self.head_stride if head_stride is None else head_stride, slot, k_cache, v_cache)
        if rc:
            raise self._failed(rc, "store")

    def load(self, k_cache: int, v_cache: int, slot: int, k: int, v: int, token_stride: int | None = None,
             head_stride: int | None = None) -> None:
        rc = self._lib.cutt_pages_load(self._h, k_cache, v_cache, slot, k, v,
                                       self.token_stride if token_stride is None else token_stride,
                                       self.head_stride if head_stride is None else head_stride)
        if rc:
            raise self._failed(rc, "load")
