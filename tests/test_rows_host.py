"""Row operators without a GPU: limits and refusals, and the index arithmetic of block tables, slot
maps and pages run on host arrays against plain Python (include/cutt_rows.h)."""
import ctypes
import os
import random
import re
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD = 2


@pytest.fixture(scope="module")
def hc(native):
    L = ctypes.CDLL(os.path.join(ROOT, "cutt_b200", "lib", "libcutt_hostcheck.so"))
    i, vp, ll, sz = ctypes.c_int, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_size_t
    L.cutt_hostcheck_rows_shape.argtypes = [i] * 8
    L.cutt_hostcheck_pages_shape.argtypes = [i] * 4
    L.cutt_hostcheck_paged_shape.argtypes = [i] * 6 + [ll] * 3
    L.cutt_hostcheck_rows_sort.argtypes = [vp, vp, sz, vp, vp, vp, vp]
    L.cutt_hostcheck_rows_move.argtypes = [vp, vp, ll, vp, ll, vp, vp, vp, vp, vp, ll, vp, i]
    L.cutt_hostcheck_pages_build.argtypes = [vp] * 7 + [ll] + [vp] * 3
    L.cutt_hostcheck_paged_move.argtypes = [vp, vp, vp, vp, ll, ll, vp, vp, vp, i]
    L.cutt_hostcheck_pages_run.argtypes = [i, i, i, i, vp, vp, vp, i, vp, vp, vp, ll, vp, vp, vp]
    L.cutt_hostcheck_pages_run.restype = ll
    L.cutt_hostcheck_cache_offset.argtypes = [i, i, ll, ll, ll]
    L.cutt_hostcheck_cache_offset.restype = ll
    L.cutt_hostcheck_paged_run.argtypes = [vp, vp, ll, ll, vp, vp, ll, vp, ll, i]
    L.cutt_hostcheck_paged_run.restype = ll
    L.cutt_hostcheck_local_expert.argtypes = [ll, i, i]
    return L


def _ints(*v):
    return (ctypes.c_int * len(v))(*v)


def test_library_exports_the_header(native):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "cutt_rows.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(cutt_(?:rows|pages)_\w+)\s*\(", text)))
    assert len(names) == 11
    for path, flag in ((native.lib_path(), "-D"), (native.lib_path()[:-2] + "a", "-g")):
        syms = subprocess.run(["nm", flag, "--defined-only", path], stdout=subprocess.PIPE, text=True, check=True).stdout
        have = set(line.split()[-1] for line in syms.splitlines() if line.strip())
        assert set(names) <= have


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(choices=0), dict(tokens=1 << 29, choices=3), dict(experts=0), dict(experts=4097), dict(first=-1),
    dict(first=0x7fffffff), dict(align=0), dict(align=4097), dict(capacity=0), dict(capacity=(1 << 30) + 1), dict(width=0),
    dict(width=(1 << 24) + 1), dict(type=4), dict(type=-1)])
def test_row_plan_refusals(native, hc, change):
    good = dict(tokens=4, choices=2, experts=8, first=0, align=1, capacity=8, width=16, type=2)
    assert hc.cutt_hostcheck_rows_shape(*good.values()) == 0
    bad = dict(good, **change)
    assert hc.cutt_hostcheck_rows_shape(*bad.values()) == BAD
    h = ctypes.c_uint(7)
    assert native.lib().cutt_rows_plan(ctypes.byref(h), *bad.values(), None) == BAD
    assert native.lib().cutt_rows_plan(None, *good.values(), None) == BAD
    with pytest.raises(native.CuttError):
        native.RowPlan(bad["tokens"], bad["choices"], bad["experts"], bad["width"], bad["type"], bad["first"],
                       bad["align"], bad["capacity"])


def test_row_plan_limits_are_inclusive(hc):
    assert hc.cutt_hostcheck_rows_shape(0, 1, 1, 0, 1, 1, 1, 0) == 0
    assert hc.cutt_hostcheck_rows_shape(1 << 30, 1, 4096, 0x7fffffff - 4096, 4096, 1 << 30, 1 << 24, 3) == 0


@pytest.mark.parametrize("shape", [(0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, -1), (1 << 15, 1, 1 << 15, 1),
                                   (1, (1 << 30) + 1, 1, 1), (1, 1, 1, (1 << 30) + 1)])
def test_page_plan_refusals(native, hc, shape):
    assert hc.cutt_hostcheck_pages_shape(*shape) == BAD
    h = ctypes.c_uint(0)
    assert native.lib().cutt_pages_plan(ctypes.byref(h), *shape, None) == BAD
    assert native.lib().cutt_pages_plan(None, 1, 1, 1, 1, None) == BAD


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(heads=0), dict(size=0), dict(elt=0), dict(elt=3), dict(elt=16), dict(pages=0), dict(page=0),
    dict(slot=15), dict(head=15), dict(pstride=15), dict(pstride=1 << 60), dict(slot=1 << 60), dict(head=1 << 60),
    dict(slot=-16), dict(heads=(1 << 16) + 1), dict(heads=1 << 16, size=1 << 9, slot=1 << 9, head=1 << 9)])
def test_paged_plan_refusals(native, hc, change):
    good = dict(tokens=4, heads=2, size=16, elt=2, pages=3, page=8, pstride=256, slot=32, head=16)
    assert hc.cutt_hostcheck_paged_shape(*good.values()) == 0
    bad = dict(good, **change)
    assert hc.cutt_hostcheck_paged_shape(*bad.values()) == BAD
    h = ctypes.c_uint(0)
    assert native.lib().cutt_pages_plan_rows(ctypes.byref(h), *bad.values(), None) == BAD


def test_numbers_beyond_32_bits_are_refused_in_python(native):
    for make in (lambda: native.RowPlan(2**32 + 4, 1, 8, 16, 2), lambda: native.RowPlan(4, 1, 8, 2**32 + 16, 2),
                 lambda: native.PagePlan(1, 2**32 + 1, 4, 4), lambda: native.PagedRows(4, 1, 8, 2, 2**32 + 2, 8, 64, 8, 8)):
        with pytest.raises(native.CuttError) as e:
            make()
        assert e.value.code == BAD


def test_calls_on_unknown_handles(native):
    L = native.lib()
    for h in (0x80000000 + 12345, 3, 0xffffffff):
        assert L.cutt_rows_sort(h, 16, 4, 32, 48, 64, 80) == native.CUTT_INVALID_PLAN
        assert L.cutt_rows_dispatch(h, 16, 8, 32, 48, 64, 0, 80, 8) == native.CUTT_INVALID_PLAN
        assert L.cutt_rows_combine(h, 16, 8, 32, 0, 48, 8) == native.CUTT_INVALID_PLAN
        assert L.cutt_rows_dispatch_grad(h, 16, 8, 32, 0, 0, 8, 48, 8, 0) == native.CUTT_INVALID_PLAN
        assert L.cutt_rows_combine_grad(h, 16, 8, 32, 48, 64, 0, 0, 8, 80, 8, 0) == native.CUTT_INVALID_PLAN
        assert L.cutt_pages_build(h, 16, 32, 48, 64, 64, 80, 8, 96, 112, 128) == native.CUTT_INVALID_PLAN
        assert L.cutt_pages_store(h, 16, 0, 8, 8, 32, 48, 0) == native.CUTT_INVALID_PLAN
        assert L.cutt_pages_load(h, 16, 0, 32, 48, 0, 8, 8) == native.CUTT_INVALID_PLAN
        assert native.cuttExecute(h, 16, 32) == native.CUTT_INVALID_PLAN
    assert native.cuttDestroy(0x80000000 + 12345) == native.CUTT_INVALID_PLAN
    with pytest.raises(native.CuttError):
        native.plan_describe(0x80000000 + 12345)


def test_sort_refusals(hc):
    shape = _ints(4, 2, 8, 0, 1, 8, 16, 2)
    good = [64, 4, 128, 192, 256, 320]
    f = hc.cutt_hostcheck_rows_sort
    assert f(shape, *good) == 0
    assert f(shape, 64, 8, *good[2:]) == 0
    for size in (0, 1, 2, 16):
        assert f(shape, 64, size, *good[2:]) == BAD
    for i in (0, 2, 3, 4, 5):                       # null, misaligned, one address twice
        for value in (0, good[i] + 2, 64 if i else 128):
            assert f(shape, *[value if k == i else v for k, v in enumerate(good)]) == BAD
    assert f(shape, 68, 8, *good[2:]) == BAD        # 64-bit indices on a 4-byte boundary
    empty = _ints(0, 2, 8, 0, 1, 8, 16, 2)
    assert f(empty, 0, 4, 128, 192, 0, 320) == 0


def test_move_refusals(hc):
    f = hc.cutt_hostcheck_rows_move
    shape = _ints(4, 2, 8, 0, 1, 8, 16, 2)
    names = ["token", "tokenStride", "row", "rowStride", "rowOf", "count", "offset", "weight", "other", "otherStride", "dweight", "rowsOut"]
    good = dict(zip(names, [64, 16, 128, 16, 192, 256, 320, 0, 0, 0, 0, 1]))

    def rc(shape=shape, **change):
        return f(shape, *dict(good, **change).values())

    assert rc() == 0 and rc(rowsOut=0) == 0
    assert rc(tokenStride=0) == 0                    # one row for all tokens
    assert rc(rowsOut=0, rowStride=0) == 0
    for change in (dict(token=0), dict(row=0), dict(rowOf=0), dict(count=0), dict(offset=0), dict(row=64), dict(token=65),
                   dict(row=129), dict(rowOf=194), dict(weight=386), dict(rowStride=15), dict(tokenStride=-1),
                   dict(rowsOut=0, tokenStride=15), dict(rowsOut=0, rowStride=-16), dict(dweight=384), dict(other=384, otherStride=16),
                   dict(other=128, otherStride=16, dweight=384), dict(weight=384, other=512, otherStride=16, dweight=384),
                   dict(other=512, otherStride=-1, dweight=384), dict(other=513, otherStride=16, dweight=384),
                   dict(rowStride=1 << 60), dict(tokenStride=1 << 60)):
        assert rc(**change) == BAD, change
    assert rc(weight=384, other=512, otherStride=0, dweight=640) == 0
    # 1-byte rows are moved as they are: no weights, no sums
    b = _ints(4, 2, 8, 0, 1, 8, 16, 0)
    assert rc(b) == 0 and rc(b, token=65) == 0
    assert rc(b, weight=384) == BAD and rc(b, rowsOut=0) == BAD
    assert rc(_ints(0, 2, 8, 0, 1, 8, 16, 2), token=0, rowOf=0) == 0


@pytest.mark.parametrize("rows_out", [0, 1])
def test_moves_refuse_an_output_that_is_also_given_elsewhere(hc, rows_out):
    f = hc.cutt_hostcheck_rows_move
    shape = _ints(4, 2, 8, 0, 1, 8, 16, 2)
    names = ["token", "tokenStride", "row", "rowStride", "rowOf", "count", "offset", "weight", "other", "otherStride", "dweight", "rowsOut"]
    good = dict(zip(names, [64, 16, 128, 16, 192, 256, 320, 384, 448, 16, 512, rows_out]))
    pointers = ["token", "row", "rowOf", "count", "offset", "weight", "other", "dweight"]
    assert f(shape, *good.values()) == 0
    outputs = {"row" if rows_out else "token", "dweight"}
    for out in outputs:
        for name in pointers:
            if name != out:
                assert f(shape, *dict(good, **{out: good[name]}).values()) == BAD, (out, name)
    inputs = [n for n in pointers if n not in outputs and n not in ("token", "row")]
    for a in inputs:                                  # inputs may be shared
        for b in inputs:
            assert f(shape, *dict(good, **{a: good[b]}).values()) == 0, (a, b)


def test_paged_moves_refuse_an_output_that_is_also_given_elsewhere(hc):
    f = hc.cutt_hostcheck_paged_move
    shape, strides = _ints(4, 2, 16, 2, 3, 8), (ctypes.c_longlong * 3)(256, 32, 16)
    names = ["k", "v", "tokenStride", "headStride", "slot", "kCache", "vCache", "rowsOut"]
    for rows_out, outputs in ((0, ("kCache", "vCache")), (1, ("k", "v"))):
        good = dict(zip(names, [64, 128, 32, 16, 192, 256, 320, rows_out]))
        assert f(shape, strides, *good.values()) == 0
        for out in outputs:
            for name in ("k", "v", "slot", "kCache", "vCache"):
                if name != out:
                    assert f(shape, strides, *dict(good, **{out: good[name]}).values()) == BAD, (out, name)


def test_calls_of_no_tokens_take_empty_tensors(hc):
    """An empty tensor has the null address; the row side and the caches are there all the same."""
    f = hc.cutt_hostcheck_rows_move
    empty = _ints(0, 2, 8, 0, 4, 8, 16, 2)
    # dispatch; the gradient of combine with the weights' gradient; combine; the gradient of dispatch
    assert f(empty, 0, 16, 128, 16, 0, 256, 320, 0, 0, 0, 0, 1) == 0
    assert f(empty, 0, 16, 128, 16, 0, 256, 320, 0, 512, 16, 0, 1) == 0
    assert f(empty, 0, 16, 0, 16, 0, 256, 320, 0, 0, 0, 0, 1) == BAD         # the rows are written
    assert f(empty, 0, 16, 128, 16, 0, 0, 320, 0, 0, 0, 0, 1) == BAD
    g = hc.cutt_hostcheck_paged_move
    shape, strides = _ints(0, 2, 16, 2, 3, 8), (ctypes.c_longlong * 3)(256, 32, 16)
    for rows_out in (0, 1):
        assert g(shape, strides, 0, 0, 32, 16, 0, 256, 320, rows_out) == 0
        assert g(shape, strides, 0, 0, 32, 16, 0, 256, 0, rows_out) == 0
        assert g(shape, strides, 0, 0, 32, 16, 0, 0, 320, rows_out) == BAD
        assert g(shape, strides, 0, 0, 15, 16, 0, 256, 320, 1) == BAD


def test_build_refusals(hc):
    f = hc.cutt_hostcheck_pages_build
    shape = _ints(4, 16, 8, 64)
    names = ["held", "added", "free", "poolIn", "poolOut", "table", "stride", "tokenOffset", "pageOffset", "slot"]
    good = dict(zip(names, [64, 128, 192, 256, 256, 320, 8, 384, 448, 512]))

    def rc(**change):
        return f(shape, *dict(good, **change).values())

    assert rc() == 0 and rc(poolOut=640) == 0 and rc(stride=9) == 0
    assert rc(free=0, poolIn=0, poolOut=0, pageOffset=0) == 0
    for change in (dict(held=0), dict(added=0), dict(table=0), dict(tokenOffset=0), dict(slot=0), dict(free=0), dict(poolIn=0),
                   dict(poolOut=0), dict(pageOffset=0), dict(stride=7), dict(stride=1 << 58), dict(table=64), dict(tokenOffset=128),
                   dict(pageOffset=384), dict(slot=192), dict(poolOut=64), dict(poolOut=260), dict(poolOut=252), dict(slot=516), dict(held=66), dict(table=322)):
        assert rc(**change) == BAD, change


def test_paged_refusals(hc):
    f = hc.cutt_hostcheck_paged_move
    shape, strides = _ints(4, 2, 16, 2, 3, 8), (ctypes.c_longlong * 3)(256, 32, 16)
    names = ["k", "v", "tokenStride", "headStride", "slot", "kCache", "vCache", "rowsOut"]
    good = dict(zip(names, [64, 128, 32, 16, 192, 256, 320, 0]))

    def rc(**change):
        return f(shape, strides, *dict(good, **change).values())

    assert rc() == 0 and rc(rowsOut=1) == 0 and rc(v=0, vCache=0) == 0
    assert rc(tokenStride=0) == 0 and rc(headStride=0) == 0 and rc(v=64) == 0    # inputs may be shared
    for change in (dict(k=0), dict(kCache=0), dict(slot=0), dict(v=0), dict(vCache=0), dict(k=256), dict(v=320), dict(v=256), dict(k=320),
                   dict(vCache=256), dict(k=65), dict(vCache=321), dict(slot=196), dict(tokenStride=-1), dict(headStride=-1),
                   dict(rowsOut=1, tokenStride=15), dict(rowsOut=1, headStride=15), dict(rowsOut=1, v=64), dict(tokenStride=1 << 60)):
        assert rc(**change) == BAD, change


def plain_build(held, added, page, width, free, pool, table, m):
    """cutt_pages_build in Python numbers."""
    held, added = [max(0, int(x)) for x in held], [max(0, int(x)) for x in added]
    table = [list(map(int, r)) for r in table]
    at, limit = (max(0, int(pool[0])), max(0, int(pool[1]))) if free is not None else (0, 0)
    first, slots, tokens, pages = at, [-1] * m, [0], [at]
    for b in range(len(held)):
        have, want = -(-held[b] // page), min(-(-(held[b] + added[b]) // page), width)
        got = {}
        if free is not None:
            for i in range(have, want):
                got[i] = int(free[at]) if at < limit else -1
                table[b][i] = got[i]
                at += 1
        for i in range(min(added[b], max(0, m - tokens[-1]))):
            idx, off = divmod(held[b] + i, page)
            p = -1 if idx >= width else table[b][idx]
            slots[tokens[-1] + i] = p * page + off if p >= 0 else -1
        tokens.append(tokens[-1] + added[b])
        pages.append(at)
    tokens = [min(t, 0x7fffffff) for t in tokens]
    return table, tokens, pages, slots, [min(at, max(limit, first)), int(pool[1]) if free is not None else 0]


def run_build(hc, held, added, page, width, free, pool, table, m):
    held, added = np.asarray(held, np.int32), np.asarray(added, np.int32)
    b = len(held)
    table = np.ascontiguousarray(table, np.int32).copy()
    tok, pag = np.full(b + 1, -7, np.int32), np.full(b + 1, -7, np.int32)
    slot, out = np.full(max(1, m), -7, np.int64), np.full(2, -7, np.int32)
    take = free is not None
    free = np.asarray(free if take else [0], np.int32)
    pool = np.asarray(pool, np.int32)
    p = lambda a: a.ctypes.data
    bad = hc.cutt_hostcheck_pages_run(b, page, width, m, p(held), p(added), p(free) if take else None, len(free),
                                      p(pool) if take else None, p(out) if take else None, p(table), table.shape[1], p(tok),
                                      p(pag) if take else None, p(slot))
    assert bad == 0
    return table.tolist(), tok.tolist(), pag.tolist(), slot[:m].tolist(), out.tolist()


def test_block_tables_and_slots_against_plain(hc):
    rng = random.Random(5)
    for _ in range(300):
        b, page, width = rng.randint(1, 9), rng.choice([1, 2, 3, 8, 16, 24]), rng.randint(1, 12)
        top = page * width
        held = [rng.choice([0, rng.randint(0, top), top, rng.randint(0, top), -3]) for _ in range(b)]
        added = [rng.choice([0, 1, 1, rng.randint(0, top), -1, top + 5]) for _ in range(b)]
        n = rng.randint(1, 60)
        free = rng.sample(range(1000), n)
        pool = [rng.randint(0, n), rng.choice([n, n, n // 2])]
        table = [[rng.choice([-1, rng.randint(2000, 3000)]) for _ in range(width + 1)] for _ in range(b)]
        m = rng.choice([0, 1, 7, 64, 500])
        got = run_build(hc, held, added, page, width, free, pool, table, m)
        want = plain_build(held, added, page, width, free, pool, table, m)
        assert got == tuple(want), (held, added, page, width, pool, m)
        got = run_build(hc, held, added, page, width, None, pool, table, m)
        want = plain_build(held, added, page, width, None, pool, table, m)
        assert got[0] == want[0] and got[1] == want[1] and got[3] == want[3]


def test_block_tables_at_the_ends_of_the_ranges(hc):
    big = 0x7fffffff
    # lengths whose sums pass 32 bits: offsets saturate, tokens beyond the table have no slot
    got = run_build(hc, [big, big, 5], [big, big, 2], 1 << 28, 3, [4, 5, 6], [0, 3], [[1, 2, 3]] * 3, 4)
    assert got[1] == [0, big, big, big]
    assert got[3] == [-1, -1, -1, -1]            # the first request lies beyond its table
    # positions just below 2^31 in pages of one token
    got = run_build(hc, [9], [3], 1, 11, [70, 71, 72], [0, 3], [list(range(100, 111))], 3)
    assert got[0] == [[100, 101, 102, 103, 104, 105, 106, 107, 108, 70, 71]]
    assert got[3] == [70, 71, -1]
    # a pool that is used up, negative words, next beyond the entries
    got = run_build(hc, [0], [4], 2, 4, [8, 9], [-5, 1], [[-1] * 4], 4)
    assert got[0] == [[8, -1, -1, -1]] and got[3] == [16, 17, -1, -1] and got[4] == [1, 1] and got[2] == [0, 2]
    got = run_build(hc, [0], [4], 2, 4, [8, 9], [2, 1], [[-1] * 4], 4)
    assert got[3] == [-1] * 4 and got[4] == [2, 1] and got[2] == [2, 4]
    # slots that pass 32 bits
    got = run_build(hc, [1 << 20], [1], 1 << 20, 2, [1 << 15], [0, 1], [[3, -1]], 1)
    assert got[3] == [1 << 35]


@pytest.mark.parametrize("b", [31, 32, 33, 513, 1024, 1025, 2500])
def test_offsets_of_many_requests(hc, b):
    """Scans over several warps and blocks, with sums that pass 2^31 - 1 at every place of a warp."""
    rng = random.Random(b)
    for scale in (5, 2**31 // b, 2**31 // 40, 2**31 - 1):
        held = [rng.randint(0, 40) for _ in range(b)]
        added = [rng.choice([0, rng.randint(0, scale), scale]) for _ in range(b)]
        page, width, m = 16, 6, 700
        free = list(range(9000, 9000 + 3 * b))
        table = [[rng.randint(0, 99) for _ in range(width)] for _ in range(b)]
        got = run_build(hc, held, added, page, width, free, [1, 3 * b], table, m)
        assert got == tuple(plain_build(held, added, page, width, free, [1, 3 * b], table, m))


def test_cache_offsets_and_bad_slots(hc):
    f = hc.cutt_hostcheck_cache_offset
    for pages, page, ps, ss in ((7, 16, 4096, 256), (3, 24, 24 * 100, 100), (1 << 20, 1 << 14, 1 << 20, 64), (5, 1, 9, 9)):
        n = pages * page
        for slot in (0, 1, page - 1, page, n // 2 + 1, n - 1):
            want = (slot // page) * ps + (slot % page) * ss if 0 <= slot < n else -1
            assert f(pages, page, ps, ss, slot) == want
        for slot in (-1, -2**63, n, n + 1, 2**63 - 1):
            assert f(pages, page, ps, ss, slot) == -1


def test_local_expert(hc):
    f = hc.cutt_hostcheck_local_expert
    assert [f(e, 4, 3) for e in (-1, 3, 4, 6, 7)] == [-1, -1, 0, 2, -1]
    for e in (2**63 - 1, -2**63, 2**32 + 4, 2**31):
        assert f(e, 4, 3) == -1


@pytest.mark.parametrize("most", [8, 16])
def test_launch_of_the_map_fits_any_cluster(hc, most):
    """Every number of slots is covered, in clusters of at most `most` blocks, within a block's shared memory, and a
    block's ranks fit their bits."""
    out = (ctypes.c_int * 4)()
    for experts in (1, 7, 64, 256, 384, 1024, 2047, 4096):
        for n in (0, 1, 31, 32, 33, 512, 513, 1024, 1025, 2048, 2049, 4096, 8191, 30000, 65535, 65536):
            hc.cutt_hostcheck_sort_shape(n, experts, most, out)
            blocks, slots, warps, words = out
            assert 1 <= blocks <= most and blocks & (blocks - 1) == 0 and 1 <= warps <= 16
            assert blocks * slots >= n and slots % 32 == 0 and slots < 1 << 19
            assert words == 2 * slots + (2 * warps + 2) * experts + 3 * experts and words * 4 <= 216 * 1024
    hc.cutt_hostcheck_sort_shape(65537, 4096, most, out)
    assert out[0] == 0                                       # three kernels


@pytest.mark.parametrize("elt", [1, 2, 4, 8])
@pytest.mark.parametrize("heads,size,page,head_major,pad,shift", [
    (8, 128, 16, True, 0, 0), (1, 64, 1, False, 0, 0), (3, 33, 24, True, 0, 1), (2, 80, 64, False, 5, 0), (5, 1, 7, True, 1, 0),
    (1, 576, 64, False, 0, 0), (40, 128, 16, False, 0, 0), (8, 33, 16, False, 0, 0), (8, 33, 16, False, 0, 3), (3, 700, 4, False, 0, 0)])
def test_paged_accesses_on_the_host(hc, elt, heads, size, page, head_major, pad, shift):
    """Every access of the store and load kernels: inside the buffers, aligned, and the right element."""
    rng = np.random.default_rng(heads * 1000 + size)
    pages, n = 11, min(90, 11 * page - 3)
    wide = size + pad
    dt = {1: np.uint8, 2: np.uint16, 4: np.uint32, 8: np.uint64}[elt]

    def buffer(count):
        raw = np.zeros(count * elt + 64, np.uint8)
        at = -raw.ctypes.data % 16 + shift * elt
        return raw, raw[at:at + count * elt].view(dt)

    shape = (pages, heads, page, wide) if head_major else (pages, page, heads, wide)
    keep, flat = buffer(int(np.prod(shape)))
    flat[:] = rng.integers(0, 250, flat.size)
    keep2, rows = buffer(n * heads * wide)
    rows[:] = rng.integers(0, 250, rows.size)
    cache = flat.reshape(shape)
    view = cache.transpose(0, 2, 1, 3) if head_major else cache            # page, place, head, element
    strides = (ctypes.c_longlong * 3)(*[view.strides[k] // elt for k in (0, 1, 2)])
    slot = rng.permutation(pages * page)[:n].astype(np.int64)
    slot[::7] = -1
    slot[1], slot[2] = pages * page, 2**40
    live = [(q, s) for q, s in enumerate(slot.tolist()) if 0 <= s < pages * page]
    ints = _ints(n, heads, size, elt, pages, page)
    r3 = rows.reshape(n, heads, wide)
    for store in (1, 0):
        want_cache, want_rows = view.copy(), r3.copy()
        for q, s in live:
            if store:
                want_cache[s // page, s % page, :, :size] = r3[q, :, :size]
            else:
                want_rows[q, :, :size] = view[s // page, s % page, :, :size]
        assert hc.cutt_hostcheck_paged_run(ints, strides, heads * wide, wide, slot.ctypes.data, rows.ctypes.data, rows.nbytes,
                                           flat.ctypes.data, flat.nbytes, store) == 0
        assert np.array_equal(view, want_cache) and np.array_equal(r3, want_rows)
        rows[:] = rng.integers(0, 250, rows.size)


@pytest.mark.parametrize("elt,heads,size", [(2, 8, 128), (4, 3, 33), (1, 5, 1)])
def test_skipped_tokens_need_no_rows(hc, elt, heads, size):
    """Rows that end before the tokens whose slots are -1 or beyond the cache: nothing behind the end is touched."""
    pages, page, n, have = 6, 8, 40, 23
    dt = {1: np.uint8, 2: np.uint16, 4: np.uint32}[elt]
    rng = np.random.default_rng(size)
    cache = rng.integers(0, 250, (pages * page, heads, size)).astype(dt)
    rows = rng.integers(0, 250, (have, heads, size)).astype(dt)
    slot = np.full(n, -1, np.int64)
    slot[:have] = rng.permutation(pages * page)[:have]
    slot[have + 1], slot[have + 2] = pages * page, 2**50
    strides = (ctypes.c_longlong * 3)(page * heads * size, heads * size, size)
    ints = _ints(n, heads, size, elt, pages, page)
    for store in (1, 0):
        want_cache, want_rows = cache.copy(), rows.copy()
        if store:
            want_cache[slot[:have]] = rows
        else:
            want_rows[:] = cache[slot[:have]]
        assert hc.cutt_hostcheck_paged_run(ints, strides, heads * size, size, slot.ctypes.data, rows.ctypes.data, rows.nbytes,
                                           cache.ctypes.data, cache.nbytes, store) == 0
        assert np.array_equal(cache, want_cache) and np.array_equal(rows, want_rows)
        rows[:] = rng.integers(0, 250, rows.shape)
