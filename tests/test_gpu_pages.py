"""Block tables, slot maps and paged rows on the GPU (cutt_pages_* of include/cutt_rows.h): whole
numbers and moved bytes, so everything is compared exactly."""
import pytest

from test_gpu_rows import few_sms  # noqa: F401 (a fixture)
from test_rows_host import plain_build

pytestmark = pytest.mark.gpu


class Build:
    def __init__(self, native, held, added, page, width, free, pool, m, extra=0):
        import torch
        self.torch = torch
        i32 = dict(dtype=torch.int32, device="cuda")
        b = len(held)
        self.args = (page, width, m)
        self.held, self.added = torch.tensor(held, **i32), torch.tensor(added, **i32)
        self.free, self.pool = torch.tensor(free, **i32), torch.tensor(pool, **i32)
        self.table = torch.arange(b * (width + extra), **i32).view(b, width + extra) % 5000 - 1
        self.tokens, self.pages = torch.full((b + 1,), -7, **i32), torch.full((b + 1,), -7, **i32)
        self.slot = torch.full((m + 4,), -7, dtype=torch.int64, device="cuda")
        self.plan = native.PagePlan(b, page, width, m, stream=torch.cuda.current_stream().cuda_stream)

    def want(self, take=True):
        page, width, m = self.args
        return plain_build(self.held.tolist(), self.added.tolist(), page, width, self.free.tolist() if take else None,
                           self.pool.tolist(), self.table.tolist(), m)

    def build(self, pool_out=None):
        self.plan.build(self.held.data_ptr(), self.added.data_ptr(), self.free.data_ptr(), self.pool.data_ptr(),
                        (self.pool if pool_out is None else pool_out).data_ptr(), self.table.data_ptr(), self.tokens.data_ptr(), self.pages.data_ptr(),
                        self.slot.data_ptr(), table_stride=self.table.stride(0))

    def check(self, want):
        m = self.args[2]
        assert self.table.tolist() == want[0]
        assert self.tokens.tolist() == want[1]
        assert self.pages.tolist() == want[2]
        assert self.slot.tolist() == want[3] + [-7] * 4
        assert self.pool.tolist() == want[4]


def lengths(b, top, seed, decode):
    import random
    rng = random.Random(seed)
    held = [rng.choice([0, rng.randint(0, top), top - 1]) for _ in range(b)]
    added = [1 if decode else rng.choice([0, 0, 1, rng.randint(0, 3 * top // 4)]) for _ in range(b)]
    return held, added


@pytest.mark.parametrize("b,page,width,decode", [
    (1, 16, 4, True), (1, 1, 50, False), (3, 24, 9, False), (33, 16, 20, True), (257, 8, 6, False), (1024, 16, 3, True),
    (1025, 64, 2, True), (3000, 3, 4, False), (8, 128, 40, False), (2, 16, 3000, False)])
def test_build(native, b, page, width, decode):
    held, added = lengths(b, page * width, b + page, decode)
    need = sum(max(0, min(-(-(h + a) // page), width) - -(-h // page)) for h, a in zip(held, added))
    total = sum(added)
    for spare, short, extra in ((3, 0, 0), (0, max(1, need // 3), 2), (-1, 0, 0)):
        n = 5 + max(0, need - short)
        c = Build(native, held, added, page, width, list(range(7000, 7000 + n)), [5, n], max(0, total + spare), extra)
        want, table = c.want(), c.table.clone()
        apart = c.torch.zeros_like(c.pool)
        c.build(apart)                                       # into another pool, then in place
        assert apart.tolist() == want[4] and c.table.tolist() == want[0] and c.slot.tolist() == want[3] + [-7] * 4
        c.table.copy_(table)
        c.slot.fill_(-7)
        c.build()
        c.check(want)
        # the same lengths over the table as it is now, without taking pages
        m = c.args[2]
        want = c.want(take=False)
        c.slot.fill_(-7)
        c.plan.slots(c.held.data_ptr(), c.added.data_ptr(), c.table.data_ptr(), c.tokens.data_ptr(), c.slot.data_ptr(),
                     table_stride=c.table.stride(0))
        assert c.slot.tolist() == want[3] + [-7] * 4 and c.table.tolist() == want[0] and c.tokens.tolist() == want[1]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("b,m", [(1, 300000), (300, 200000), (40, 65537), (5000, 30000), (4096, 5000), (7, 16384), (7, 16385)])
def test_build_of_long_steps(native, b, m, in_place):
    import random
    rng = random.Random(m)
    cut = sorted(rng.randint(0, m - 100) for _ in range(b - 1))
    added = [y - x for x, y in zip([0] + cut, cut + [m - 100])]
    held = [rng.randint(0, 1000) for _ in range(b)]
    page = 48
    width = max(-(-(h + a) // page) for h, a in zip(held, added))
    n = sum(-(-(h + a) // page) for h, a in zip(held, added)) + 1
    c = Build(native, held, added, page, width, rng.sample(range(10 * n), n), [0, n], m)
    want = c.want()
    before = c.pool.clone()
    out = c.pool if in_place else c.torch.zeros_like(c.pool)
    c.build(out)
    if not in_place:
        assert c.torch.equal(c.pool, before)
        c.pool = out
    c.check(want)


@pytest.mark.parametrize("m", [3000, 16384, 20000])
def test_build_in_place_in_a_context_of_few_sms(native, few_sms, m):  # noqa: F811
    b, page = 5, 16
    added = [m // b] * b
    width = -(-added[0] // page) + 2
    c = Build(native, [0, 3, 16, 17, 40], added, page, width, list(range(5000, 5000 + b * width)), [2, b * width], m)
    c.plan = native.PagePlan(b, page, width, m, stream=few_sms)
    if 8192 < m <= 16384:
        assert '"cluster": 8' in c.plan.describe()
    want = c.want()
    c.torch.cuda.synchronize()
    c.build()
    c.torch.cuda.synchronize()
    c.check(want)


def test_long_build_captured_with_the_pool_in_place(native):
    """Two kernels in a CUDA graph; every replay takes pages from where the last one stopped."""
    import torch
    side = torch.cuda.Stream()
    b, m = 9, 20000
    with torch.cuda.stream(side):
        c = Build(native, [0] * b, [0] * b, 16, 400, list(range(9000, 9000 + 4000)), [0, 4000], m)
        c.build()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.build()
    held = [0] * b
    for added in ([100, 0, 3000, 7, 1, 900, 16, 31, 2], [1] * b, [0] * b, [5000, 1, 1, 0, 0, 3, 2000, 15, 1]):
        c.held.copy_(torch.tensor(held, dtype=torch.int32))
        c.added.copy_(torch.tensor(added, dtype=torch.int32))
        torch.cuda.synchronize()
        want = c.want()
        graph.replay()
        torch.cuda.synchronize()
        c.check(want)
        held = [x + y for x, y in zip(held, added)]


@pytest.mark.parametrize("b,n,steps", [(6, 1, 300), (40, 300, 25), (3, 9000, 4)])
def test_steps_without_a_pause(native, b, n, steps):
    """Tables, stores and loads one behind the other with nothing between them; errors counted on the device."""
    import torch
    page, heads, size = 8, 2, 16
    m = b * n
    width = -(-n * steps // page) + 1
    pages = b * width + 1
    c = Build(native, [0] * b, [n] * b, page, width, list(range(1, pages)), [0, pages - 1], m)
    rows = native.PagedRows(m, heads, size, 4, pages, page, heads * page * size, size, page * size,
                            stream=torch.cuda.current_stream().cuda_stream)
    cache, src, back = torch.zeros(pages, heads, page, size, device="cuda"), torch.randn(m, heads, size, device="cuda"), torch.zeros(m, heads, size, device="cuda")
    wrong = torch.zeros(1, dtype=torch.int64, device="cuda")
    for i in range(steps):
        src.add_(1.0)
        c.build()
        rows.store(src.data_ptr(), 0, c.slot.data_ptr(), cache.data_ptr(), 0)
        rows.load(cache.data_ptr(), 0, c.slot.data_ptr(), back.data_ptr(), 0)
        c.held.add_(n)
        wrong += (back != src).any() + (c.slot[:m] < 0).any() + (c.slot[:m].sort().values.diff() == 0).any()
    assert wrong.item() == 0
    taken = b * -(-n * steps // page)
    assert c.pool.tolist() == [taken, pages - 1]
    used = c.table[:, :-(-n * steps // page)]
    assert used.unique().numel() == taken


def test_build_of_empty_and_odd_lengths(native):
    for held, added in (([0, 0, 0], [0, 0, 0]), ([0], [0]), ([-5, 7, -1], [3, -9, 0]), ([100, 32, 31], [5, 1, 2])):
        c = Build(native, held, added, 8, 4, list(range(50, 70)), [2, 20], 9)
        want = c.want()
        c.build()
        c.check(want)
    c = Build(native, [0, 3], [4, 1], 8, 4, list(range(50, 70)), [2, 20], 0)     # no room for slots
    want = c.want()
    c.build()
    c.check(want)
    big = 2**31 - 1
    c = Build(native, [big, 3], [big, big], 1 << 20, 2, [50, 51, 52], [0, 3], 9)  # sums beyond 32 bits
    want = c.want()
    c.build()
    c.check(want)


def _views(cache, head_major):
    """(slots, heads, size) view of a cache."""
    return cache.transpose(1, 2) if head_major else cache


@pytest.mark.parametrize("elt", [1, 2, 4, 8])
@pytest.mark.parametrize("heads,size,page,head_major,pad", [
    (8, 128, 16, True, 0), (1, 64, 1, False, 0), (3, 33, 24, True, 0), (2, 80, 64, False, 5), (5, 1, 7, True, 1), (1, 576, 64, False, 0),
    (40, 128, 16, False, 0)])
def test_store_and_load(native, elt, heads, size, page, head_major, pad):
    import torch
    dt = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[elt]
    pages, n = 11, min(150, 11 * page - 3)
    g = torch.Generator(device="cuda").manual_seed(elt)
    rand = lambda *s: torch.randint(0, 200, s, device="cuda", generator=g, dtype=dt)
    shape = (pages, heads, page, size + pad) if head_major else (pages, page, heads, size + pad)
    caches = [rand(*shape) for _ in range(2)]
    views = [_views(c, head_major)[..., :size] for c in caches]            # (pages, page, heads, size)
    strides = [views[0].stride(i) for i in (0, 1, 2)]
    qkv = rand(n, 3 * heads, size + pad)
    k, v = qkv[:, heads:2 * heads, :size], qkv[:, 2 * heads:, :size]
    slot = torch.randperm(pages * page, device="cuda", generator=g)[:n]
    slot[::7] = -1
    if n > 20:
        slot[3], slot[5], slot[9] = pages * page, 2**40, -2**50             # not slots of this cache
    ok = (slot >= 0) & (slot < pages * page)
    plan = native.PagedRows(n, heads, size, elt, pages, page, *strides, stream=torch.cuda.current_stream().cuda_stream)
    for both in (True, False):
        before = [c.clone() for c in caches]
        plan.store(k.data_ptr(), v.data_ptr() if both else 0, slot.data_ptr(), caches[0].data_ptr(),
                   caches[1].data_ptr() if both else 0, token_stride=qkv.stride(0), head_stride=qkv.stride(1))
        for c, old, new, used in ((caches[0], before[0], k, True), (caches[1], before[1], v, both)):
            if used:
                w = _views(old, head_major)
                w[slot[ok] // page, slot[ok] % page, :, :size] = new[ok]
            assert torch.equal(c, old)
        outs = [rand(n, heads, size + pad) for _ in range(2)]
        olds = [o.clone() for o in outs]
        plan.load(caches[0].data_ptr(), caches[1].data_ptr() if both else 0, slot.data_ptr(), outs[0].data_ptr(),
                  outs[1].data_ptr() if both else 0, token_stride=outs[0].stride(0), head_stride=outs[0].stride(1))
        for o, old, c, used in ((outs[0], olds[0], caches[0], True), (outs[1], olds[1], caches[1], both)):
            if used:
                old[ok, :, :size] = _views(c, head_major)[slot[ok] // page, slot[ok] % page, :, :size]
            assert torch.equal(o, old)
        k, v = v, k


@pytest.mark.parametrize("elt,heads,size", [(2, 8, 128), (2, 16, 36), (4, 8, 33), (2, 8, 33), (1, 9, 57)])      # 16, 8, 4, 2, 1 bytes
@pytest.mark.parametrize("have", [9000, 8111])
def test_store_of_many_rows(native, elt, heads, size, have):
    """Stores of more blocks than the device holds at once, with slots that are none and rows that end early."""
    import torch
    dt = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[elt]
    n, page = 9000, 16
    pages = -(-n // page) + 3
    g = torch.Generator(device="cuda").manual_seed(size)
    rand = lambda *s: torch.randint(0, 200, s, device="cuda", generator=g, dtype=dt)
    caches = [rand(pages, heads, page, size) for _ in range(2)]
    rows = [rand(have, heads, size) for _ in range(2)]
    slot = torch.randperm(pages * page, device="cuda", generator=g)[:n]
    slot[::11] = -1
    slot[have:] = pages * page
    slot = slot.contiguous()
    ok = slot[:have] >= 0
    want = [c.clone() for c in caches]
    for w, r in zip(want, rows):
        w.transpose(1, 2)[slot[:have][ok] // page, slot[:have][ok] % page] = r[ok]
    p = native.PagedRows(n, heads, size, elt, pages, page, heads * page * size, size, page * size,
                         stream=torch.cuda.current_stream().cuda_stream)
    p.store(rows[0].data_ptr(), rows[1].data_ptr(), slot.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr())
    assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])


@pytest.mark.parametrize("size", [64, 33])
def test_rows_end_before_skipped_tokens(native, size):
    """A batch shorter than the plan's tokens: the slots behind its last row are -1."""
    import torch
    n, have, pages, page, heads = 300, 37, 9, 8, 4
    cache = torch.zeros(pages, page, heads, size, device="cuda")
    k = torch.randn(have, heads, size, device="cuda")
    slot = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    slot[:have] = torch.randperm(pages * page, device="cuda")[:have]
    p = native.PagedRows(n, heads, size, 4, pages, page, *cache.stride()[:3], stream=torch.cuda.current_stream().cuda_stream)
    p.store(k.data_ptr(), 0, slot.data_ptr(), cache.data_ptr(), 0)
    flat = cache.view(pages * page, heads, size)
    assert torch.equal(flat[slot[:have]], k) and flat.abs().sum((1, 2)).count_nonzero() == have
    back = torch.zeros_like(k)
    p.load(cache.data_ptr(), 0, slot.data_ptr(), back.data_ptr(), 0)
    assert torch.equal(back, k)


def test_one_row_to_many_slots_and_no_tokens(native):
    import torch
    cache = torch.zeros(4, 8, 2, 16, device="cuda")
    row = torch.randn(2, 16, device="cuda")
    slot = torch.tensor([3, 31, 8], device="cuda")
    p = native.PagedRows(3, 2, 16, 4, 4, 8, 256, 32, 16)
    torch.cuda.synchronize()
    p.store(row.data_ptr(), 0, slot.data_ptr(), cache.data_ptr(), 0, token_stride=0)
    torch.cuda.synchronize()
    flat = cache.view(32, 2, 16)
    assert torch.equal(flat[slot], row.expand(3, 2, 16)) and flat.abs().sum((1, 2)).count_nonzero() == 3
    none = native.PagedRows(0, 2, 16, 4, 4, 8, 256, 32, 16)
    none.store(row.data_ptr(), 0, slot.data_ptr(), cache.data_ptr(), 0)
    torch.cuda.synchronize()
    assert flat.abs().sum((1, 2)).count_nonzero() == 3


def test_no_tokens_as_empty_tensors(native):
    import torch
    caches = [torch.ones(4, 8, 2, 16, device="cuda") for _ in range(2)]
    row, slot = torch.zeros(0, 2, 16, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    assert row.data_ptr() == 0 and slot.data_ptr() == 0
    p = native.PagedRows(0, 2, 16, 4, 4, 8, 256, 32, 16)
    p.store(row.data_ptr(), row.data_ptr(), slot.data_ptr(), *[c.data_ptr() for c in caches])
    p.load(*[c.data_ptr() for c in caches], slot.data_ptr(), row.data_ptr(), row.data_ptr())
    torch.cuda.synchronize()
    assert all((c == 1).all() for c in caches)


def test_cache_offsets_beyond_32_bits(native):
    """A cache of more than 2^32 bytes: the last pages hold what was stored there."""
    import torch
    pages, page, heads, size = 1200, 64, 2, 128
    stride = 4 << 20                                       # elements (bytes) between pages
    cache = torch.zeros(pages * stride, dtype=torch.uint8, device="cuda")
    assert cache.numel() > 2**32
    slot = torch.tensor([0, pages * page - 1, 1100 * page + 5, 1030 * page], device="cuda")
    x = torch.randint(0, 255, (4, heads, size), device="cuda", dtype=torch.uint8)
    p = native.PagedRows(4, heads, size, 1, pages, page, stride, heads * size, size, stream=torch.cuda.current_stream().cuda_stream)
    p.store(x.data_ptr(), 0, slot.data_ptr(), cache.data_ptr(), 0)
    at = torch.as_strided(cache, (pages, page, heads, size), (stride, heads * size, size, 1))
    assert torch.equal(at[slot // page, slot % page], x)
    y = torch.zeros_like(x)
    p.load(cache.data_ptr(), 0, slot.data_ptr(), y.data_ptr(), 0)
    assert torch.equal(x, y)


def test_steps_of_a_server(native):
    """Everything together: prefill and decoding steps of several requests through one captured graph; at the
    end each request's rows, loaded back through its table, are what was stored."""
    import torch
    b, page, width, heads, size, m = 5, 8, 20, 2, 16, 64
    num_pages = 120
    side = torch.cuda.Stream()
    i32 = dict(dtype=torch.int32, device="cuda")
    held, added = torch.zeros(b, **i32), torch.zeros(b, **i32)
    g = torch.Generator().manual_seed(0)
    free = torch.randperm(num_pages, generator=g).int().cuda()
    pool = torch.tensor([0, num_pages], **i32)
    table = torch.full((b, width), -1, **i32)
    tokens, pages_at = torch.zeros(b + 1, **i32), torch.zeros(b + 1, **i32)
    slot = torch.zeros(m, dtype=torch.int64, device="cuda")
    k = torch.zeros(m, heads, size, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    caches = [torch.zeros(num_pages, heads, page, size, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    plan = native.PagePlan(b, page, width, m, stream=side.cuda_stream)
    rows = native.PagedRows(m, heads, size, 2, num_pages, page, heads * page * size, size, page * size, stream=side.cuda_stream)

    def step():
        plan.build(held.data_ptr(), added.data_ptr(), free.data_ptr(), pool.data_ptr(), pool.data_ptr(), table.data_ptr(),
                   tokens.data_ptr(), pages_at.data_ptr(), slot.data_ptr())
        rows.store(k.data_ptr(), v.data_ptr(), slot.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr())
        held.add_(added)

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()                                             # nothing added yet
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    kept = [[[], []] for _ in range(b)]
    for n in ([17, 0, 30, 1, 9], [1, 8, 1, 1, 1], [0, 50, 0, 7, 0], [1, 1, 1, 1, 1], [1, 1, 0, 1, 1], [40, 1, 1, 1, 15]):
        new_k, new_v = [torch.randn(m, heads, size, generator=g).bfloat16() for _ in range(2)]
        added.copy_(torch.tensor(n, dtype=torch.int32))
        k.copy_(new_k)
        v.copy_(new_v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for i, c in enumerate(n):
            kept[i][0].append(new_k[at:at + c])
            kept[i][1].append(new_v[at:at + c])
            at += c
    total = [sum(x.shape[0] for x in kept[i][0]) for i in range(b)]
    assert held.tolist() == total
    assert pool.tolist() == [sum(-(-t // page) for t in total), num_pages]
    used = table[table >= 0].tolist()
    assert len(used) == len(set(used)) == pool[0].item()
    # the whole context of all requests, token by token
    zero = torch.zeros(b, **i32)
    whole = native.PagePlan(b, page, width, sum(total) + 3)
    slots = torch.zeros(sum(total) + 3, dtype=torch.int64, device="cuda")
    whole.slots(zero.data_ptr(), held.data_ptr(), table.data_ptr(), tokens.data_ptr(), slots.data_ptr())
    outs = [torch.full((sum(total) + 3, heads, size), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    back = native.PagedRows(sum(total) + 3, heads, size, 2, num_pages, page, heads * page * size, size, page * size)
    back.load(caches[0].data_ptr(), caches[1].data_ptr(), slots.data_ptr(), outs[0].data_ptr(), outs[1].data_ptr())
    torch.cuda.synchronize()
    for j in range(2):
        want = torch.cat([x for i in range(b) for x in kept[i][j]])
        assert torch.equal(outs[j][:-3].cpu(), want)
        assert (outs[j][-3:] == 7).all()                   # behind the last token: left alone
