"""Rows sorted by expert, moved there and back, and the gradients, on the GPU against plain 64-bit
arithmetic (cutt_rows_* of include/cutt_rows.h).

Tolerances.  Every output is one rounding of a 32-bit result: half a step of the type relative to the
value, plus what the 32-bit arithmetic loses - a product or a sum of n terms by at most n + 1 roundings
of 2^-24 relative to the sum of the terms' magnitudes - plus half of the type's smallest step for values
near zero.  Moves without weights are exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134), "f32": (2.0 ** -24, 2.0 ** -150)}


def _types(native):
    import torch
    return {"bytes": (native.CUTT_ROWS_BYTES, torch.uint8), "f16": (native.CUTT_ROWS_F16, torch.float16),
            "bf16": (native.CUTT_ROWS_BF16, torch.bfloat16), "f32": (native.CUTT_ROWS_F32, torch.float32)}


def plain_map(ids, first, experts, align, capacity):
    """The map by its definition, slot by slot."""
    ids = [int(x) - first for x in ids]
    n = [0] * experts
    for e in ids:
        if 0 <= e < experts:
            n[e] += 1
    start, at = [], 0
    for e in range(experts):
        start.append(at)
        at += -(-n[e] // align) * align
    offset = [min(s, capacity) for s in start + [at]]
    count = [min(start[e] + n[e], capacity) - min(start[e], capacity) for e in range(experts)]
    row_of, slot_of, seen = [-1] * len(ids), [-1] * capacity, [0] * experts
    for s, e in enumerate(ids):
        if not 0 <= e < experts:
            continue
        r = start[e] + seen[e]
        seen[e] += 1
        if r < capacity:
            row_of[s], slot_of[r] = r, s
    return count, offset, row_of, slot_of


class Run:
    """Plan, map and device buffers of one routing."""

    def __init__(self, native, ids, width, kind, experts, first=0, align=1, capacity=None, index=None):
        import torch
        self.torch, self.C = torch, native
        t, k = ids.shape
        self.t, self.k, self.h, self.kind = t, k, width, kind
        self.code, self.dtype = _types(native)[kind]
        self.plan = native.RowPlan(t, k, experts, width, self.code, first=first, align=align, capacity=capacity,
                                   stream=torch.cuda.current_stream().cuda_stream)
        self.r, self.e = self.plan.capacity, experts
        self.ids = ids.to(index or torch.int32).cuda().contiguous()
        i32 = dict(dtype=torch.int32, device="cuda")
        self.count, self.offset = torch.full((experts,), -7, **i32), torch.full((experts + 1,), -7, **i32)
        self.row_of, self.slot_of = torch.full((t, k), -7, **i32), torch.full((self.r,), -7, **i32)
        self.want = plain_map(ids.reshape(-1).tolist(), first, experts, align, self.r)

    def sort(self):
        self.plan.sort(self.ids.data_ptr(), self.ids.element_size(), self.count.data_ptr(), self.offset.data_ptr(),
                       self.row_of.data_ptr(), self.slot_of.data_ptr())

    def check_map(self):
        got = (self.count.tolist(), self.offset.tolist(), self.row_of.reshape(-1).tolist(), self.slot_of.tolist())
        for name, g, w in zip(("count", "offset", "row_of", "slot_of"), got, self.want):
            assert g == w, name

    def maps(self):
        return self.row_of.data_ptr(), self.count.data_ptr(), self.offset.data_ptr()

    def rows(self, n, g, pad=0, shift=0):
        """n rows; `pad` elements between rows, the first `shift` elements behind an aligned address."""
        torch = self.torch
        flat = torch.randn(shift + n * (self.h + pad) + 8, generator=g)
        flat = (flat * 40).to(torch.uint8) if self.kind == "bytes" else flat.to(self.dtype)
        return flat.cuda()[shift:shift + n * (self.h + pad)].view(n, self.h + pad)[:, :self.h]

    def live(self):
        row = self.torch.tensor(self.want[2]).view(self.t, self.k)
        return row, row >= 0

    def padding(self):
        c, o = self.want[0], self.want[1]
        return [r for e in range(self.e) for r in range(o[e] + c[e], o[e + 1])]


def close(got, want, magnitude, terms, kind):
    rel, least = HALF[kind]
    got = got.double().cpu()
    tol = rel * want.abs() * 1.001 + (terms + 1) * 2.0 ** -24 * magnitude * 1.001 + least
    worst = ((got - want).abs() - tol).max().item() if got.numel() else -1
    assert worst <= 0, worst


def routing(t, k, e, seed, drop=0.0, first=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    k2 = min(k, e)
    ids = torch.rand(t, e, generator=g).topk(k2, dim=1).indices if t else torch.zeros(0, k2, dtype=torch.int64)
    if k > k2:                       # more choices than experts: experts come twice
        ids = torch.cat([ids, torch.randint(0, e, (t, k - k2), generator=g)], 1)
    ids = ids + first
    if drop:
        ids[torch.rand(t, k, generator=g) < drop] = first - 1
    return ids


MAPS = [(1, 1, 1, 1), (1, 8, 64, 1), (7, 3, 5, 4), (48, 6, 64, 1), (33, 8, 256, 16), (513, 4, 17, 128), (2000, 8, 384, 8),
        (40000, 2, 300, 64), (257, 10, 4096, 1), (3, 5, 2, 7)]


@pytest.mark.parametrize("t,k,e,align", MAPS)
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_map(native, t, k, e, align, drop):
    import torch
    r = Run(native, routing(t, k, e, t + e, drop, first=5), 8, "bf16", e, first=5, align=align,
            index=torch.int64 if t % 2 else torch.int32)
    r.sort()
    r.check_map()


def test_map_of_nothing_and_of_dropped_slots(native):
    import torch
    r = Run(native, torch.zeros(0, 4, dtype=torch.int64), 8, "bf16", 6, align=8, capacity=10)
    r.sort()
    r.check_map()
    assert r.slot_of.tolist() == [-1] * 10
    for value in (-1, 6, 2**31 - 1, -2**31, 2**62, -2**63):
        r = Run(native, torch.full((70, 2), value), 8, "bf16", 6, align=8, index=torch.int64 if abs(value) > 2**31 else torch.int32)
        r.sort()
        r.check_map()
        assert r.offset.tolist() == [0] * 7


@pytest.mark.parametrize("t,capacity", [(100, 1), (100, 63), (100, 200), (5000, 4096), (5000, 9999)])
def test_map_drops_what_does_not_fit(native, t, capacity):
    r = Run(native, routing(t, 2, 9, 3), 8, "bf16", 9, align=16, capacity=capacity)
    r.sort()
    r.check_map()


@pytest.mark.parametrize("t,k,e", [(30000, 2, 64), (131072, 1, 8), (20000, 8, 4096), (70001, 3, 129)])
def test_map_one_expert_for_all_and_long_ones(native, t, k, e):
    import torch
    r = Run(native, torch.full((t, k), e - 1), 8, "bf16", e, align=128)
    r.sort()
    r.check_map()
    r = Run(native, routing(t, k, e, 9, 0.1), 8, "bf16", e, align=128)
    r.sort()
    r.check_map()


def test_calls_of_no_tokens(native):
    """A step without tokens: empty tensors (null addresses); the calls succeed, rows keep what they hold."""
    import torch
    r = Run(native, torch.zeros(0, 2, dtype=torch.int64), 16, "f32", 4, align=8, capacity=16)
    x, w = torch.zeros(0, 16, device="cuda"), torch.zeros(0, 2, device="cuda")
    y, dy = torch.ones(16, 16, device="cuda"), torch.full((16, 16), 77.0, device="cuda")
    assert x.data_ptr() == 0
    r.sort()
    r.plan.dispatch(x.data_ptr(), *r.maps(), dy.data_ptr(), weight=w.data_ptr())
    r.plan.combine(y.data_ptr(), r.row_of.data_ptr(), x.data_ptr(), weight=w.data_ptr())
    r.plan.combine_grad(x.data_ptr(), *r.maps(), dy.data_ptr(), weight=w.data_ptr(), y=y.data_ptr(), dweight=w.data_ptr())
    r.plan.dispatch_grad(y.data_ptr(), r.row_of.data_ptr(), x.data_ptr(), weight=w.data_ptr(), x=x.data_ptr(), dweight=w.data_ptr())
    r.check_map()
    assert (dy == 77).all() and (y == 1).all()            # no segment has rows, so none is padded


@pytest.mark.parametrize("n,e,wide", [(1300001, 256, False), (2500000, 4096, True), (1 << 24, 60, False), (1 << 30, 300, False)])
def test_maps_up_to_the_limit(native, n, e, wide):
    """Maps whose chunks take several waves of blocks, up to 2^30 slots.  Checked on the device: counts, segments, each
    slot's row in its expert's segment, each row's slot the one that has it, and slots ascending in every segment -
    which together leave one map."""
    import torch
    align = 1 if n == 1 << 30 else 16
    capacity = n + e * (align - 1)
    g = torch.Generator(device="cuda").manual_seed(e)
    ids = torch.randint(0, e + 1, (n,), device="cuda", generator=g, dtype=torch.int64 if wide else torch.int32)   # e: dropped
    i32 = dict(dtype=torch.int32, device="cuda")
    count, offset = torch.full((e,), -7, **i32), torch.full((e + 1,), -7, **i32)
    row_of, slot_of = torch.full((n,), -7, **i32), torch.full((capacity,), -7, **i32)
    plan = native.RowPlan(n, 1, e, 8, native.CUTT_ROWS_BF16, align=align, capacity=capacity, stream=torch.cuda.current_stream().cuda_stream)
    plan.sort(ids.data_ptr(), ids.element_size(), count.data_ptr(), offset.data_ptr(), row_of.data_ptr(), slot_of.data_ptr())
    torch.cuda.synchronize()
    step = 1 << 26
    want = sum(torch.bincount(ids[a:a + step], minlength=e + 1) for a in range(0, n, step))[:e]
    assert torch.equal(count.long(), want)
    assert torch.equal(offset.long(), torch.cat([want.new_zeros(1), ((want + align - 1) // align * align).cumsum(0)]))
    first, end = torch.cat([offset[:e], offset.new_full((1,), -1)]), torch.cat([offset[:e] + count, offset.new_zeros(1)])
    for a in range(0, n, step):
        expert, row = ids[a:a + step].long(), row_of[a:a + step]
        live = expert < e
        assert ((row == -1) | live).all() and ((row >= first[expert]) & ((row < end[expert]) | ~live)).all()
        back = slot_of[row.clamp_min(0).long()]
        assert ((back == torch.arange(a, a + row.numel(), **i32)) | ~live).all()
        del expert, row, live, back
    held = 0
    for a in range(0, capacity, step):                # rows: a slot (ascending in its segment) or none
        slot = slot_of[a:a + step + 1]
        one, two = slot[:-1], slot[1:]
        at = torch.arange(a + 1, a + slot.numel(), **i32)
        starts = torch.isin(at, offset)
        assert ((two == -1) | (one < two) | starts).all()
        assert ((two == -1) | (one >= 0) | starts).all()
        held += (slot_of[a:a + step] >= 0).sum().item()
    assert held == want.sum().item()


SHAPES = [  # tokens, choices, experts, width, align, pad, shift, drop
    (1, 8, 16, 512, 1, 0, 0, 0.0), (5, 1, 3, 1, 1, 0, 0, 0.0), (48, 6, 64, 2048, 1, 8, 0, 0.0), (33, 3, 7, 1111, 1, 0, 0, 0.2),
    (64, 4, 16, 264, 16, 0, 1, 0.2), (17, 10, 12, 136, 128, 24, 0, 0.3), (300, 2, 8, 40, 8, 3, 0, 0.9), (6000, 5, 24, 72, 8, 0, 0, 0.1),
    (5000, 9, 24, 33, 1, 0, 0, 0.0), (9, 3, 2, 4100, 64, 0, 0, 0.0)]


@pytest.mark.parametrize("kind", ["bytes", "f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_dispatch(native, kind, shape):
    import torch
    t, k, e, h, align, pad, shift, drop = shape
    r = Run(native, routing(t, k, e, 11, drop), h, kind, e, align=align)
    r.sort()
    g = torch.Generator().manual_seed(1)
    x = r.rows(t, g, pad, shift)
    row, ok = r.live()
    for weighted in ([False] if kind == "bytes" else [False, True]):
        w = torch.randn(t, k, generator=g) if weighted else None
        y = torch.full((r.r, h + pad), 77, dtype=r.dtype, device="cuda")
        r.plan.dispatch(x.data_ptr(), *r.maps(), y.data_ptr(), weight=w.cuda().data_ptr() if weighted else 0,
                        x_stride=x.stride(0), y_stride=y.stride(0))
        assert (y[:, h:] == 77).all()                     # between the rows nothing is written
        got, xs = y[:, :h].cpu(), x.cpu()
        used = r.want[1][-1]
        assert (got[used:] == 77).all()                   # rows behind the last segment are left alone
        assert (got[r.padding()] == 0).all()
        src = xs[:, None, :].expand(t, k, h)[ok]
        if weighted:
            want = src.double() * w.double()[ok][:, None]
            close(got[row[ok].long()], want, want.abs(), 1, kind)
        else:
            assert torch.equal(got[row[ok].long()], src)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_combine(native, kind, shape):
    import torch
    t, k, e, h, align, pad, shift, drop = shape
    r = Run(native, routing(t, k, e, 12, drop), h, kind, e, align=align)
    r.sort()
    g = torch.Generator().manual_seed(2)
    y = r.rows(r.r, g, pad, shift)
    y[r.padding()] = float("nan")                         # rows that no slot owns are not read
    y[r.want[1][-1]:] = float("nan")
    row, ok = r.live()
    ys = y.double().cpu()
    parts = torch.where(ok[:, :, None], ys[row.clamp_min(0).long()], 0.0)
    for weighted in (False, True):
        w = torch.randn(t, k, generator=g) if weighted else torch.ones(t, k)
        w[~ok] = float("nan")                             # nor are their weights
        out = torch.full((t, h + pad), 77, dtype=r.dtype, device="cuda")
        r.plan.combine(y.data_ptr(), r.row_of.data_ptr(), out.data_ptr(), weight=w.cuda().data_ptr() if weighted else 0,
                       y_stride=y.stride(0), out_stride=out.stride(0))
        assert (out[:, h:] == 77).all()
        terms = torch.where(ok[:, :, None], parts * w.double()[:, :, None], 0.0)
        close(out[:, :h], terms.sum(1), terms.abs().sum(1), k, kind)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(native, kind, shape):
    import torch
    t, k, e, h, align, pad, shift, drop = shape
    r = Run(native, routing(t, k, e, 13, drop), h, kind, e, align=align)
    r.sort()
    g = torch.Generator().manual_seed(3)
    token, rows = r.rows(t, g, pad, shift), r.rows(r.r, g, pad, shift)
    rows[r.padding()] = float("nan")
    row, ok = r.live()
    ts, rs = token.double().cpu(), rows.double().cpu()
    parts = torch.where(ok[:, :, None], rs[row.clamp_min(0).long()], 0.0)
    products = parts * ts[:, None, :]
    for weighted in (False, True):
        w = torch.randn(t, k, generator=g)
        wd = w.double() if weighted else torch.ones(t, k, dtype=torch.float64)
        wp = w.cuda()
        for want_dw in (False, True):
            dw = torch.full((t, k), 77.0, device="cuda")
            # the gradient of combine: rows written, the token side read
            dy = torch.full((r.r, h + pad), 77, dtype=r.dtype, device="cuda")
            r.plan.combine_grad(token.data_ptr(), *r.maps(), dy.data_ptr(), weight=wp.data_ptr() if weighted else 0,
                                y=rows.data_ptr() if want_dw else 0, dweight=dw.data_ptr() if want_dw else 0,
                                dout_stride=token.stride(0), y_stride=rows.stride(0), dy_stride=dy.stride(0))
            got = dy[:, :h].cpu()
            assert (got[r.want[1][-1]:] == 77).all() and (dy[:, h:] == 77).all() and (got[r.padding()] == 0).all()
            want = (ts[:, None, :] * wd[:, :, None])[ok]
            close(got[row[ok].long()], want, want.abs() if weighted else want * 0, 1, kind)
            if want_dw:
                close(dw, products.sum(2), products.abs().sum(2), h, "f32")
                assert (dw.cpu()[~ok] == 0).all()
            # the gradient of dispatch: the token side written
            dx = torch.full((t, h + pad), 77, dtype=r.dtype, device="cuda")
            dw.fill_(77.0)
            r.plan.dispatch_grad(rows.data_ptr(), r.row_of.data_ptr(), dx.data_ptr(), weight=wp.data_ptr() if weighted else 0,
                                 x=token.data_ptr() if want_dw else 0, dweight=dw.data_ptr() if want_dw else 0,
                                 dy_stride=rows.stride(0), x_stride=token.stride(0), dx_stride=dx.stride(0))
            terms = parts * wd[:, :, None]
            close(dx[:, :h], terms.sum(1), terms.abs().sum(1), k, kind)
            assert (dx[:, h:] == 77).all()
            if want_dw:
                close(dw, products.sum(2), products.abs().sum(2), h, "f32")
                assert (dw.cpu()[~ok] == 0).all()
            else:
                assert (dw == 77).all()


@pytest.mark.parametrize("kind", ["bytes", "bf16", "f32"])
@pytest.mark.parametrize("t,k,h,shift", [(1300, 3, 1111, 0), (1300, 4, 2312, 0), (1200, 8, 4096, 0), (1200, 8, 4096, 3), (1190, 2, 4100, 1),
                                         (1500, 1, 2048, 0), (2500, 6, 520, 0), (1300, 9, 1023, 0), (300, 8, 8200, 0), (1200, 40, 72, 0)])
def test_every_launch_shape(native, kind, t, k, h, shift):
    """Tokens enough for every number of threads of a block; compared on the device in 64 bits."""
    import torch
    r = Run(native, routing(t, k, max(8, k // 2), 17, 0.3), h, kind, max(8, k // 2), align=8)
    r.sort()
    g = torch.Generator().manual_seed(5)
    token, rows = r.rows(t, g, 0, shift), r.rows(r.r, g, 0, shift)
    row = torch.tensor(r.want[2], device="cuda").view(t, k)
    ok = row >= 0
    y = torch.full((r.r, h), 77, dtype=r.dtype, device="cuda")
    r.plan.dispatch(token.data_ptr(), *r.maps(), y.data_ptr())
    assert torch.equal(y[row[ok]], token[:, None, :].expand(t, k, h)[ok])
    assert (y[r.want[1][-1]:] == 77).all() and (y[r.padding()] == 0).all()
    if kind == "bytes":
        return
    w = torch.randn(t, k, generator=g).cuda()
    ts = token.double()
    parts = torch.where(ok[:, :, None], rows.double()[row.clamp_min(0)], 0.0)
    dw = torch.full((t, k), 77.0, device="cuda")
    out = torch.full((t, h), 77, dtype=r.dtype, device="cuda")
    r.plan.combine(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr(), weight=w.data_ptr())
    terms = parts * w.double()[:, :, None]
    want, size = terms.sum(1).cpu(), terms.abs().sum(1).cpu()
    close(out, want, size, k, kind)
    out.fill_(77)
    r.plan.dispatch_grad(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr(), weight=w.data_ptr(), x=token.data_ptr(), dweight=dw.data_ptr())
    close(out, want, size, k, kind)
    products = parts * ts[:, None, :]
    want, size = products.sum(2).cpu(), products.abs().sum(2).cpu()
    close(dw, want, size, h, "f32")
    dw.fill_(77)
    y.fill_(77)
    r.plan.combine_grad(token.data_ptr(), *r.maps(), y.data_ptr(), weight=w.data_ptr(), y=rows.data_ptr(), dweight=dw.data_ptr())
    close(dw, want, size, h, "f32")
    want = (ts[:, None, :] * w.double()[:, :, None])[ok].cpu()
    close(y[row[ok]], want, want.abs(), 1, kind)
    assert (y[r.want[1][-1]:] == 77).all() and (y[r.padding()] == 0).all()


MANY = [  # more choices than a walk over the row takes at once (16 with the weights' gradient, 8 without)
    (50, 17, 20, 2048, 1, 0, 0, 0.2), (1300, 17, 32, 33, 8, 0, 0, 0.1), (40, 33, 16, 1111, 1, 0, 1, 0.3), (9, 100, 64, 264, 16, 8, 0, 0.5),
    (1500, 24, 48, 136, 1, 0, 0, 0.0), (3, 16, 16, 515, 1, 0, 0, 0.0)]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", MANY)
def test_many_choices(native, kind, shape):
    test_dispatch(native, kind, shape)
    test_combine(native, kind, shape)
    test_gradients(native, kind, shape)


def test_broadcast_inputs(native):
    """Inputs of row stride 0: an expanded gradient, one row for all."""
    import torch
    r = Run(native, routing(50, 3, 6, 1), 64, "bf16", 6, align=4)
    r.sort()
    one = torch.randn(64).bfloat16().cuda()
    y = torch.zeros(r.r, 64, dtype=torch.bfloat16, device="cuda")
    r.plan.combine_grad(one.data_ptr(), *r.maps(), y.data_ptr(), dout_stride=0)
    row, ok = r.live()
    assert torch.equal(y[row[ok].long().cuda()], one.expand(int(ok.sum()), 64))
    out = torch.zeros(50, 64, dtype=torch.bfloat16, device="cuda")
    r.plan.combine(one.data_ptr(), r.row_of.data_ptr(), out.data_ptr(), y_stride=0)
    close(out, 3 * one.double().cpu().expand(50, 64), 3 * one.double().cpu().abs().expand(50, 64), 3, "bf16")


@pytest.mark.parametrize("h", [33, 7, 2001])
def test_broadcast_inputs_at_any_address(native, h):
    """Row stride 0 and rows that start anywhere: nothing outside the one row is read (its neighbours are NaN
    and would show)."""
    import torch
    r = Run(native, routing(1300, 3, 6, 1), h, "bf16", 6, align=4)
    r.sort()
    buf = torch.full((h + 64,), float("nan"), dtype=torch.bfloat16, device="cuda")
    one = buf[5:5 + h]
    one.copy_(torch.randn(h))
    y = torch.zeros(r.r, h, dtype=torch.bfloat16, device="cuda")
    dw = torch.zeros(1300, 3, device="cuda")
    w = torch.ones(1300, 3, device="cuda")
    r.plan.combine_grad(one.data_ptr(), *r.maps(), y.data_ptr(), weight=w.data_ptr(), y=one.data_ptr(), dweight=dw.data_ptr(),
                        dout_stride=0, y_stride=0)
    row, ok = r.live()
    assert torch.equal(y[row[ok].long().cuda()], one.expand(int(ok.sum()), h))
    square = (one.double() ** 2).sum().cpu()
    close(dw, square.expand(1300, 3), square.expand(1300, 3), h, "f32")
    out = torch.zeros(1300, h, dtype=torch.bfloat16, device="cuda")
    r.plan.dispatch_grad(one.data_ptr(), r.row_of.data_ptr(), out.data_ptr(), x=one.data_ptr(), dweight=dw.data_ptr(), dy_stride=0,
                         x_stride=0)
    size = 3 * one.double().cpu().expand(1300, h)
    close(out, size, size.abs(), 3, "bf16")
    close(dw, square.expand(1300, 3), square.expand(1300, 3), h, "f32")


def test_long_map_captured_and_replayed(native):
    """The map in three kernels inside a CUDA graph, replayed with other routings; twice the same input gives
    the same map."""
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        r = Run(native, routing(70000, 2, 200, 1), 8, "bf16", 200, align=16)
        r.sort()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        r.sort()
    for seed in (2, 3, 3):
        ids = routing(70000, 2, 200, seed, 0.2)
        r.ids.copy_(ids)
        for t in (r.count, r.offset, r.row_of, r.slot_of):
            t.fill_(-9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        r.want = plain_map(ids.reshape(-1).tolist(), 0, 200, 16, r.r)
        r.check_map()


def test_not_a_number_stays_in_its_row(native):
    import torch
    r = Run(native, routing(40, 4, 8, 2), 256, "f32", 8)
    r.sort()
    y = torch.randn(r.r, 256, device="cuda")
    row, _ = r.live()
    y[row[7, 2]] = float("nan")
    y[row[9, 0], 3] = float("inf")
    out = torch.zeros(40, 256, device="cuda")
    r.plan.combine(y.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
    bad = ~torch.isfinite(out)
    assert bad[7].all() and bad[9, 3] and bad.sum().item() == 257


def test_maps_out_of_range_are_taken_as_dropped(native):
    """A damaged map: entries beyond the capacity move nothing."""
    import torch
    r = Run(native, routing(20, 2, 4, 4), 32, "f32", 4)
    r.sort()
    r.row_of.view(-1)[5] = r.r
    r.row_of.view(-1)[6] = 2**31 - 1
    r.row_of.view(-1)[7] = -2**31
    x = torch.randn(20, 32, device="cuda")
    y = torch.full((r.r, 32), 77.0, device="cuda")
    r.plan.dispatch(x.data_ptr(), *r.maps(), y.data_ptr())
    want = torch.full((r.r, 32), 77.0, device="cuda")
    for s, p in enumerate(r.row_of.view(-1).tolist()):
        if 0 <= p < r.r:
            want[p] = x[s // 2]
    assert torch.equal(y, want)
    out = torch.zeros(20, 32, device="cuda")
    r.plan.combine(y.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
    assert torch.equal(out[0], 2 * x[0]) and torch.equal(out[3], 0 * x[3])


def _layer(native, t, k, e, h, kind, align, stream=0):
    """A layer of experts as a user writes it: forward and backward through the row operators, the experts'
    products by segments of the sorted rows."""
    import torch

    class Layer:
        plan = native.RowPlan(t, k, e, h, _types(native)[kind][0], align=align, stream=stream)
        dtype = _types(native)[kind][1]

        def __init__(self):
            r, i32 = self.plan.capacity, dict(dtype=torch.int32, device="cuda")
            self.count, self.offset = torch.zeros(e, **i32), torch.zeros(e + 1, **i32)
            self.row_of, self.slot_of = torch.zeros(t, k, **i32), torch.zeros(r, **i32)
            new = lambda *s: torch.zeros(*s, dtype=self.dtype, device="cuda")
            self.rows, self.y, self.dy, self.drows = new(r, h), new(r, h), new(r, h), new(r, h)
            self.out, self.dx, self.dw = new(t, h), new(t, h), torch.zeros(t, k, device="cuda")

        def forward(self, x, ids, w, scale):
            p = self.plan
            p.sort(ids.data_ptr(), ids.element_size(), self.count.data_ptr(), self.offset.data_ptr(), self.row_of.data_ptr(),
                   self.slot_of.data_ptr())
            p.dispatch(x.data_ptr(), self.row_of.data_ptr(), self.count.data_ptr(), self.offset.data_ptr(), self.rows.data_ptr())
            self.expert = (torch.searchsorted(self.offset[1:].contiguous(), torch.arange(p.capacity, device="cuda", dtype=torch.int32),
                                              right=True)).clamp_max(e - 1)
            self.y.copy_(self.rows * scale[self.expert])
            p.combine(self.y.data_ptr(), self.row_of.data_ptr(), self.out.data_ptr(), weight=w.data_ptr())
            return self.out

        def backward(self, dout, w, scale):
            p = self.plan
            p.combine_grad(dout.data_ptr(), self.row_of.data_ptr(), self.count.data_ptr(), self.offset.data_ptr(), self.dy.data_ptr(),
                           weight=w.data_ptr(), y=self.y.data_ptr(), dweight=self.dw.data_ptr())
            self.drows.copy_(self.dy * scale[self.expert])
            self.dscale = torch.zeros_like(scale).index_add_(0, self.expert, self.dy * self.rows)
            p.dispatch_grad(self.drows.data_ptr(), self.row_of.data_ptr(), self.dx.data_ptr())
            return self.dx, self.dw, self.dscale
    return Layer()


def test_layer_forward_and_backward(native):
    """All operators together: outputs and gradients against autograd in 64 bits and against differences."""
    import torch
    t, k, e, h = 29, 3, 5, 48
    g = torch.Generator().manual_seed(8)
    ids = routing(t, k, e, 21, 0.1)
    x, w, scale = torch.randn(t, h, generator=g), torch.randn(t, k, generator=g), torch.randn(e, h, generator=g)
    dout = torch.randn(t, h, generator=g)
    layer = _layer(native, t, k, e, h, "f32", 8)
    ws, sc = w.cuda(), scale.cuda()
    out = layer.forward(x.cuda(), ids.int().cuda(), ws, sc).cpu()
    dx, dw, dscale = [v.cpu() for v in layer.backward(dout.cuda(), ws, sc)]

    def plain(x, w, scale):
        ok = (ids >= 0).double()[:, :, None]
        return (x[:, None, :] * scale[ids.clamp_min(0)] * w[:, :, None] * ok).sum(1)

    xd, wd, sd = [v.double().requires_grad_() for v in (x, w, scale)]
    want = plain(xd, wd, sd)
    want.backward(dout.double())
    # three products in a row and a sum of k (dx, out) or h (dw) or t * k (dscale) terms
    big = 16.0 * 16 * 16
    for got, ref, n in ((out, want.detach(), k), (dx, xd.grad, k), (dw, wd.grad, h), (dscale, sd.grad, t * k)):
        assert (got.double() - ref).abs().max().item() <= (n + 4) * n * 2.0 ** -24 * big
    # differences of the operators' own forward pass: d/dx in a direction; the layer is linear in x, so the
    # difference quotient is exact up to rounding (2^-24 of the outputs' size, over the step)
    step, direction = 2.0 ** -4, torch.randn(t, h, generator=g)
    loss = lambda xs: (layer.forward(xs.cuda(), ids.int().cuda(), ws, sc).cpu().double() * dout.double()).sum().item()
    slope = (loss(x + step * direction) - loss(x - step * direction)) / (2 * step)
    assert abs(slope - (dx.double() * direction.double()).sum().item()) <= t * h * (k + 4) * 2.0 ** -24 * big / step / 16
    loss_w = lambda ws_: (layer.forward(x.cuda(), ids.int().cuda(), ws_.cuda(), sc).cpu().double() * dout.double()).sum().item()
    direction = torch.randn(t, k, generator=g)
    slope = (loss_w(w + step * direction) - loss_w(w - step * direction)) / (2 * step)
    assert abs(slope - (dw.double() * direction.double()).sum().item()) <= t * h * (k + 4) * 2.0 ** -24 * big / step / 16


def test_layer_gradients_element_by_element(native):
    """Every output and gradient of a layer within the roundings of its own terms, against autograd in 64 bits and
    against differences.  A result of n terms, each made by at most three roundings of 2^-24, has at most n more in
    its sum: (n + 4) * 2^-24 times the sum of its terms' magnitudes."""
    import torch
    t, k, e, h = 29, 3, 5, 48
    g = torch.Generator().manual_seed(8)
    ids = routing(t, k, e, 21, 0.1)
    x, w, scale = torch.randn(t, h, generator=g), torch.randn(t, k, generator=g), torch.randn(e, h, generator=g)
    dout = torch.randn(t, h, generator=g)
    layer = _layer(native, t, k, e, h, "f32", 8)
    on = ids.int().cuda()

    def run(x, w):
        return layer.forward(x.cuda(), on, w.cuda(), scale.cuda()).double().cpu()

    out = run(x, w)
    dx, dw, dscale = [v.double().cpu() for v in layer.backward(dout.cuda(), w.cuda(), scale.cuda())]
    ok = (ids >= 0).double()

    def plain(x, w, scale):
        return (x[:, None, :] * scale[ids.clamp_min(0)] * (w * ok)[:, :, None]).sum(1)

    def gradients(x, w, scale, dout):
        v = [a.double().clone().requires_grad_() for a in (x, w, scale)]
        y = plain(*v)
        y.backward(dout.double())
        return [y.detach()] + [a.grad for a in v]

    u = 2.0 ** -24 * 1.001
    got, want = (out, dx, dw, dscale), gradients(x, w, scale, dout)
    # of magnitudes alone, the formulas give the sums of the terms' magnitudes
    size = gradients(x.abs(), w.abs(), scale.abs(), dout.abs())
    terms = (k, k, h, t * k)
    limits = [(n + 4) * u * s for n, s in zip(terms, size)]
    for a, b, limit in zip(got, want, limits):
        assert ((a - b).abs() <= limit).all()
    # the limits would show a term that is left out: the last column of dw, the last choice of out and dx
    column = dout[:, None, -1] * x[:, None, -1] * scale[ids.clamp_min(0), -1] * ok
    assert (column.abs() > limits[2])[ok > 0].double().mean() > 0.95
    short = w.clone()
    short[:, -1] = 0
    for a, b, limit in zip(gradients(x, short, scale, dout)[:2], want, limits):
        assert ((a - b).abs() > limit)[ok[:, -1] > 0].double().mean() > 0.95
    # differences of the operators' own forward pass, which is linear in x and in w
    step = 2.0 ** -4

    def magnitude(x, w):
        return ((k + 4) * u * plain(x.abs().double(), w.abs().double(), scale.abs().double()) * dout.abs().double()).sum().item()

    for which, grad, limit in ((0, dx, limits[1]), (1, dw, limits[2])):
        base = (x, w)[which]
        direction = torch.randn(base.shape, generator=g)
        ends = [[x, w], [x, w]]
        for i, sign in enumerate((1, -1)):
            ends[i][which] = base + sign * step * direction
        moved = ends[0][which].double() - ends[1][which].double()
        difference = ((run(*ends[0]) - run(*ends[1])) * dout.double()).sum().item()
        assert abs(difference - (grad * moved).sum().item()) <= magnitude(*ends[0]) + magnitude(*ends[1]) + (limit * moved.abs()).sum().item()


def test_layer_captured_and_replayed_with_new_routing(native):
    """A whole step in a CUDA graph on the plan's stream; replays read the routing that is in the buffers then,
    while an eager layer of the same inputs lives.  Results equal the eager ones bit for bit."""
    import torch
    t, k, e, h = 600, 4, 32, 256
    side = torch.cuda.Stream()
    captured, eager = _layer(native, t, k, e, h, "bf16", 16, side.cuda_stream), _layer(native, t, k, e, h, "bf16", 16)
    g = torch.Generator().manual_seed(4)
    ids = routing(t, k, e, 1).int().cuda()
    x, dout = torch.randn(t, h, generator=g).bfloat16().cuda(), torch.randn(t, h, generator=g).bfloat16().cuda()
    w, scale = torch.rand(t, k, generator=g).cuda(), torch.randn(e, h, generator=g).bfloat16().cuda()
    eager.forward(x, ids, w, scale)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        captured.forward(x, ids, w, scale)
        captured.backward(dout, w, scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured.forward(x, ids, w, scale)
        captured.backward(dout, w, scale)
    for seed in (2, 3):
        ids.copy_(routing(t, k, e, seed, 0.2 * (seed - 2)).int().cuda())
        x.copy_(torch.randn(t, h, generator=g).bfloat16().cuda())
        for layer in (captured, eager):
            layer.rows.zero_()
            layer.dy.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.forward(x, ids, w, scale)
        eager.backward(dout, w, scale)
        torch.cuda.synchronize()
        for name in ("row_of", "slot_of", "rows", "out", "dy", "dx", "dw"):
            assert torch.equal(getattr(captured, name), getattr(eager, name)), name


@pytest.mark.parametrize("t,e,steps", [(40, 16, 400), (3000, 64, 200), (20000, 48, 60)])
def test_steps_without_a_pause(native, t, e, steps):
    """Kernels that start while the one before still runs: buffers that change from step to step, nothing
    between the calls, errors counted on the device."""
    import torch
    k, h = 4, 128
    r = Run(native, routing(t, k, e, 1), h, "f32", e, align=4)
    g = torch.Generator().manual_seed(3)
    base, x = r.ids.clone(), torch.randn(t, h, generator=g).cuda()
    rows, out = torch.zeros(r.r, h, device="cuda"), torch.zeros(t, h, device="cuda")
    dx, dy = torch.zeros(t, h, device="cuda"), torch.zeros(r.r, h, device="cuda")
    wrong = torch.zeros(1, dtype=torch.int64, device="cuda")
    slots = torch.arange(t * k, device="cuda").view(t, k)
    for i in range(steps):
        r.ids.copy_((base + i) % e)
        x.add_(1.0)
        r.sort()
        r.plan.dispatch(x.data_ptr(), *r.maps(), rows.data_ptr())
        r.plan.combine(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
        r.plan.combine_grad(out.data_ptr(), *r.maps(), dy.data_ptr())
        r.plan.dispatch_grad(dy.data_ptr(), r.row_of.data_ptr(), dx.data_ptr())
        wrong += (out != 4 * x).any() + (dx != 16 * x).any() + (r.slot_of[r.row_of.long()] != slots).any()
        wrong += (r.count != torch.bincount(r.ids.view(-1).long(), minlength=e)).any()
    assert wrong.item() == 0          # sums of 4 and 16 equal numbers are exact


@pytest.mark.parametrize("wide", [False, True])
def test_long_map_of_indices_written_just_before(native, wide):
    """The map in three kernels: its last one reads the indices before it waits for the others.  Every step
    writes other indices with a kernel right before the map, where the step before left its own in the caches."""
    import torch
    n, e = 300000, 256
    r = Run(native, torch.zeros(n, 1, dtype=torch.int64), 8, "bf16", e, align=16, index=torch.int64 if wide else torch.int32)
    base = torch.randint(0, e, (n, 1), device="cuda").to(r.ids.dtype)
    wrong = torch.zeros(1, dtype=torch.int64, device="cuda")
    slots = torch.arange(n, device="cuda").view(n, 1)
    for i in range(150):
        torch.remainder(base + i * 37, e, out=r.ids)
        r.sort()
        row = r.row_of.view(-1).long()
        expert = torch.searchsorted(r.offset[1:].contiguous(), r.row_of.view(-1), right=True)      # of the segment of each slot's row
        wrong += (expert != r.ids.view(-1)).any() + (r.slot_of[row].view(n, 1) != slots).any()
        wrong += (r.count != torch.bincount(r.ids.view(-1).long(), minlength=e)).any()
    assert wrong.item() == 0


def test_capture_behind_copies_and_other_streams(native):
    """Graph nodes before the operators that are not kernels (copies, a fill), and a join with another stream."""
    import torch
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        r = Run(native, routing(500, 4, 30, 1), 256, "bf16", 30, align=8)
        r.sort()
    new_ids, new_x = r.ids.clone(), torch.zeros(500, 256, dtype=torch.bfloat16, device="cuda")
    x, rows = torch.zeros_like(new_x), torch.zeros(r.r, 256, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros_like(x)
    host = torch.zeros(500, 256, dtype=torch.bfloat16).pin_memory()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.wait_stream(side)
        with torch.cuda.stream(other):
            x.copy_(new_x)
        r.ids.copy_(new_ids)                      # a copy node
        r.sort()
        rows.zero_()                              # a fill node
        side.wait_stream(other)                   # two dependencies
        r.plan.dispatch(x.data_ptr(), *r.maps(), rows.data_ptr())
        r.plan.combine(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
        host.copy_(out, non_blocking=True)
    g = torch.Generator().manual_seed(2)
    for seed in (4, 5, 6):
        ids = routing(500, 4, 30, seed)
        new_ids.copy_(ids)
        new_x.copy_(torch.randn(500, 256, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        r.want = plain_map(ids.reshape(-1).tolist(), 0, 30, 8, r.r)
        r.check_map()
        assert torch.equal(host, (4 * new_x.float()).bfloat16().cpu())
        assert (rows[r.want[1][-1]:] == 0).all()


def test_waits_for_events_of_other_streams(native):
    """A call behind an event of another stream, with this stream's own kernels just before it."""
    import torch
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        r = Run(native, routing(3000, 4, 30, 1), 64, "f32", 30, align=4)
    x, rows, out = torch.zeros(3000, 64, device="cuda"), torch.zeros(r.r, 64, device="cuda"), torch.zeros(3000, 64, device="cuda")
    ids = [routing(3000, 4, 30, k).int().cuda() for k in range(2, 6)]
    wrong = torch.zeros(1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for i, new in enumerate(ids * 3):
        with torch.cuda.stream(side):
            r.sort()
        other.wait_stream(side)
        with torch.cuda.stream(other):
            torch.cuda._sleep(1000000)
            r.ids.copy_(new)
            x.fill_(float(i))
        with torch.cuda.stream(side):
            r.plan.combine(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr())      # overlaps the other stream
            side.wait_stream(other)
            r.sort()
            r.plan.dispatch(x.data_ptr(), *r.maps(), rows.data_ptr())
            r.plan.combine(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
            wrong += (out != 4.0 * i).any() + (r.count != torch.bincount(new.view(-1).long(), minlength=30)).any()
    torch.cuda.synchronize()
    assert wrong.item() == 0


def test_one_plan_from_several_threads(native):
    import threading
    import torch
    r = Run(native, routing(200, 4, 12, 1), 512, "f32", 12)
    r.sort()
    x, rows = torch.randn(200, 512, device="cuda"), torch.zeros(r.r, 512, device="cuda")
    r.plan.dispatch(x.data_ptr(), *r.maps(), rows.data_ptr())
    outs = [torch.zeros(200, 512, device="cuda") for _ in range(4)]
    failed = []

    def work(out):
        try:
            torch.cuda.set_device(0)
            for _ in range(200):
                r.plan.combine(rows.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
                p = native.RowPlan(3, 1, 2, 8, native.CUTT_ROWS_F32)
                p.destroy()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for out in outs:
        assert torch.equal(out, 4 * x)


@pytest.mark.parametrize("tokens", [(1024, 8192), (20000, 60000)])
def test_sorts_of_several_sizes_from_several_threads(native, tokens):
    """Two threads whose maps need different amounts of one kernel's shared memory."""
    import threading
    import torch
    runs, failed = [], []
    for t in tokens:
        with torch.cuda.stream(torch.cuda.Stream()):
            runs.append(Run(native, routing(t, 8, 256, t), 8, "bf16", 256, align=8))
    torch.cuda.synchronize()

    def work(r):
        torch.cuda.set_device(0)
        for _ in range(3000):
            try:
                r.sort()
            except native.CuttError as e:
                failed.append(e)

    threads = [threading.Thread(target=work, args=(r,)) for r in runs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for r in runs:
        r.check_map()


@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
def test_sorts_of_several_sizes_in_one_graph(native, order):
    """A graph is instantiated after all its calls were captured, the smaller maps among them."""
    import torch
    side, runs = torch.cuda.Stream(), []
    with torch.cuda.stream(side):
        for t in (1024, 8192):
            runs.append(Run(native, routing(t, 8, 256, t), 8, "bf16", 256, align=8))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for i in order:
            runs[i].sort()
    graph.replay()
    torch.cuda.synchronize()
    for r in runs:
        r.check_map()


@pytest.fixture
def few_sms():
    """A stream whose context has 16 SMs, which cannot hold a cluster of 16 blocks."""
    import torch
    d = pytest.importorskip("cuda.bindings.driver")
    torch.zeros(1, device="cuda")

    def ok(r):
        assert int(r[0]) == 0, r
        return r[1] if len(r) == 2 else r[1:]

    dev = ok(d.cuDeviceGet(torch.cuda.current_device()))
    sms = ok(d.cuDeviceGetDevResource(dev, d.CUdevResourceType.CU_DEV_RESOURCE_TYPE_SM))
    parts = ok(d.cuDevSmResourceSplitByCount(1, sms, 0, 16))[0]
    context = ok(d.cuGreenCtxCreate(ok(d.cuDevResourceGenerateDesc(parts[:1], 1)), dev, d.CUgreenCtxCreate_flags.CU_GREEN_CTX_DEFAULT_STREAM))
    stream = ok(d.cuGreenCtxStreamCreate(context, d.CUstream_flags.CU_STREAM_NON_BLOCKING, 0))
    yield int(stream)
    torch.cuda.synchronize()
    d.cuStreamDestroy(stream)
    d.cuGreenCtxDestroy(context)


def test_plans_made_while_their_stream_is_captured(native):
    """A plan may be made inside a capture: it asks what its stream's context can hold, and launches nothing."""
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        r = Run(native, routing(1024, 8, 64, 1), 8, "bf16", 64, align=8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        r.plan = native.RowPlan(1024, 8, 64, 8, r.code, align=8, stream=side.cuda_stream)
        pages = native.PagePlan(4, 16, 1100, 16384, stream=side.cuda_stream)
        r.sort()
    assert '"cluster": 16' in r.plan.describe() and '"cluster": 16' in pages.describe()
    graph.replay()
    torch.cuda.synchronize()
    r.check_map()


@pytest.mark.parametrize("t,k,e", [(1024, 8, 64), (8192, 8, 256), (257, 10, 4096), (70001, 3, 129)])
def test_map_in_a_context_of_few_sms(native, few_sms, t, k, e):
    import torch
    r = Run(native, routing(t, k, e, 6, 0.1), 8, "bf16", e, align=8)
    r.plan = native.RowPlan(t, k, e, 8, r.code, align=8, stream=few_sms)
    if 2048 < t * k <= 65536:
        assert '"cluster": 8' in r.plan.describe()
    torch.cuda.synchronize()
    r.sort()
    torch.cuda.synchronize()
    r.check_map()


def test_calls_on_another_device_are_refused(native):
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    r = Run(native, routing(20, 2, 4, 1), 32, "f32", 4)
    with torch.cuda.device(1):
        with pytest.raises(native.CuttError) as e:
            r.sort()
    assert e.value.code == native.CUTT_INVALID_DEVICE
    r.sort()
    r.check_map()


def test_two_plans_on_two_streams_at_once(native):
    import torch
    sets = []
    for i in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            sets.append((s, Run(native, routing(3000, 4, 40, 30 + i), 512, "bf16", 40, align=8)))
    torch.cuda.synchronize()
    xs = [torch.randn(3000, 512, device="cuda").bfloat16() for _ in sets]
    ys = [torch.zeros(r.r, 512, dtype=torch.bfloat16, device="cuda") for _, r in sets]
    outs = [torch.zeros(3000, 512, dtype=torch.bfloat16, device="cuda") for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for (_, r), x, y, out in zip(sets, xs, ys, outs):
            r.sort()
            r.plan.dispatch(x.data_ptr(), *r.maps(), y.data_ptr())
            r.plan.combine(y.data_ptr(), r.row_of.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    for (_, r), x, out in zip(sets, xs, outs):
        r.check_map()
        assert torch.equal(out, (4 * x.float()).bfloat16())     # four copies of a row: exact


def test_handles_and_devices(native):
    import torch
    n0 = native.launch_count()
    r = Run(native, routing(4, 2, 4, 0), 16, "bf16", 4)
    h = r.plan.handle
    assert '"rows"' in r.plan.describe()
    assert native.cuttExecute(h, 16, 32) == native.CUTT_INVALID_PLAN
    L = native.lib()
    assert L.cutt_pages_store(h, 16, 0, 8, 8, 32, 48, 0) == native.CUTT_INVALID_PLAN       # a handle of another kind
    x = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(native.CuttError) as bad:
        r.plan.dispatch(x.data_ptr(), *r.maps(), x.data_ptr())
    assert bad.value.code == native.CUTT_INVALID_PARAMETER
    assert native.launch_count() == n0
    r.sort()
    assert native.launch_count() > n0
    r.plan.destroy()
    assert native.cuttDestroy(h) == native.CUTT_INVALID_PLAN
    with pytest.raises(native.CuttError):
        r.plan.describe()
    with pytest.raises(native.CuttError):
        r.sort()


def test_row_offsets_beyond_32_bits(native):
    """Rows whose byte offsets pass 2^32 (and whose element offsets pass 2^31)."""
    import torch
    t, k, e, h = 40, 2, 3, 1 << 20
    stride = (1 << 26) + 8
    r = Run(native, routing(t, k, e, 5), 512, "bf16", e)
    r.sort()
    x = torch.randn(t, 512, device="cuda").bfloat16()
    y = torch.zeros(stride * (r.r - 1) + 512, dtype=torch.bfloat16, device="cuda")
    assert y.numel() > 2**32
    r.plan.dispatch(x.data_ptr(), *r.maps(), y.data_ptr(), y_stride=stride)
    rows = torch.as_strided(y, (r.r, 512), (stride, 1))
    row, ok = r.live()
    assert torch.equal(rows[row.view(-1).long().cuda()], x[:, None].expand(t, k, 512).reshape(-1, 512))
    out = torch.zeros_like(x)
    r.plan.combine(y.data_ptr(), r.row_of.data_ptr(), out.data_ptr(), y_stride=stride)
    assert torch.equal(out, (2 * x.float()).bfloat16())
