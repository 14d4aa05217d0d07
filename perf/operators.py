"""Measured cases of the operators that move rows by an index map built on the GPU.

Six operators: rows sorted by expert (`sort`), moved into that order (`dispatch`) and back with weights
(`combine`), the backward pass of both moves (`backward`), block tables and slot maps of a paged cache
(`tables`), and rows stored into and loaded from its pages (`paged`).

`own` false: elementary torch operations; `own` true: the calls a user makes of cutt_b200.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}


def _rows(name, op, **kw):
    """A case of sort, dispatch, combine or backward.  tokens x choices slots, `drop` of them without an
    expert of this process; segments start at multiples of `align`; `pad`: elements between token rows;
    `weights`: "" or the move that applies them ("dispatch", "combine"); `skew`: how uneven experts are."""
    c = dict(op=op, tokens=64, choices=8, experts=64, first=0, align=1, width=2048, type="bf16",
             weights="", drop=0.0, skew=1.0, pad=0, index=4)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the map of one decoding step of a small batch
        _rows("sort_decode", "sort", tokens=48, choices=6, experts=64),
        # the map of a long prefill: segments padded to whole tiles of 128 rows, 64-bit indices as topk gives them
        _rows("sort_prefill", "sort", tokens=65536, choices=8, experts=256, align=128, index=8, skew=2.0),
        # rows of a decoding step
        _rows("dispatch_decode", "dispatch", tokens=48, choices=6, experts=64, width=2048),
        # rows of a prefill, padded segments
        _rows("dispatch_prefill", "dispatch", tokens=16384, choices=8, experts=128, align=128, width=4096),
        # a single token on its way back: latency only
        _rows("combine_single", "combine", tokens=1, choices=8, experts=128, width=5120, type="fp16", weights="combine"),
        # a prefill on its way back
        _rows("combine_prefill", "combine", tokens=8192, choices=4, experts=32, align=16, width=2560, weights="combine"),
        # an odd fp32 width, weights applied on the way in, some slots dropped
        _rows("backward_odd", "backward", tokens=1023, choices=3, experts=17, width=1111, type="fp32",
              weights="dispatch", drop=0.1),
        # the backward pass of a training step of one process among several: half of the slots are elsewhere
        _rows("backward_train", "backward", tokens=16384, choices=8, experts=32, first=32, align=128, width=2048,
              weights="combine", drop=0.5),
        # one decoding step of 256 requests: one token each
        dict(name="tables_decode", op="tables", requests=256, page=16, width=2048, tokens=256, spare=0, most=32768),
        # a prefill step: chunks of many lengths, some requests with nothing to add
        dict(name="tables_prefill", op="tables", requests=61, page=64, width=2048, tokens=131072, spare=1000, most=65536),
        # K and V of one decoding step, head-major pages
        dict(name="paged_decode", op="paged", store=256, load=0, heads=8, size=128, page=16, pages=2048, type="bf16",
             headmajor=True, skip=0.0),
        # a chunk of a prefill: its K and V stored, the context loaded in token order
        dict(name="paged_chunk", op="paged", store=8192, load=131072, heads=8, size=128, page=64, pages=2304,
             type="bf16", headmajor=True, skip=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "dispatch", "combine", "backward", "tables", "paged"])
    if op == "tables":
        requests = _log(rng, 1, 2048)
        page = rng.choice([1, 8, 16, 24, 32, 64, 128])
        decode = rng.random() < 0.5
        most = _log(rng, 64, 65536)
        tokens = requests if decode else max(requests, _log(rng, 64, 131072))
        width = max(4, 2 * -(-(most + tokens) // page) if page > 1 else most + tokens)
        while requests * width > 4_000_000:
            width = -(-width // 2)
        return dict(op=op, requests=requests, page=page, width=width, tokens=tokens, spare=rng.choice([0, 1, 77]),
                    most=min(most, width * page))
    if op == "paged":
        heads = rng.choice([1, 2, 3, 4, 8, 16])
        size = rng.choice([64, 72, 80, 96, 128, 192, 256, 33])
        page = rng.choice([1, 8, 16, 24, 32, 64, 128])
        kind = rng.choice(["bf16", "bf16", "fp32", "int8"])
        most = 131072 * 8 * 128 * 2 // (heads * size * _BYTES[kind])
        load = 0 if rng.random() < 0.4 else _log(rng, 16, max(17, min(most, 131072)))
        store = _log(rng, 1, 8192)
        pages = -(-(store + load) // page) + rng.choice([1, 7, 64])
        return dict(op=op, store=store, load=load, heads=heads, size=size, page=page, pages=pages, type=kind,
                    headmajor=rng.random() < 0.5, skip=rng.choice([0.0, 0.0, 0.1]))
    choices = rng.choice([1, 2, 3, 4, 6, 8, 8, 10])
    experts = rng.choice([8, 16, 17, 32, 60, 64, 96, 128, 256, 384])
    experts = max(experts, choices)
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    width = 8 * _log(rng, 32, 1024) if rng.random() < 0.8 else _log(rng, 200, 5000)
    top = 16384 * 8 * 4096 * 2 if op != "backward" else 16384 * 8 * 2048 * 2
    tokens = min(_log(rng, 1, 65536 if op == "sort" else 32768), max(1, top // (choices * width * _BYTES[kind])))
    weights = ""
    if op == "dispatch":
        weights = rng.choice(["", "", "dispatch"])
        if not weights and rng.random() < 0.2:
            kind = "int8"
    elif op == "combine":
        weights = rng.choice(["", "combine", "combine"])
    elif op == "backward":
        weights = rng.choice(["combine", "combine", "dispatch"])
    align = rng.choice([1, 1, 8, 16, 64, 128])
    if tokens * choices < 8 * experts:  # few rows: whole tiles of padding are not what such a step uses
        align = min(align, 8)
    return _rows("", op, tokens=tokens, choices=choices, experts=experts, first=rng.choice([0, 0, experts]),
                 align=align, width=width, type=kind, weights=weights, drop=rng.choice([0.0, 0.0, 0.1, 0.5]),
                 skew=rng.choice([0.0, 1.0, 2.0]), pad=rng.choice([0, 0, 8, 64]) if kind != "int8" else 0,
                 index=rng.choice([4, 8]))


# ---------------------------------------------------------------------------------------------- inputs

def _capacity(case):
    n = case["tokens"] * case["choices"]
    return n + min(case["experts"], n) * (case["align"] - 1)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _routing(case, seed):
    """Expert of each slot: the top choices of uneven scores, no expert twice in a token; dropped slots hold
    an expert of another process (or -1 where there is none)."""
    g = _generator(seed)
    t, k, e = case["tokens"], case["choices"], case["experts"]
    bias = case["skew"] * torch.randn(e, device="cuda", generator=g)
    out = torch.empty(t, k, dtype=torch.int64, device="cuda")
    for at in range(0, t, 16384):
        n = min(16384, t - at)
        gumbel = -torch.log(-torch.log(torch.rand(n, e, device="cuda", generator=g).clamp_(1e-7, 1 - 1e-6)))
        out[at:at + n] = torch.topk(bias + gumbel, k, dim=1).indices
    out += case["first"]
    if case["drop"]:
        away = torch.rand(t, k, device="cuda", generator=g) < case["drop"]
        out[away] = case["first"] - 1
    return out.to(torch.int32 if case["index"] == 4 else torch.int64)


def _map(case, expert_of):
    """The map in elementary operations (int64 inside): count, offset, row of each slot, slot of each row."""
    n, e, a, r = expert_of.numel(), case["experts"], case["align"], _capacity(case)
    local = expert_of.reshape(-1).long() - case["first"]
    valid = (local >= 0) & (local < e)
    key = torch.where(valid, local, e)
    count = torch.zeros(e + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))[:e]
    size = (count + a - 1) // a * a
    offset = torch.cat([size.new_zeros(1), size.cumsum(0)])
    order = torch.sort(key, stable=True).indices
    start = torch.cat([count.new_zeros(1), count.cumsum(0)])
    sorted_key = key[order]
    rank = torch.arange(n, device="cuda") - start[sorted_key]
    row_sorted = torch.where(sorted_key < e, offset[sorted_key] + rank, -1)
    row_of = torch.empty_like(key)
    row_of[order] = row_sorted
    slot_of = torch.full((r + 1,), -1, dtype=torch.int64, device="cuda")
    slot_of[torch.where(row_of >= 0, row_of, r)] = torch.arange(n, device="cuda")
    return count.int(), offset.int(), row_of.int(), slot_of[:r].int()


def _token_rows(case, g, kind, pad=True):
    t, h = case["tokens"], case["width"]
    wide = h + (case["pad"] if pad else 0)
    if kind == torch.int8:
        full = torch.randint(-127, 128, (t, wide), device="cuda", generator=g, dtype=torch.int8)
    else:
        full = torch.randn(t, wide, device="cuda", generator=g).to(kind)
    return full[:, :h]


def prepare(case, seed):
    return {"tables": _prepare_tables, "paged": _prepare_paged}.get(case["op"], _prepare_rows)(case, seed)


def _prepare_rows(case, seed):
    t, k, h, r = case["tokens"], case["choices"], case["width"], _capacity(case)
    kind = _TYPES[case["type"]]
    s = {"case": case, "experts": _routing(case, seed)}
    g = _generator(seed + 1)
    if own:
        import cutt_b200 as C
        s["plan"] = C.RowPlan(t, k, case["experts"], h, {"int8": C.CUTT_ROWS_BYTES, "fp16": C.CUTT_ROWS_F16, "bf16": C.CUTT_ROWS_BF16,
                                                         "fp32": C.CUTT_ROWS_F32}[case["type"]],
                              first=case["first"], align=case["align"], capacity=r,
                              stream=torch.cuda.current_stream().cuda_stream)
    if case["op"] == "sort":
        s["count"] = torch.zeros(case["experts"], dtype=torch.int32, device="cuda")
        s["offset"] = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
        s["row_of"] = torch.zeros(t, k, dtype=torch.int32, device="cuda")
        s["slot_of"] = torch.zeros(r, dtype=torch.int32, device="cuda")
        return s
    s["count"], s["offset"], row_of, s["slot_of"] = _map(case, s["experts"])
    s["row_of"] = row_of.view(t, k)
    s["weight"] = torch.softmax(torch.randn(t, k, device="cuda", generator=g), 1) if case["weights"] else None
    if case["op"] == "dispatch":
        s["x"] = _token_rows(case, g, kind)
        s["y"] = torch.zeros(r, h, dtype=kind, device="cuda")
    elif case["op"] == "combine":
        s["y"] = torch.randn(r, h, device="cuda", generator=g).to(kind)
        s["out"] = torch.zeros(t, h + case["pad"], dtype=kind, device="cuda")[:, :h]
    else:
        # x -> dispatch -> rows -> (the experts' products) -> y -> combine -> out, and the gradients back
        s["dout"] = _token_rows(case, g, kind)
        s["y"] = torch.randn(r, h, device="cuda", generator=g).to(kind)
        s["x"] = _token_rows(case, g, kind)
        s["drows"] = torch.randn(r, h, device="cuda", generator=g).to(kind)
        s["dy"] = torch.zeros(r, h, dtype=kind, device="cuda")
        s["dx"] = torch.zeros(t, h, dtype=kind, device="cuda")
        s["dweight"] = torch.zeros(t, k, device="cuda")
    return s


def _lengths(case, seed):
    """Tokens held and added by each request.  A decoding step adds one to each; a prefill step splits its
    tokens unevenly, and some requests add nothing."""
    g = torch.Generator().manual_seed(seed)
    b, n, top = case["requests"], case["tokens"], case["width"] * case["page"]
    if n == b:
        added = torch.ones(b, dtype=torch.int64)
    else:
        share = torch.rand(b, generator=g) ** 3 * (torch.rand(b, generator=g) < 0.9)
        added = (share / share.sum().clamp_min(1e-9) * n).floor().long()
    added = added.clamp_max(top)
    held = (torch.rand(b, generator=g) ** 2 * min(case["most"], top)).long()
    return torch.minimum(held, top - added), added


def _prepare_tables(case, seed):
    b, p, w = case["requests"], case["page"], case["width"]
    held, added = _lengths(case, seed)
    have = (held + p - 1) // p
    g = _generator(seed)
    total = int(((held + added + p - 1) // p).sum()) + 8
    ids = torch.randperm(total, device="cuda", generator=g).int()
    table = torch.full((b, w), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(w, device="cuda")[None, :]
    before = (have.cumsum(0) - have).cuda()
    taken = column < have.cuda()[:, None]
    table[taken] = ids[(before[:, None] + column)[taken]]
    used = int(have.sum())
    s = {"case": case, "held": held.int().cuda(), "added": added.int().cuda(), "free": ids,
         "pool": torch.tensor([used, total], dtype=torch.int32, device="cuda"), "table": table}
    s["slots"] = torch.zeros(case["tokens"] + case["spare"], dtype=torch.int64, device="cuda")
    s["pool_out"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    s["token_offset"] = torch.zeros(b + 1, dtype=torch.int32, device="cuda")
    s["page_offset"] = torch.zeros(b + 1, dtype=torch.int32, device="cuda")
    if own:
        import cutt_b200 as C
        s["plan"] = C.PagePlan(b, p, w, s["slots"].numel(), stream=torch.cuda.current_stream().cuda_stream)
    return s


def _cache_shape(case):
    """Shape of a cache and its element strides by page, slot and head.  The last page takes what the plain
    form writes for skipped rows; no slot reaches it."""
    p, h, d = case["page"], case["heads"], case["size"]
    if case["headmajor"]:
        return (case["pages"] + 1, h, p, d), (h * p * d, d, p * d)
    return (case["pages"] + 1, p, h, d), (p * h * d, h * d, d)


def _values(shape, kind, g):
    if kind == torch.int8:
        return torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8)
    return torch.randn(shape, device="cuda", generator=g).to(kind)


def _prepare_paged(case, seed):
    g = _generator(seed)
    kind, p = _TYPES[case["type"]], case["page"]
    shape, strides = _cache_shape(case)
    n, m, h, d = case["store"], case["load"], case["heads"], case["size"]
    s = {"case": case, "k_cache": _values(shape, kind, g), "v_cache": _values(shape, kind, g)}
    # sequences occupy whole pages in an arbitrary order; the new rows follow the loaded context
    pages = torch.randperm(case["pages"], device="cuda", generator=g)
    at = torch.arange(n + m, device="cuda")
    slots = pages[at // p] * p + at % p
    if n and m == 0:  # a decoding step: rows of unrelated requests
        slots = torch.randperm(case["pages"] * p, device="cuda", generator=g)[:n]
    s["load_slots"], s["store_slots"] = slots[:m].clone(), slots[slots.numel() - n:].clone()
    if case["skip"]:
        for name in ("load_slots", "store_slots"):
            s[name][torch.rand(s[name].numel(), device="cuda", generator=g) < case["skip"]] = -1
    # new rows are slices of one projection: q, k and v side by side
    s["qkv"] = _values((n, 3 * h, d), kind, g)
    s["k"], s["v"] = s["qkv"][:, h:2 * h], s["qkv"][:, 2 * h:]
    s["k_rows"] = torch.zeros(m, h, d, dtype=kind, device="cuda")
    s["v_rows"] = torch.zeros(m, h, d, dtype=kind, device="cuda")
    if own:
        import cutt_b200 as C
        stream = torch.cuda.current_stream().cuda_stream
        s["store"] = C.PagedRows(n, h, d, _BYTES[case["type"]], case["pages"], p, strides[0], strides[1], strides[2], stream=stream)
        s["load"] = C.PagedRows(max(1, m), h, d, _BYTES[case["type"]], case["pages"], p, strides[0], strides[1], strides[2], stream=stream)
    return s


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return _RUN[state["case"]["op"]](state)


def _sort(s):
    if own:
        e = s["experts"]
        s["plan"].sort(e.data_ptr(), e.element_size(), s["count"].data_ptr(), s["offset"].data_ptr(),
                       s["row_of"].data_ptr(), s["slot_of"].data_ptr())
        return s["count"], s["offset"], s["row_of"], s["slot_of"]
    count, offset, row_of, slot_of = _map(s["case"], s["experts"])
    return count, offset, row_of.view(s["row_of"].shape), slot_of


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _scatter(case, rows, row_of, weight, r):
    """rows (T, H) -> (r, H): each slot's row, times its weight; rows that no slot owns are zero."""
    at = torch.where(row_of >= 0, row_of, r).reshape(-1).long()
    values = rows.float()[:, None, :].expand(-1, case["choices"], -1)
    if weight is not None:
        values = values * weight[:, :, None]
    out = torch.zeros(r + 1, rows.shape[1], dtype=rows.dtype, device="cuda")
    out[at] = values.to(rows.dtype).reshape(-1, rows.shape[1])
    return out[:r]


def _gather(rows, row_of):
    """(T, k, H) in 32 bits, zero where a slot was dropped."""
    return torch.where((row_of >= 0)[:, :, None], rows[row_of.clamp_min(0).long()].float(), 0.0)


def _dispatch(s):
    case, x, y = s["case"], s["x"], s["y"]
    if own:
        s["plan"].dispatch(x.data_ptr(), s["row_of"].data_ptr(), s["count"].data_ptr(), s["offset"].data_ptr(),
                           y.data_ptr(), weight=_ptr(s["weight"]), x_stride=x.stride(0))
        return y
    return _scatter(case, x, s["row_of"], s["weight"], y.shape[0])


def _combine(s):
    y, out = s["y"], s["out"]
    if own:
        s["plan"].combine(y.data_ptr(), s["row_of"].data_ptr(), out.data_ptr(), weight=_ptr(s["weight"]),
                          out_stride=out.stride(0))
        return out
    values = _gather(y, s["row_of"])
    if s["weight"] is not None:
        values = values * s["weight"][:, :, None]
    return values.sum(1).to(y.dtype)


def _backward(s):
    case, plan = s["case"], s.get("plan")
    w_in = s["weight"] if case["weights"] == "dispatch" else None
    w_out = s["weight"] if case["weights"] == "combine" else None
    dout, y, x, drows = s["dout"], s["y"], s["x"], s["drows"]
    if own:
        dw = s["dweight"].data_ptr()
        plan.combine_grad(dout.data_ptr(), s["row_of"].data_ptr(), s["count"].data_ptr(), s["offset"].data_ptr(),
                          s["dy"].data_ptr(), weight=_ptr(w_out), y=y.data_ptr() if w_out is not None else 0,
                          dweight=dw if w_out is not None else 0, dout_stride=dout.stride(0))
        plan.dispatch_grad(drows.data_ptr(), s["row_of"].data_ptr(), s["dx"].data_ptr(), weight=_ptr(w_in),
                           x=x.data_ptr() if w_in is not None else 0, dweight=dw if w_in is not None else 0,
                           x_stride=x.stride(0))
        return s["dy"], s["dx"], s["dweight"]
    dy = _scatter(case, dout, s["row_of"], w_out, y.shape[0])
    back = _gather(drows, s["row_of"])
    if w_out is not None:
        dweight = (_gather(y, s["row_of"]) * dout.float()[:, None, :]).sum(-1)
    else:
        dweight = (back * x.float()[:, None, :]).sum(-1)
        back = back * w_in[:, :, None]
    return dy, back.sum(1).to(drows.dtype), dweight


def _tables(s):
    case = s["case"]
    b, p, w, m = case["requests"], case["page"], case["width"], s["slots"].numel()
    if own:
        s["plan"].build(s["held"].data_ptr(), s["added"].data_ptr(), s["free"].data_ptr(), s["pool"].data_ptr(),
                        s["pool_out"].data_ptr(), s["table"].data_ptr(), s["token_offset"].data_ptr(),
                        s["page_offset"].data_ptr(), s["slots"].data_ptr())
        return s["table"], s["token_offset"], s["page_offset"], s["slots"], s["pool_out"]
    held, added, free = s["held"].long(), s["added"].long(), s["free"]
    first, limit = s["pool"][0].long(), s["pool"][1].long()
    have = (held + p - 1) // p
    taken = (torch.minimum((held + added + p - 1) // p, have.new_full((), w)) - have).clamp_min(0)
    zero = taken.new_zeros(1)
    page_offset = first + torch.cat([zero, taken.cumsum(0)])
    token_offset = torch.cat([zero, added.cumsum(0)])
    column = torch.arange(w, device="cuda")[None, :] - have[:, None]
    new = (column >= 0) & (column < taken[:, None])
    at = page_offset[:-1, None] + column
    fresh = torch.where(at < limit, free[at.clamp(0, free.numel() - 1)], -1)
    table = torch.where(new, fresh, s["table"])
    q = torch.arange(m, device="cuda")
    r = (torch.searchsorted(token_offset, q, right=True) - 1).clamp(0, b - 1)
    position = held[r] + q - token_offset[r]
    page = torch.where(position // p < w, table[r, (position // p).clamp(0, w - 1)].long(), -1)
    slots = torch.where((q < token_offset[-1]) & (page >= 0), page * p + position % p, -1)
    after = torch.minimum(page_offset[-1], torch.maximum(limit, first))
    return table, token_offset.int(), page_offset.int(), slots, torch.stack([after, limit]).int()


def _place(case, slots):
    """Indices of the slots' rows in a cache; the spare last page stands for skipped ones."""
    slots = torch.where(slots >= 0, slots, case["pages"] * case["page"])
    page, at = slots // case["page"], slots % case["page"]
    return (page, slice(None), at) if case["headmajor"] else (page, at)


def _paged(s):
    case = s["case"]
    n, m, h, d = case["store"], case["load"], case["heads"], case["size"]
    if own:
        s["store"].store(s["k"].data_ptr(), s["v"].data_ptr(), s["store_slots"].data_ptr(), s["k_cache"].data_ptr(),
                         s["v_cache"].data_ptr(), token_stride=s["k"].stride(0), head_stride=s["k"].stride(1))
        if m:
            s["load"].load(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["load_slots"].data_ptr(),
                           s["k_rows"].data_ptr(), s["v_rows"].data_ptr())
    else:
        where = _place(case, s["store_slots"])
        s["k_cache"][where] = s["k"]
        s["v_cache"][where] = s["v"]
        if m:
            where, ok = _place(case, s["load_slots"]), (s["load_slots"] >= 0)[:, None, None]
            s["k_rows"] = torch.where(ok, s["k_cache"][where], s["k_rows"])
            s["v_rows"] = torch.where(ok, s["v_cache"][where], s["v_rows"])
    used = case["pages"]
    return s["k_cache"][:used], s["v_cache"][:used], s["k_rows"], s["v_rows"]


_RUN = {"sort": _sort, "dispatch": _dispatch, "combine": _combine, "backward": _backward, "tables": _tables, "paged": _paged}


# ---------------------------------------------------------------------------------------------- work and exact values

def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    if case["op"] == "tables":
        pages = case["tokens"] / case["page"] + case["requests"] / 2 if case["tokens"] != case["requests"] else case["requests"] / case["page"]
        return {"bytes": 8 * (case["tokens"] + case["spare"]) + 8 * pages + 16 * case["requests"], "flops": 0}
    if case["op"] == "paged":
        row = case["heads"] * case["size"] * _BYTES[case["type"]]
        return {"bytes": (case["store"] + case["load"]) * (1 - case["skip"]) * 4 * row + 8 * (case["store"] + case["load"]), "flops": 0}
    n, e = case["tokens"] * case["choices"], case["experts"]
    if case["op"] == "sort":
        return {"bytes": n * (case["index"] + 4) + 4 * _capacity(case) + 8 * e, "flops": 0}
    held = n * (1 - case["drop"])
    padding = min(e, n) * (case["align"] - 1) / 2
    token, row = case["tokens"] * case["width"], case["width"] * _BYTES[case["type"]]
    size = _BYTES[case["type"]]
    maps = n * (8 if case["weights"] else 4)
    moved = held * case["width"]
    if case["op"] == "dispatch":
        return {"bytes": token * size + (held + padding) * row + maps, "flops": moved if case["weights"] else 0}
    if case["op"] == "combine":
        return {"bytes": token * size + held * row + maps, "flops": 2 * moved}
    # backward: dout and drows read, dy and dx written; the weights' gradient reads the other factor once more
    other = held * row if case["weights"] == "combine" else token * size
    return {"bytes": 2 * token * size + (2 * held + padding) * row + other + maps + 4 * n, "flops": 6 * moved}


def exact(case, seed):
    return {"tables": _exact_tables, "paged": _exact_paged}.get(case["op"], _exact_rows)(case, seed)


def _exact_rows(case, seed):
    t, k, h, r, e = case["tokens"], case["choices"], case["width"], _capacity(case), case["experts"]
    s = prepare(case, seed)
    if case["op"] == "sort":
        # expert by expert: the slots that name it, in their order
        ids = s["experts"].reshape(-1).cpu()
        count = torch.zeros(e, dtype=torch.int32)
        offset = torch.zeros(e + 1, dtype=torch.int32)
        row_of = torch.full((t * k,), -1, dtype=torch.int32)
        slot_of = torch.full((r,), -1, dtype=torch.int32)
        at = 0
        for i in range(e):
            mine = torch.nonzero(ids == case["first"] + i).reshape(-1).int()
            offset[i], count[i] = at, mine.numel()
            slot_of[at:at + mine.numel()] = mine
            row_of[mine.long()] = torch.arange(at, at + mine.numel(), dtype=torch.int32)
            at += -(-mine.numel() // case["align"]) * case["align"]
        offset[e] = at
        return count.cuda(), offset.cuda(), row_of.view(t, k).cuda(), slot_of.cuda()
    slot_of = s["slot_of"].long()
    live = torch.nonzero(slot_of >= 0).reshape(-1)
    slots = slot_of[live]
    weight = s["weight"].double().reshape(-1) if s["weight"] is not None else None

    def outward(rows, scaled, like):
        if like == torch.int8:
            out = torch.zeros(r, h, dtype=torch.int8, device="cuda")
        else:
            out = torch.zeros(r, h, dtype=torch.float64, device="cuda")
        for at in range(0, live.numel(), 32768):
            part = rows[slots[at:at + 32768] // k]
            if like != torch.int8:
                part = part.double()
                if scaled:
                    part = part * weight[slots[at:at + 32768], None]
            out[live[at:at + 32768]] = part
        return out

    def inward(rows, scaled):
        out = torch.zeros(t, h, dtype=torch.float64, device="cuda")
        row_of = s["row_of"].long()
        for j in range(k):
            has = torch.nonzero(row_of[:, j] >= 0).reshape(-1)
            part = rows[row_of[has, j]].double()
            if scaled:
                part *= weight.view(t, k)[has, j, None]
            out[has] += part
        return out

    def products(rows, tokens):
        out = torch.zeros(t * k, dtype=torch.float64, device="cuda")
        for at in range(0, live.numel(), 16384):
            pick = slots[at:at + 16384]
            out[pick] = torch.einsum("rh,rh->r", rows[live[at:at + 16384]].double(), tokens[pick // k].double())
        return out.view(t, k)

    kind = _TYPES[case["type"]]
    if case["op"] == "dispatch":
        return outward(s["x"], weight is not None, kind)
    if case["op"] == "combine":
        return inward(s["y"], weight is not None)
    if case["weights"] == "combine":
        return outward(s["dout"], True, kind), inward(s["drows"], False), products(s["y"], s["dout"])
    return outward(s["dout"], False, kind), inward(s["drows"], True), products(s["drows"], s["x"])


def _exact_tables(case, seed):
    s = prepare(case, seed)
    held, added = s["held"].tolist(), s["added"].tolist()
    (at, limit), p, w = s["pool"].tolist(), case["page"], case["width"]
    table, free = s["table"].cpu(), s["free"].cpu()
    slots = torch.full((s["slots"].numel(),), -1, dtype=torch.int64)
    tokens, pages = [0], [at]
    for b in range(case["requests"]):
        have = -(-held[b] // p)
        want = min(-(-(held[b] + added[b]) // p), w)
        for i in range(have, want):
            table[b, i] = free[at] if at < limit else -1
            at += 1
        place = torch.arange(held[b], held[b] + added[b])
        page = torch.where(place // p < w, table[b, (place // p).clamp(max=w - 1)].long(), -1)
        slots[tokens[-1]:tokens[-1] + added[b]] = torch.where(page >= 0, page * p + place % p, -1)
        tokens.append(tokens[-1] + added[b])
        pages.append(at)
    whole = torch.int32
    return (table.cuda(), torch.tensor(tokens, dtype=whole).cuda(), torch.tensor(pages, dtype=whole).cuda(),
            slots.cuda(), torch.tensor([min(at, max(limit, s["pool"][0].item())), limit], dtype=whole).cuda())


def _exact_paged(case, seed):
    s = prepare(case, seed)
    p, used = case["page"], case["pages"]
    out = []
    for name in ("k", "v"):
        cache = s[name + "_cache"][:used]
        flat = (cache.transpose(1, 2) if case["headmajor"] else cache).reshape(used * p, case["heads"], case["size"]).clone()
        live = torch.nonzero(s["store_slots"] >= 0).reshape(-1)
        flat[s["store_slots"][live]] = s[name][live]
        rows = torch.zeros_like(s[name + "_rows"])
        live = torch.nonzero(s["load_slots"] >= 0).reshape(-1)
        rows[live] = flat[s["load_slots"][live]]
        back = flat.view(used, p, case["heads"], case["size"])
        out.append(((back.transpose(1, 2) if case["headmajor"] else back).contiguous(), rows))
    return out[0][0], out[1][0], out[0][1], out[1][1]
