"""Performance cases of the paged 8-bit key/value cache: append, attention over it, and the care of its pages.

Operators: new key/value rows enter the cache (`kv8.Kv8Cache.append`), attention reads it (`flash_atten.sdpa_kv8`),
and the pages are given out and copied where they are shared (`reserve`), shared (`fork`), given back (`truncate`)
and moved together (`compact`). Sizes are those of the benchmark, the tests and the decode and prefill harnesses,
and generic odd ones.

The cache: a page holds `page` tokens of every kv head (and layer). `table[b, c]` is the page of sequence b's tokens
c * page .. (c + 1) * page - 1, or -1; `refs[p]` counts the table entries that are p. Within a page, 32 consecutive
tokens of a head are a block: one scale byte e, standing for 2^(e - 127), and a code of 8 bits (e4m3) for each
channel. With `a` the block's largest finite magnitude, e is the exponent byte of float32(a), one more where its
mantissa is over 1.75, less 8, kept where the type holds all codes; a value becomes the code nearest to
value / 2^(e - 127), ties to the even code, at most 448. Infinities and NaN become NaN.

append: rows t < count[b] of sequence b become tokens start[b] + t. A block that gets tokens is encoded anew from
what its earlier tokens stand for and the new rows; tokens of the block behind them become zeros. Rows outside the
capacity, or whose page is missing or has other holders, are dropped.

reserve: entries for tokens start[b] .. start[b] + count[b] - 1 that have no page get the free pages (refs 0) in
order, lowest page first, sequence by sequence; those whose page has other holders get a copy of it, but for the last of
them where every holder is among them.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "flash-attn-economical-gpu_amd")
_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_RANGE = {torch.float16: (112, 134), torch.bfloat16: (10, 246)}  # of scale bytes: 2^-9 and 448 times them fit the type
_BLOCK = 32


def _modules():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import flash_atten
    import kv8

    return flash_atten, kv8


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _append(name, dtype, B, H_kv, rows, capacity, D, page=64, ragged=False):
    return _named(name, {"op": "append", "dtype": dtype, "B": B, "H_kv": H_kv, "rows": rows, "capacity": capacity, "D": D,
                         "page": page, "ragged": ragged})


def _attend(name, dtype, B, H, H_kv, M, capacity, D, page=64, ragged=False, lse=False):
    return _named(name, {"op": "attend", "dtype": dtype, "B": B, "H": H, "H_kv": H_kv, "M": M, "capacity": capacity, "D": D,
                         "page": page, "ragged": ragged, "lse": lse})


def _step(name, B, pages, capacity, page=64):
    return _named(name, {"op": "step", "B": B, "H_kv": 1, "D": 64, "layers": 1, "pages": pages, "capacity": capacity, "page": page})


def _turnover(name, B, rows, pages, capacity, page=64):
    return _named(name, {"op": "turnover", "B": B, "rows": rows, "H_kv": 1, "D": 64, "layers": 1, "pages": pages,
                         "capacity": capacity, "page": page})


def _beams(name, B, beams, children, H_kv, D, layers, pages, capacity, page=64):
    return _named(name, {"op": "beams", "B": B, "beams": beams, "children": children, "H_kv": H_kv, "D": D, "layers": layers,
                         "pages": pages, "capacity": capacity, "page": page})


def _compact(name, B, H_kv, D, layers, pages, live, capacity, page=64):
    return _named(name, {"op": "compact", "B": B, "H_kv": H_kv, "D": D, "layers": layers, "pages": pages, "live": live,
                         "capacity": capacity, "page": page})


def listed():
    return [
        # one new token for each sequence of a serving batch (latency)
        _append("append_bf16_b32_token", "bf16", 32, 8, 1, 8192, 128),
        # prompts of unequal lengths enter the cache; the layer goes on with the values that the cache now holds
        _append("append_bf16_b4_prompts", "bf16", 4, 8, 4096, 8192, 128, ragged=True),
        # decode step of a single sequence against 8k cached tokens
        _attend("attend_bf16_b1_8k", "bf16", 1, 32, 8, 1, 8192, 128),
        # decode step of a serving batch with long caches of unequal lengths (bandwidth)
        _attend("attend_bf16_b8_32k", "bf16", 8, 32, 8, 1, 32768, 128, ragged=True),
        # four drafted tokens are checked at once, head dimension 64, log-sum-exp kept
        _attend("attend_f16_d64_m4", "f16", 4, 16, 2, 4, 65536, 64, ragged=True, lse=True),
        # the large head dimension, an odd capacity and small pages
        _attend("attend_bf16_d256_odd", "bf16", 3, 16, 4, 1, 12345, 256, page=32),
        # a chunk of a long prompt attends to what is cached and to itself (the largest call)
        _attend("attend_f16_chunk_509", "f16", 2, 28, 4, 509, 16384, 128, ragged=True),
        # a first chunk: nothing is cached but the chunk itself
        _attend("attend_bf16_first_2k", "bf16", 2, 32, 8, 2048, 2048, 128),
        # the decode loop's care of pages: what was drafted in vain goes back, the next token gets its page (latency)
        _step("pages_step_b32", 32, 8192, 8192),
        # half of the sequences end and prompts of up to 4k tokens take their places
        _turnover("pages_turnover_b64", 64, 4096, 8192, 8192),
        # beam search over 32 layers: every second beam goes on twice, the last pages are copied
        _beams("pages_beams_l32", 32, 8, 2, 8, 128, 32, 256, 2048),
        # pages in use move together after sequences have come and gone
        _compact("pages_compact_l4", 16, 8, 128, 4, 2048, 1024, 8192),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "step", "turnover", "beams", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    D = rng.choice([64, 128, 128, 256])
    page = rng.choice([32, 64, 64, 128])
    if op == "append":
        H_kv = rng.choice([1, 2, 4, 8])
        B = rng.choice([1, 2, 4, 8, 32])
        rows = rng.choice([1, 1, 4, _log_uniform(rng, 16, 8192), _log_uniform(rng, 16, 8192)])
        while B * H_kv * rows * D > 1 << 25:
            rows = (rows + 1) // 2
        capacity = rows + _log_uniform(rng, 64, 8192)
        while B * H_kv * capacity * D > 1 << 28:
            capacity = rows + (capacity - rows + 1) // 2
        return _append(None, dtype, B, H_kv, rows, capacity, D, page, rng.random() < 0.5)
    if op == "attend":
        H_kv = rng.choice([1, 2, 4, 8])
        H = H_kv * rng.choice([1, 2, 4, 6, 7, 8])
        B = rng.choice([1, 1, 2, 4, 8, 16])
        capacity = _log_uniform(rng, 64, 131072)
        while B * H_kv * capacity * D > 8 * 8 * 32768 * 128:
            capacity = (capacity + 1) // 2
        M = min(rng.choice([1, 1, 1, 3, 8, _log_uniform(rng, 16, 1024)]), capacity)
        while B * H * M * capacity * D > 2 * 28 * 509 * 16384 * 128 // 2:
            M = (M + 1) // 2
        return _attend(None, dtype, B, H, H_kv, M, capacity, D, page, rng.random() < 0.5, M <= 8 and rng.random() < 0.5)
    if op == "step":
        B = rng.choice([1, 8, 32, 64, 128])
        capacity = _log_uniform(rng, 1024, 16384)
        return _step(None, B, B * -(-capacity // page) + rng.randrange(1, 4096), capacity, page)
    if op == "turnover":
        B = rng.choice([8, 16, 32, 64])
        rows = _log_uniform(rng, 64, 4096)
        capacity = rows + _log_uniform(rng, 64, 4096)
        return _turnover(None, B, rows, B * -(-capacity // page) + rng.randrange(1, 1024), capacity, page)
    layers = rng.choice([1, 2, 4, 8])
    H_kv = rng.choice([1, 2, 4, 8])
    if op == "beams":
        beams = rng.choice([2, 3, 4, 8])
        B = beams * rng.choice([1, 2, 4])
        capacity = _log_uniform(rng, 3 * page, 2048)
        return _beams(None, B, beams, rng.choice([c for c in (2, 3, 4, 8) if c <= beams]), H_kv, D, layers,
                      B * -(-capacity // page) + rng.randrange(1, 64), capacity, page)
    pages = _log_uniform(rng, 64, 1024)
    live = rng.randrange(pages // 4, pages - 8)
    B = rng.choice([1, 3, 8, 16])
    return _compact(None, B, H_kv, D, layers, pages, live, -(-live // B) * page, page)


def _lengths(case):
    """Cached tokens of each sequence, new ones included, and how many of the rows given are new tokens."""
    B, capacity = case["B"], case["capacity"]
    rows = case["M"] if case["op"] == "attend" else case["rows"]
    out = []
    for b in range(B):
        total = capacity - (capacity // 2) * b // B if case["ragged"] else capacity
        total = max(total, 1)
        new = min(rows, total)
        if case["ragged"] and rows > 16:
            new = max(1, min(new, rows - (rows // 2) * b // B))
        out.append((total, new))
    return out


def _columns(case):
    return -(-case["capacity"] // case["page"])


def _expand(scales):
    """float32 scale of scale bytes."""
    return (scales.to(torch.int32) << 23).view(torch.float32)


def _quantize(x, dtype):
    """Scale bytes [...] and codes [..., 32, D] of float32 blocks [..., 32, D] of values of the type."""
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), 0.0).amax(dim=(-2, -1)).view(torch.int32)
    e = (((top + 0x1FFFFF) >> 23) - 8).clamp(*_RANGE[dtype])
    y = (x * ((254 - e) << 23).view(torch.float32)[..., None, None]).clamp(-448.0, 448.0)
    codes = y.to(torch.float8_e4m3fn).view(torch.uint8)
    return e.to(torch.uint8), torch.where(finite, codes, 127)


def _dequantize(scales, codes):
    """float32 values of scale bytes [...] and codes [..., 32, D]."""
    return codes.view(torch.float8_e4m3fn).float() * _expand(scales)[..., None, None]


def _tables(case, gen, held):
    """A page table in which sequence b holds pages for its first held[b] tokens, all of them its own, the page
    numbers in no order; and refs."""
    B, page, columns = case["B"], case["page"], _columns(case)
    pages = case.get("pages", B * columns + 7)
    need = torch.tensor([-(-n // page) for n in held], device="cuda")
    column = torch.arange(columns, device="cuda")
    used = column[None, :] < need[:, None]
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((B, columns), -1, device="cuda", dtype=torch.int32)
    rank = used.flatten().cumsum(0).view(B, columns) - 1
    table = torch.where(used, order[rank.clamp(min=0)], table)
    refs = torch.zeros(pages, device="cuda", dtype=torch.int32)
    refs.index_add_(0, table[used].long(), torch.ones_like(table[used]))
    return table, refs


def _random_pages(case, gen):
    """Buffers of a pool whose pages hold codes that are numbers, and scales of ordinary values."""
    shape = (case["layers"], case["pages"], case["H_kv"], case["page"])
    out = []
    for _ in range(2):
        out += [torch.randint(115, 125, (*shape[:3], shape[3] // _BLOCK), device="cuda", generator=gen, dtype=torch.uint8),
                torch.randint(0, 120, (*shape, case["D"]), device="cuda", generator=gen, dtype=torch.uint8)]
    return out


def _inputs(case, seed):
    """The case's tensors: the same values for prepare() and exact()."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    B, D, H_kv, op = case["B"], case["D"], case["H_kv"], case["op"]

    def i32(x):
        return torch.tensor(x, device=dev, dtype=torch.int32)

    def randint(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=dev, generator=gen, dtype=torch.int32)

    if op == "step":  # a third of the sequences stand at the end of a page
        page = case["page"]
        start = randint(1, case["capacity"] - page, B)
        at_end = torch.arange(B, device=dev) % 3 == 0
        start = torch.where(at_end, start // page * page, start)
        table, refs = _tables(case, gen, (start + page).tolist())
        return table, refs, None, start
    if op == "turnover":  # every second sequence ends
        ends = torch.arange(B, device=dev) % 2 == 0
        count = torch.where(ends, randint(case["rows"] // 2, case["rows"] + 1, B), 0)
        held = randint(1, case["capacity"] + 1, B)
        table, refs = _tables(case, gen, held.tolist())
        return table, refs, None, torch.where(ends, 0, held), torch.zeros_like(count), count
    if op == "beams":  # the beams of a prompt have the same length, inside a page
        page, beams = case["page"], case["beams"]
        start = randint(0, _columns(case) - 1, B // beams) * page + randint(1, page, B // beams)
        table, refs = _tables({**case, "B": B // beams}, gen, start.tolist())
        table, start = (t.repeat_interleave(beams, dim=0) for t in (table, start))
        b = torch.arange(B, device=dev, dtype=torch.int32)
        free = (refs == 0).nonzero()[:B, 0].to(torch.int32)  # each beam has written its last page
        table.scatter_(1, (start // page)[:, None].long(), free[:, None])
        refs = _count(table[table >= 0], refs)
        parent = b // beams * beams + b % beams // case["children"]
        return table, refs, _random_pages(case, gen), parent, start
    if op == "compact":
        pages, live = case["pages"], case["live"]
        moved = live * (pages - live) // pages
        low = torch.randperm(live, device=dev, generator=gen)[:live - moved]
        high = live + torch.randperm(pages - live, device=dev, generator=gen)[:moved]
        at = torch.cat((low, high))[torch.randperm(live, device=dev, generator=gen)].to(torch.int32)
        table = torch.full((B * _columns(case),), -1, device=dev, dtype=torch.int32)
        table[:live] = at
        refs = torch.zeros(pages, device=dev, dtype=torch.int32).index_add_(0, at.long(), torch.ones_like(at))
        table = table.view(B, -1)
        return table, refs, _random_pages(case, gen), table.clone(), refs.clone()

    dtype, page = _DTYPES[case["dtype"]], case["page"]
    lengths = _lengths(case)
    order = torch.randperm(B, device=dev, generator=gen).tolist()
    total = [lengths[b][0] for b in order]
    new = [lengths[b][1] for b in order]
    start, count = i32([t - n for t, n in zip(total, new)]), i32(new)
    table, refs = _tables(case, gen, total)
    # channels of keys differ in size by a factor of ten or so, those of values less
    sizes = [(torch.randn(H_kv, 1, D, device=dev, generator=gen) * s).exp() for s in (0.6, 0.2)]
    cache = []
    for size in sizes:
        x = torch.randn(refs.numel(), H_kv, page, D, device=dev, generator=gen) * size
        e, c = _quantize(x.to(dtype).float().unflatten(2, (-1, _BLOCK)), dtype)
        cache += [e[None], c.flatten(2, 3)[None]]
    if op == "append":
        k, v = ((torch.randn(B, case["rows"], H_kv, D, device=dev, generator=gen).transpose(1, 2) * s).to(dtype)
                for s in sizes)
        return table, refs, cache, k, v, start, count
    q = torch.randn(B, case["M"], case["H"], D, device=dev, generator=gen).to(dtype).transpose(1, 2)
    return table, refs, cache, q, start, count


def prepare(case, seed):
    table, refs, pages, *x = _inputs(case, seed)
    state = {"case": case, "table": table, "refs": refs, "pages": pages, "in": x}
    if own:
        cache = _modules()[1].Kv8Cache(
            case["B"], case["H_kv"], case["capacity"], case["D"], dtype=_DTYPES[case.get("dtype", "bf16")],
            pages=refs.numel(), page_size=case["page"], layers=case.get("layers", 1))
        cache.table.copy_(table)
        cache.refs.copy_(refs)
        if pages is not None:
            for held, given in zip((cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes), pages):
                held.copy_(given)
        state = {"case": case, "cache": cache, "in": x}
    return state


def _plain_append(case, table, refs, pages, k, v, start, count):
    """Rows of k and v into the cache. Returns what those rows now stand for (zeros in rows that are no new
    token)."""
    B, H_kv, rows, D = k.shape
    page, columns = case["page"], table.shape[1]
    blocks = (rows + _BLOCK - 2) // _BLOCK + 1  # that rows tokens can lie in
    first = torch.div(start, _BLOCK, rounding_mode="floor")
    at = ((first[:, None] + torch.arange(blocks, device=k.device))[:, :, None] * _BLOCK
          + torch.arange(_BLOCK, device=k.device)).long()  # positions [B, blocks, 32]
    low, high = start.clamp(min=0), (start + count.clamp(0, rows)).clamp(max=case["capacity"])
    row = at - start[:, None, None]
    fresh = (at >= low[:, None, None]) & (at < high[:, None, None])
    kept = at < low[:, None, None]
    column = at[:, :, 0] // page
    there = (column >= 0) & (column < columns)
    p = torch.where(there, table.gather(1, column.clamp(0, columns - 1)), -1).long()
    there &= (p >= 0) & (p < refs.numel())
    p = p.clamp(0, refs.numel() - 1)
    write = there & (refs[p] == 1) & fresh.any(dim=2)
    sub = at[:, :, 0] % page // _BLOCK
    out = []
    for x, scales, codes in ((k, pages[0][0], pages[1][0]), (v, pages[2][0], pages[3][0])):
        codes = codes.view(codes.shape[0], H_kv, page // _BLOCK, _BLOCK, D)
        old = _dequantize(scales[p, :, sub], codes[p, :, sub])  # [B, blocks, H_kv, 32, D]
        index = row.clamp(0, rows - 1).flatten(1)[:, None, :, None].expand(-1, H_kv, -1, D)
        new = x.gather(2, index).float().unflatten(2, (blocks, _BLOCK)).transpose(1, 2)
        block = torch.where(fresh[:, :, None, :, None], new, torch.where(kept[:, :, None, :, None], old, 0.0))
        e, c = _quantize(block, x.dtype)
        where = (p[write], slice(None), sub[write])
        scales[where], codes[where] = e[write], c[write]
        held = _dequantize(e, c).masked_fill(~(write[:, :, None] & fresh)[:, :, None, :, None], 0.0)
        held = held.transpose(1, 2).flatten(2, 3)  # [B, H_kv, blocks * 32, D], position first * 32 on
        take = (torch.arange(rows, device=k.device)[None, :] + (start - first * _BLOCK)[:, None]).long()
        out.append(held.gather(2, take[:, None, :, None].expand(-1, H_kv, -1, D)).to(x.dtype))
    return out


def _plain_attend(case, table, refs, pages, q, start, count):
    B, H, M, D = q.shape
    H_kv, N = case["H_kv"], case["capacity"]
    p = table.long().clamp(min=0)
    values = []
    for scales, codes in ((pages[0][0], pages[1][0]), (pages[2][0], pages[3][0])):
        x = _dequantize(scales[p], codes[p].unflatten(3, (-1, _BLOCK)))  # [B, columns, H_kv, blocks, 32, D]
        values.append(x.transpose(1, 2).reshape(B, H_kv, -1, D)[:, :, :N])
    row, column = torch.arange(M, device=q.device), torch.arange(N, device=q.device)
    there = (table >= 0).repeat_interleave(case["page"], dim=1)[:, :N] & (column < (start + count)[:, None])
    seen = (column <= (start[:, None] + row)[:, :, None]) & (row < count[:, None])[:, :, None] & there[:, None, :]
    kf, vf = (t.masked_fill_(~there[:, None, :, None], 0.0) for t in values)
    qf = q.float().reshape(B, H_kv, -1, D)
    s = (qf @ kf.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(B, H_kv, -1, M, N)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = s.sub_(top).exp_()
    total = e.sum(dim=-1, keepdim=True)
    o = (e.view(B, H_kv, -1, N) @ vf).view_as(e[..., :1].expand(-1, -1, -1, -1, D)) / total
    o = o.masked_fill(total == 0, 0.0).reshape(B, H, M, D).to(q.dtype)
    return (o, (top + total.log()).reshape(B, H, M)) if case["lse"] else o


def _count(entries, like):
    return torch.zeros_like(like).index_add_(0, entries.long(), torch.ones_like(entries, dtype=like.dtype))


def _plain_truncate(case, table, refs, length):
    gone = torch.arange(table.shape[1], device=table.device) >= ((length + case["page"] - 1) // case["page"])[:, None]
    refs -= _count(table[gone & (table >= 0)], refs)
    table.masked_fill_(gone, -1)


def _plain_fork(table, refs, parent):
    old = table.clone()
    table.copy_(torch.where((parent >= 0)[:, None], old[parent.clamp(min=0).long()], -1))
    refs += _count(table[table >= 0], refs) - _count(old[old >= 0], refs)


def _plain_reserve(case, table, refs, pages, start, rows, count):
    """Returns how many pages were wanting."""
    page, columns = case["page"], table.shape[1]
    low, high = start.clamp(min=0), (start + count.clamp(0, rows)).clamp(max=case["capacity"])
    span = (rows + page - 2) // page + 1
    column = low[:, None] // page + torch.arange(span, device=table.device)
    active = (column * page < high[:, None]) & (high > low)[:, None]
    column = column.clamp(max=columns - 1).long()
    entry = table.gather(1, column)
    held = active & (entry >= 0)
    shared = held & (refs[entry.clamp(min=0).long()] > 1)
    item = torch.arange(entry.numel(), device=table.device).view_as(entry)
    safe = entry.clamp(min=0).long()
    writers = _count(entry[shared], refs)
    last = torch.full((refs.numel(),), -1, device=table.device).scatter_reduce_(0, safe[shared], item[shared], "amax")
    keeps = shared & (writers == refs)[safe] & (last[safe] == item)
    copied = shared & ~keeps
    wants = (active & ~held) | copied
    rank = wants.flatten().cumsum(0).view_as(entry) - 1
    free = refs == 0
    order = torch.sort(free, descending=True, stable=True).indices  # free pages first, lowest first
    given = wants & (rank < free.sum())
    page_of = order[rank.clamp(0, refs.numel() - 1)].to(torch.int32)
    refs += _count(page_of[given], refs) - _count(entry[given & copied], refs)
    b = torch.arange(table.shape[0], device=table.device)[:, None].expand_as(column)
    table[b[given], column[given]] = page_of[given]
    if pages is not None:
        source, target = entry[given & copied].long(), page_of[given & copied].long()
        for x in pages:
            x[:, target] = x[:, source]
    return (wants.sum() - given.sum()).to(torch.int32).view(1)


def _plain_compact(table, refs, pages):
    """Returns the number of pages in use."""
    used = refs > 0
    live = used.sum()
    index = torch.arange(refs.numel(), device=refs.device)
    source, target = index[used & (index >= live)], index[~used & (index < live)]
    for x in pages:
        x[:, target] = x[:, source]
    to = index.to(torch.int32)
    to[source] = target.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[target] = refs[source]
    refs[source] = 0
    return live.to(torch.int32).view(1)


def _run_own(case, cache, x):
    op, held = case["op"], (cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes)
    if op == "append":
        return (*cache.append(x[0], x[1], x[2], count=x[3], return_values=True), *held)
    if op == "attend":
        return _modules()[0].sdpa_kv8(x[0], cache, x[1], count=x[2], return_lse=case["lse"])
    if op == "step":
        cache.truncate(x[0])
        return cache.reserve(x[0], 1), cache.table, cache.refs
    if op == "turnover":
        cache.truncate(x[0])
        return cache.reserve(x[1], case["rows"], count=x[2]), cache.table, cache.refs
    if op == "beams":
        cache.fork(x[0])
        return (cache.reserve(x[1], 1), cache.table, cache.refs, *held)
    cache.table.copy_(x[0])
    cache.refs.copy_(x[1])
    return (cache.compact(), cache.table, cache.refs, *held)


def run(state):
    if own:
        return _run_own(state["case"], state["cache"], state["in"])
    case, table, refs, pages, x = (state[n] for n in ("case", "table", "refs", "pages", "in"))
    op = case["op"]
    if op == "append":
        return (*_plain_append(case, table, refs, pages, *x), *pages)
    if op == "attend":
        return _plain_attend(case, table, refs, pages, *x)
    if op == "step":
        _plain_truncate(case, table, refs, x[0])
        return _plain_reserve(case, table, refs, pages, x[0], 1, torch.ones_like(x[0])), table, refs
    if op == "turnover":
        _plain_truncate(case, table, refs, x[0])
        return _plain_reserve(case, table, refs, pages, x[1], case["rows"], x[2]), table, refs
    if op == "beams":
        _plain_fork(table, refs, x[0])
        return (_plain_reserve(case, table, refs, pages, x[1], 1, torch.ones_like(x[1])), table, refs, *pages)
    table.copy_(x[0])
    refs.copy_(x[1])
    return (_plain_compact(table, refs, pages), table, refs, *pages)


def work(case):
    B, D, H_kv, op, page = (case[n] for n in ("B", "D", "H_kv", "op", "page"))
    if op == "append":
        new = sum(n for _, n in _lengths(case))
        # rows in, codes out, what the rows stand for out (two bytes a channel for all rows)
        return {"bytes": 2 * H_kv * D * (new * 3 + 2 * B * case["rows"]), "flops": 4 * H_kv * new * D}
    if op == "attend":
        H, M = case["H"], case["M"]
        keys = pairs = 0
        for total, new in _lengths(case):
            keys += total
            pairs += sum(total - new + i + 1 for i in range(new))
        return {"bytes": 2 * H_kv * keys * D + 4 * B * H * M * D + (4 * B * H * M if case["lse"] else 0),
                "flops": 4 * H * pairs * D}
    table = 4 * B * _columns(case)
    if op in ("step", "turnover"):  # entries and lengths are read, half of the entries or so change
        return {"bytes": 8 * B + 2 * table, "flops": 0}
    # a page's bytes in all layers, read once and written once for each page that is copied
    size = 2 * case["layers"] * H_kv * (page * D + page // _BLOCK)
    if op == "beams":
        copies = B // case["beams"] * (case["beams"] - -(-case["beams"] // case["children"]))
        return {"bytes": 2 * copies * size + 2 * table, "flops": 0}
    moved = case["live"] * (case["pages"] - case["live"]) // case["pages"]
    return {"bytes": 2 * moved * size + 2 * table + 8 * case["pages"], "flops": 0}


def _power(n):
    """2^n in 64 bits, of whole numbers n (a power function may be off in the last bit, which moves ties)."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _exact_codes(scales, codes):
    """64-bit values of scale bytes [...] and codes [..., 32, D], from sign, exponent and mantissa."""
    c = codes.int()
    exponent, mantissa = (c >> 3) & 15, (c & 7).double()
    value = torch.where(exponent > 0, (8 + mantissa) * _power(exponent - 10), mantissa * 2.0 ** -9)
    value = torch.where((c & 127) == 127, math.nan, value) * (1 - 2 * (c >> 7))
    return value * _power(scales.int() - 127)[..., None, None]


def _exact_values(x, dtype):
    """64-bit values that a block [..., 32, D] of 64-bit values is held as."""
    finite = torch.isfinite(x)
    a = torch.where(finite, x, 0.0).abs().amax(dim=(-2, -1), keepdim=True)
    mantissa, exponent = torch.frexp(a)  # a = mantissa 2^exponent, mantissa in [0.5, 1)
    power = torch.where(a > 0, exponent - 9 + (mantissa > 0.875), -1000).clamp(*(e - 127 for e in _RANGE[dtype]))
    scale = _power(power)
    y = torch.where(finite, x, 0.0) / scale
    # numbers of a binade are 2^-3 of its power apart, those below 2^-6 are 2^-9 apart
    step = _power((torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
    held = (torch.round(y / step) * step).clamp(-448.0, 448.0) * scale  # round() takes ties to even
    return torch.where(finite, held, math.nan)


def _exact_append(case, table, refs, cache, k, v, start, count):
    B, H_kv, rows, D = k.shape
    page, out = case["page"], []
    for x, scales, codes in ((k, cache[0][0], cache[1][0]), (v, cache[2][0], cache[3][0])):
        values = torch.zeros(B, H_kv, rows, D, device=k.device, dtype=torch.float64)
        for b in range(B):
            s, n = int(start[b]), int(count[b])
            lead = s % _BLOCK
            line = torch.zeros(H_kv, -(-(lead + n) // _BLOCK) * _BLOCK, D, device=k.device, dtype=torch.float64)
            line[:, lead:lead + n] = x[b, :, :n].double()
            if lead:  # earlier tokens of the first block
                p, sub = int(table[b, s // page]), s % page // _BLOCK
                block = codes[p, :, sub * _BLOCK:sub * _BLOCK + _BLOCK]
                line[:, :lead] = _exact_codes(scales[p, :, sub], block)[:, :lead]
            held = _exact_values(line.unflatten(1, (-1, _BLOCK)), x.dtype).flatten(1, 2)
            values[b, :, :n] = held[:, lead:lead + n]
        out.append(values)
    # the cache's own bytes are whole numbers: equal to the plain form's, or wrong
    return (*out, None, None, None, None)


def _exact_attend(case, table, refs, cache, q, start, count):
    B, H, M, D = q.shape
    group = H // case["H_kv"]
    out = torch.zeros(B, H, M, D, device=q.device, dtype=torch.float64)
    lse = torch.full((B, H, M), -math.inf, device=q.device, dtype=torch.float64)
    for b in range(B):
        first, new = int(start[b]), int(count[b])
        n = first + new
        p = table[b, : -(-n // case["page"])].long()
        for h in range(case["H_kv"]):
            keys, held = (_exact_codes(s[0, p, h], c[0, p, h].unflatten(1, (-1, _BLOCK))).reshape(-1, D)[:n]
                          for s, c in ((cache[0], cache[1]), (cache[2], cache[3])))
            hidden = torch.ones(new, n, device=q.device, dtype=torch.bool).triu(first + 1)
            for g in range(h * group, (h + 1) * group):
                s = (q[b, g, :new].double() @ keys.t().contiguous() / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                out[b, g, :new] = torch.softmax(s, dim=1) @ held
                lse[b, g, :new] = torch.logsumexp(s, dim=1)
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    if case["op"] not in ("append", "attend"):
        return None  # whole numbers only
    return (_exact_append if case["op"] == "append" else _exact_attend)(case, *_inputs(case, seed))
