"""The paged 8-bit key/value cache: what append writes and what the page operations do against the definition (equal),
attention over it against the softmax in 64 bits, and all of them together as a serving loop uses them."""
from __future__ import annotations

import math
import random

import pytest
import torch

import flash_atten
import hip_lib
import kv8
from kv8_model import Model, check_attention

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(seed, *shape, dtype, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).to(dtype)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _deal(cache, tokens, seed=0):
    """Pages for the sequences' first tokens, in no order."""
    pages = list(range(cache.pages))
    random.Random(seed).shuffle(pages)
    for b, n in enumerate(tokens):
        for c in range(-(-n // cache.page_size)):
            page = pages.pop()
            cache.table[b, c] = page
            cache.refs[page] = 1


def _fill(cache, byte=0xAB):
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.fill_(byte)


def _equal(got, want):
    return torch.equal(got.double().cpu().nan_to_num(1e9), want.nan_to_num(1e9))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_writes_the_format(gpu, dtype, D):
    """Rows of all sizes, ties, infinities and NaN, in blocks that are begun, continued and begun again."""
    print(f"[kv8] append {dtype} {D}", flush=True)
    B, Hk, rows, capacity = 2, 3, 75, 200
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=dtype, pages=11, page_size=64, layers=2)
    _fill(cache)
    _deal(cache, [200, 200])
    model = Model(cache)
    k = _rand(1, B, rows, Hk, D, dtype=torch.float32)
    v = _rand(2, B, rows, Hk, D, dtype=torch.float32) * torch.logspace(-9, 4, rows)[None, :, None, None]
    k[0, 0] = 0
    k[0, 1] = -0.0
    k[0, 2, 0, :8] = torch.tensor([448.0, 432.0, 416.0, 0.2578125, 0.0009765625, 0.00293, 0.0029296875, 1.0625])
    k[1, 40:, :] *= 3e-7
    k, v = k.to(dtype), v.to(dtype)
    k[1, 3, 1, 5], k[1, 4, 0, 40], v[1, 5, 2, 0] = math.inf, math.nan, -math.inf
    v[0, 30:, 1] = math.nan
    k[1, 6, 0], v[1, 6, 0] = torch.finfo(dtype).max, torch.finfo(dtype).tiny / 4
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    kd, vd = k.cuda(), v.cuda()
    for layer, start, count in ((0, (5, 64), (75, 20)), (1, (0, 31), None), (0, (80, 70), (1, 75)), (0, (81, 3), (1, 1)),
                                (0, (79, 90), (17, 0)), (1, (75, 106), (40, 75)), (0, (32, 96), (32, 32))):
        counts = None if count is None else _i32(*count)
        held = cache.append(kd, vd, _i32(*start), count=counts, layer=layer, return_values=True)
        want = model.append(k, v, start, count, layer)
        assert _equal(held[0], want[0]) and _equal(held[1], want[1]), (layer, start, count)
        model.check(cache, (layer, start, count))
    # without values, from contiguous memory
    assert cache.append(kd.contiguous(), vd.contiguous(), _i32(100, 7), layer=1) is None
    model.append(k, v, (100, 7), None, 1)
    model.check(cache)


@pytest.mark.parametrize("page", [32, 64, 128, 256])
def test_append_drops_what_has_no_place(gpu, page):
    """Rows outside the capacity, on missing, foreign and shared pages; lengths at the ends of the type."""
    B, Hk, D, capacity = 5, 2, 64, 300
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=BF16, pages=60, page_size=page)
    _fill(cache)
    _deal(cache, [300, 300, 300, 300, 300])
    cache.table[1, 0] = -1
    cache.table[2, 0] = cache.pages
    cache.table[3, 0] = -2 ** 31
    cache.refs[cache.table[4, 0].long()] = 2
    model = Model(cache)
    k, v = (_rand(i, B, Hk, 70, D, dtype=BF16) for i in (3, 4))
    kd, vd = k.cuda(), v.cuda()
    for start, count in (((-20, 0, 0, 0, 0), None), ((250, 20, 20, 20, 20), None), ((299, 300, 301, -70, -71), None),
                         ((2 ** 31 - 1, -2 ** 31, 2 ** 31 - 40, 290, 250), (70, 70, 70, 2 ** 31 - 1, 3)), ((0,) * 5, (0, -1, -2 ** 31, 0, 0))):
        values = cache.append(kd, vd, _i32(*start), count=None if count is None else _i32(*count), return_values=True)
        want = model.append(k, v, start, count)
        assert _equal(values[0], want[0]) and _equal(values[1], want[1]), (start, count)
        model.check(cache, (start, count))
    cache.append(kd[:, :, :0], vd[:, :, :0], _i32(*[0] * 5))
    model.check(cache)


CASES = [  # B, H, Hk, M, capacity, D, page, starts, counts
    (1, 1, 1, 1, 1, 64, 32, [0], None), (2, 4, 4, 1, 40, 64, 32, [39, 0], None), (1, 8, 2, 1, 700, 128, 64, [650], None),
    (3, 6, 2, 1, 300, 128, 64, [-1, 31, 299], None), (1, 8, 1, 1, 1000, 256, 128, [777], None), (2, 7, 1, 4, 333, 64, 256, [100, 329], None),
    (1, 16, 2, 4, 600, 128, 32, [500], None), (2, 4, 2, 5, 90, 256, 64, [60, 3], [5, 2]), (1, 4, 2, 70, 500, 128, 64, [400], None),
    (2, 2, 1, 129, 400, 64, 32, [0, 200], [129, 64]), (2, 6, 2, 100, 260, 128, 128, [-50, 160], [100, 0]),
    (1, 4, 4, 65, 130, 256, 64, [50], None), (1, 32, 8, 1, 9000, 128, 64, [8500], None), (2, 28, 4, 3, 2100, 128, 32, [2000, 513], None),
    (1, 2, 2, 300, 2500, 64, 64, [2100], None), (2, 3, 1, 8, 64, 128, 64, [60, 2 ** 31 - 5], None), (1, 2, 1, 33, 3000, 256, 32, [2900], [30]),
    (2, 2, 1, 200, 200, 128, 32, [0, 0], [200, 77]), (1, 1, 1, 2, 40000, 64, 32, [39900], None), (3, 12, 2, 40, 1000, 64, 256, [900, 31, 480], [40, 40, 1]),
]


def _full(seed, B, Hk, capacity, D, page, dtype, layers=1):
    """A cache whose every token is written."""
    columns = -(-capacity // page)
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=dtype, pages=B * columns + 3, page_size=page, layers=layers)
    _deal(cache, [capacity] * B, seed)
    for layer in range(layers):
        k, v = (_rand(seed + i + 10 * layer, B, Hk, capacity, D, dtype=dtype).cuda() for i in range(2))
        cache.append(k, v, _i32(*[0] * B), layer=layer)
    return cache


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:7])))
def test_attention_over_the_cache(gpu, case, dtype, causal):
    B, H, Hk, M, capacity, D, page, starts, counts = case
    print(f"[kv8] {case} {dtype} causal={causal}", flush=True)
    cache = _full(10 + capacity, B, Hk, capacity, D, page, dtype)
    # what lies behind a sequence is not read, NaN there changes nothing; nor are its table entries
    for b in range(B):
        n = M if counts is None else max(0, counts[b])
        end = max(0, min(capacity, starts[b] + n)) if n else 0
        for t in range(end, capacity if capacity < 3000 else end + 40):
            for codes in (cache.k_codes, cache.v_codes):
                codes[0, cache.table[b, t // page].long(), :, t % page] = 127
        cache.table[b, -(-end // page):] = 2 ** 31 - 1
    q = _rand(20, B, M, H, D, dtype=dtype).cuda().transpose(1, 2)
    count = None if counts is None else _i32(*counts)
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(*starts), count=count, is_causal=causal, return_lse=True)
    want = Model(cache).attention(q, starts, counts, causal=causal)
    check_attention(o, lse, *want, (case, dtype, causal))
    assert torch.equal(o, flash_atten.sdpa_kv8(q.contiguous(), cache, _i32(*starts), count=count, is_causal=causal))


@pytest.mark.parametrize("splits", [1, 2, 5, 33])
@pytest.mark.parametrize("M", [1, 6, 40])
def test_any_number_of_splits(gpu, monkeypatch, splits, M):
    B, H, Hk, capacity, D = 2, 8, 2, 3000, 128
    cache = _full(40, B, Hk, capacity, D, 64, BF16)
    q = _rand(41, B, H, M, D, dtype=BF16).cuda()
    starts = [capacity - M, 700]
    monkeypatch.setattr(kv8, "choose_splits", lambda *a: splits)
    monkeypatch.setattr(flash_atten, "_plans", {})
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(*starts), scale=0.2, return_lse=True)
    check_attention(o, lse, *Model(cache).attention(q, starts, scale=0.2), (splits, M))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("M", [3, 9, 150])
def test_missing_pages_are_not_seen(gpu, M, D):
    """Entries -1 and out of range at the front, in the middle and at the end; a sequence without any page."""
    B, H, Hk, capacity = 4, 4, 2, 600
    cache = _full(50, B, Hk, capacity, D, 32, F16)
    cache.table[0, 0], cache.table[0, 7], cache.table[0, 8] = -1, cache.pages, -5
    cache.table[1, 10:] = -1
    cache.table[2, ::2] = -1
    cache.table[3] = -1
    q = _rand(51, B, H, M, D, dtype=F16).cuda()
    starts = [capacity - M, 400, 250, 300]
    for causal in (True, False):
        o, lse = flash_atten.sdpa_kv8(q, cache, _i32(*starts), is_causal=causal, return_lse=True)
        want = Model(cache).attention(q, starts, causal=causal)
        check_attention(o, lse, *want, (M, D, causal))
        assert not o[3].any() and torch.isinf(lse[3]).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("M", [6, 14, 130])
def test_nan_reaches_the_rows_that_see_it(gpu, M, D, dtype):
    """A NaN in a value takes its channel of the rows that see its token, one in a key the rows; no others, although they
    are computed in the same tiles."""
    B, H, Hk, capacity = 1, 2, 1, 400
    cache = _full(60, B, Hk, capacity, D, 64, dtype)
    q = _rand(61, B, H, M, D, dtype=dtype).cuda()
    start = 230
    clean, clean_lse = flash_atten.sdpa_kv8(q, cache, _i32(start), return_lse=True)
    for token, channel, key in ((start + 1, 5, False), (start + M // 2, D - 1, False), (start + M // 2, 17, True), (start + M - 1, 0, False)):
        codes = cache.k_codes if key else cache.v_codes
        page = int(cache.table[0, token // 64])
        was = codes[0, page, 0, token % 64, channel].clone()
        codes[0, page, 0, token % 64, channel] = 255
        o, lse = flash_atten.sdpa_kv8(q, cache, _i32(start), return_lse=True)
        codes[0, page, 0, token % 64, channel] = was
        first = token - start
        assert torch.equal(o[:, :, :first], clean[:, :, :first]) and torch.equal(lse[:, :, :first], clean_lse[:, :, :first])
        if key:
            assert torch.isnan(o[:, :, first:]).all() and torch.isnan(lse[:, :, first:]).all()
        else:
            assert torch.isnan(o[:, :, first:, channel]).all() and torch.equal(lse, clean_lse)
            rest = [c for c in range(D) if c != channel]
            assert torch.isfinite(o[..., rest]).all()


def test_large_scores_and_odd_scale_bytes(gpu):
    """Scores far apart (the running maximum moves); scale bytes past the largest read as that."""
    B, H, Hk, capacity, D = 1, 4, 2, 500, 64
    for dtype in (F16, BF16):
        cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=dtype)
        _deal(cache, [capacity])
        k, v = (_rand(70 + i, B, Hk, capacity, D, dtype=torch.float32) for i in range(2))
        k = (k * torch.linspace(0.1, 12, capacity)[None, None, :, None]).to(dtype).cuda()
        cache.append(k, v.to(dtype).cuda(), _i32(0))
        q = _rand(72, B, H, 1, D, dtype=dtype, sigma=4.0).cuda()
        o, lse = flash_atten.sdpa_kv8(q, cache, _i32(capacity - 1), return_lse=True)
        want = Model(cache).attention(q, [capacity - 1])
        assert ((o.double().cpu() - want[0]).abs() <= 1.01 * want[2]).all()
        top = 134 if dtype == F16 else 246
        q.mul_(2.0 ** -30 if dtype == BF16 else 2.0 ** -9)
        out = []
        for e in (top, top + 1, 255):
            cache.k_scales.fill_(e)
            out.append(flash_atten.sdpa_kv8(q, cache, _i32(capacity - 1)))
        assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_scores_far_from_zero(gpu, monkeypatch, dtype, M, splits):
    """Scores of 2^21 that differ by a few: softmax is of the differences, whatever the scores themselves are.

    Scores are exact (two channels: 2^11 x 2^10, and 1 x a multiple of 1/2), so are their differences. An exponent is
    a difference times scale x log2 e, rounded: 2^-24 x 2 x 24 x 1.45 x ln 2 < 2^-18. Where parts are joined, each is
    known by fl(m c), of about 3 x 2^20: half a step is 1/8, two of them 1/4, a factor of 2^(1/4) at most."""
    B, H, Hk, capacity, D = 1, 2, 2, 400, 64
    monkeypatch.setattr(kv8, "choose_splits", lambda *a: splits)
    monkeypatch.setattr(flash_atten, "_plans", {})
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=dtype)
    _deal(cache, [capacity])
    k, v = torch.zeros(B, Hk, capacity, D), _rand(5, B, Hk, capacity, D, dtype=dtype)
    k[..., 0] = 2.0 ** 10
    k[..., 1] = torch.arange(capacity)[None, None] // 64 * 3.5 + torch.arange(capacity)[None, None] % 3  # it keeps growing
    cache.append(k.to(dtype).cuda(), v.cuda(), _i32(0))
    q = torch.zeros(B, H, M, D)
    q[..., 0], q[..., 1] = 2.0 ** 11, 1.0
    q = q.to(dtype).cuda()
    for start in (capacity - M, 300, 100):
        o = flash_atten.sdpa_kv8(q, cache, _i32(start), scale=1.0)
        model = Model(cache)
        want, lse, _ = model.attention(q, [start], scale=1.0)
        keys, values, _ = model.line(0, 0)
        mass = torch.stack([torch.softmax((q[0, h].double().cpu() @ keys[h].t()).masked_fill(
            torch.arange(capacity)[None] > start + torch.arange(M)[:, None], -math.inf), -1) @ values[h].abs() for h in range(H)])
        u = torch.finfo(dtype).eps / 2
        e = 2 * 2.0 ** -18 + (0.0 if splits == 1 else 2 * (2.0 ** 0.25 - 1))
        assert ((o[0].double().cpu() - want[0]).abs() <= 1.01 * ((u + e) * mass + u * want[0].abs() + 2.0 ** -24)).all()


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("M", [1, 40])
def test_a_scale_of_almost_nothing(gpu, monkeypatch, M, splits):
    """A scale below the smallest normal number: every key weighs the same, the result is the mean of the values (of 400
    terms at most, summed in fp32; the weights are exact)."""
    B, H, Hk, capacity, D = 1, 4, 2, 400, 64
    monkeypatch.setattr(kv8, "choose_splits", lambda *a: splits)
    monkeypatch.setattr(flash_atten, "_plans", {})
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=F16)
    _deal(cache, [capacity])
    cache.append(*(_rand(i, B, Hk, capacity, D, dtype=F16).cuda() for i in range(2)), _i32(0))
    q = _rand(2, B, H, M, D, dtype=F16).cuda()
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(capacity - M), scale=1e-39, return_lse=True)
    _, values, _ = Model(cache).line(0, 0)
    for h in range(H):
        for i in range(M):
            v = values[h // 2, :capacity - M + i + 1]
            mean, u = v.mean(0), 2.0 ** -11
            assert ((o[0, h, i].double().cpu() - mean).abs() <= u * mean.abs() + 400 * 2.0 ** -24 * v.abs().mean(0) + 2.0 ** -25).all()
            assert abs(float(lse[0, h, i]) - math.log(len(v))) <= 2e-6


def _state(seed, B, capacity, page, pages, layers=1, D=64, Hk=1):
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=BF16, pages=pages, page_size=page, layers=layers)
    g = torch.Generator().manual_seed(seed)
    cache._data.copy_(torch.randint(0, 256, cache._data.shape, generator=g, dtype=torch.uint8))
    return cache, Model(cache)


@pytest.mark.parametrize("seed", range(12))
def test_page_operations(gpu, seed):
    """Any order of reserve, fork, truncate and compact, with pools that run short: table, counts and every page's bytes."""
    rng = random.Random(seed)
    B, page, layers = rng.choice([1, 2, 5, 9, 70]), rng.choice([32, 64, 128, 256]), rng.choice([1, 3])
    capacity = rng.choice([1, 100, 900, 5000])
    columns = -(-capacity // page)
    pages = rng.choice([1, 3, B * columns // 2 + 1, B * columns + 5, 9000 // layers])
    print(f"[kv8] pages seed={seed} B={B} page={page} layers={layers} capacity={capacity} pages={pages}", flush=True)
    cache, model = _state(seed, B, capacity, page, pages, layers)
    for step in range(14):
        op = rng.choice(["reserve", "reserve", "reserve", "fork", "truncate", "compact"])
        if op == "reserve":
            rows = rng.choice([0, 1, 1, 4, page, page + 1, capacity, capacity + 500])
            start = [rng.randint(-3, capacity + 3) for _ in range(B)]
            count = None if rng.random() < 0.4 else [rng.choice([-1, 0, 1, rows, rows + 9, rng.randint(0, rows + 1)]) for _ in range(B)]
            got = cache.reserve(_i32(*start), rows, count=None if count is None else _i32(*count))
            assert int(got) == model.reserve(start, rows, count), (seed, step)
        elif op == "fork":
            parent = [rng.choice([b, rng.randint(0, B - 1), rng.randint(0, B - 1), rng.choice([-1, B, -2 ** 31, 2 ** 31 - 1])]) for b in range(B)]
            cache.fork(_i32(*parent))
            model.fork(parent)
        elif op == "truncate":
            length = [rng.choice([-1, 0, capacity, 2 ** 31 - 1, rng.randint(0, capacity)]) for _ in range(B)]
            cache.truncate(_i32(*length))
            model.truncate(length)
        else:
            assert int(cache.compact()) == model.compact(), (seed, step)
        model.check(cache, (seed, step, op))
    assert torch.equal(torch.bincount(model.table[model.table >= 0], minlength=pages).int(), model.refs)


def test_writers_of_a_shared_page(gpu):
    """Of a page's holders that write, all but the last are copied where every holder writes, and all of them otherwise."""
    for writes, kept in (((1, 1, 1, 1), 3), ((1, 1, 0, 1), None), ((1, 0, 0, 0), None), ((0, 0, 0, 0), None)):
        cache, model = _state(5, 4, 256, 64, 30, layers=2)
        for x in (cache, model):
            x.reserve(_i32(0, 0, 0, 0) if x is cache else [0] * 4, 200, count=_i32(200, 0, 0, 0) if x is cache else [200, 0, 0, 0])
            x.fork(_i32(0, 0, 0, 0) if x is cache else [0] * 4)
        before = cache.table.clone()
        cache.reserve(_i32(*[199] * 4), 1, count=_i32(*writes))
        model.reserve([199] * 4, 1, writes)
        model.check(cache, writes)
        changed = (cache.table != before).any(1).tolist()
        assert changed == [bool(w) and b != kept for b, w in enumerate(writes)]
        for b, w in enumerate(writes):
            assert not w or int(cache.refs[cache.table[b, 3].long()]) == 1


def test_the_same_page_twice(gpu):
    """A table written by hand that names one page in two columns: each is a holder."""
    cache, model = _state(6, 2, 256, 64, 9)
    cache.table[0, 0] = cache.table[0, 1] = cache.table[1, 0] = 4
    cache.refs[4] = 3
    model.pull(cache)
    cache.reserve(_i32(0, 0), 128, count=_i32(128, 1))
    model.reserve([0, 0], 128, [128, 1])
    model.check(cache)
    cache.compact()
    model.compact()
    model.check(cache)


def test_no_sequences(gpu):
    cache = kv8.Kv8Cache(0, 2, 100, 64, dtype=F16, pages=5, layers=2)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    kv = torch.zeros(0, 2, 3, 64, dtype=F16, device="cuda")
    assert cache.reserve(none, 3).tolist() == [0] and cache.reserve(none, 3, count=none).tolist() == [0]
    got = cache.append(kv, kv, none, return_values=True)
    assert [t.shape for t in got] == [kv.shape] * 2
    o, lse = flash_atten.sdpa_kv8(torch.zeros(0, 4, 3, 64, dtype=F16, device="cuda"), cache, none, return_lse=True)
    assert o.shape == (0, 4, 3, 64) and lse.shape == (0, 4, 3)
    cache.fork(none)
    cache.truncate(none)
    assert cache.compact().tolist() == [0] and cache.refs.tolist() == [0] * 5


def test_large_pools_and_tables(gpu):
    """Many steps of each search: 70000 pages, 130 sequences; reserve of 65000 entries, compaction of a pool in use at both
    ends."""
    B, page, capacity, pages = 130, 32, 16000, 70000
    cache = kv8.Kv8Cache(B, 1, capacity, 64, dtype=F16, pages=pages, page_size=page)
    model = Model(cache)
    rng = random.Random(9)
    for count in ([capacity] * B, [0] * 60 + [capacity] * 70):
        assert int(cache.reserve(_i32(*[0] * B), capacity, count=_i32(*count))) == model.reserve([0] * B, capacity, count)
        model.check(cache, "reserve")
        length = [rng.choice([0, capacity, rng.randint(0, capacity)]) for _ in range(B)]
        cache.truncate(_i32(*length))
        model.truncate(length)
        parent = [rng.randint(0, B - 1) if b % 3 == 0 else b for b in range(B)]
        cache.fork(_i32(*parent))
        model.fork(parent)
        model.check(cache, "fork")
        assert int(cache.compact()) == model.compact()
        model.check(cache, "compact")


def test_beam_search(gpu):
    """A prompt is shared by beams, which fork, write and are dropped, in two layers: what each step gives against the
    64-bit softmax over what the model's cache holds."""
    B, H, Hk, D, capacity, page, dtype, layers, prompt, steps = 6, 8, 2, 128, 320, 64, BF16, 2, 150, 7
    cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=dtype, pages=14, page_size=page, layers=layers)
    model = Model(cache)
    rng = random.Random(3)

    def both(name, *lists, **kw):
        got = getattr(cache, name)(*(_i32(*x) if isinstance(x, list) else x for x in lists),
                                   **{n: _i32(*x) for n, x in kw.items()})
        want = getattr(model, name)(*lists, **kw)
        if want is not None:
            assert int(got) == want, name

    first = [prompt] + [0] * (B - 1)
    both("reserve", [0] * B, prompt, count=first)
    for layer in range(layers):
        k, v, q = (_rand(80 + 3 * layer + i, B, prompt, n, D, dtype=dtype).transpose(1, 2) for i, n in enumerate((Hk, Hk, H)))
        cache.append(k.cuda(), v.cuda(), _i32(*[0] * B), count=_i32(*first), layer=layer)
        model.append(k, v, [0] * B, first, layer)
        o, lse = flash_atten.sdpa_kv8(q.cuda(), cache, _i32(*[0] * B), count=_i32(*first), layer=layer, return_lse=True)
        check_attention(o, lse, *model.attention(q, [0] * B, first, layer), ("prompt", layer))
    model.check(cache, "prompt")
    parent = [0] * B
    for step in range(steps):
        start = [prompt + step] * B
        both("fork", parent)
        both("reserve", start, 1)
        for layer in range(layers):
            k, v, q = (_rand(100 + 10 * step + 3 * layer + i, B, n, 1, D, dtype=dtype) for i, n in enumerate((Hk, Hk, H)))
            cache.append(k.cuda(), v.cuda(), _i32(*start), layer=layer)
            model.append(k, v, start, None, layer)
            o, lse = flash_atten.sdpa_kv8(q.cuda(), cache, _i32(*start), layer=layer, return_lse=True)
            check_attention(o, lse, *model.attention(q, start, None, layer), (step, layer))
        model.check(cache, step)
        parent = [rng.randint(0, B - 1) for _ in range(B)]
        if step == 3:
            both("compact")
            model.check(cache, "compact")
    both("truncate", [0] * B)
    assert not cache.refs.any() and (cache.table == -1).all()


def test_serving_loop_eager_and_captured(gpu):
    """Drafts of three tokens of which some are rejected: truncate, reserve, append, attend. Replays of one graph, with
    eager work between them, give the eager run's bits; so do two graphs of one cache that share the allocator's pool."""
    B, H, Hk, D, capacity, page, dtype, M = 3, 8, 2, 128, 400, 64, F16, 3
    lengths = [60, 125, 1]
    rounds = 6
    accepted = [[3, 1, 2], [0, 3, 3], [2, 2, 1], [3, 3, 3], [1, 0, 2], [3, 2, 3]]
    data = [_rand(200 + i, B, rounds * M, n, D, dtype=dtype).cuda().transpose(1, 2) for i, n in enumerate((H, Hk, Hk))]
    kp, vp = (_rand(210 + i, B, Hk, 130, D, dtype=dtype).cuda() for i in range(2))

    def fresh():
        cache = kv8.Kv8Cache(B, Hk, capacity, D, dtype=dtype, pages=16, page_size=page)
        start = _i32(*lengths)
        zero = _i32(0, 0, 0)
        cache.reserve(zero, 130, count=start)
        cache.append(kp, vp, zero, count=start)
        return cache, start

    def step(cache, start, q, k, v):
        cache.truncate(start)
        missing = cache.reserve(start, M)
        cache.append(k, v, start)
        return flash_atten.sdpa_kv8(q, cache, start), missing

    cache, start = fresh()
    model = Model(cache)
    eager = []
    for r in range(rounds):
        q, k, v = (x[:, :, r * M:(r + 1) * M] for x in data)
        o, missing = step(cache, start, q, k, v)
        at = start.tolist()
        model.truncate(at)
        assert int(missing) == model.reserve(at, M) == 0
        model.append(k.cpu(), v.cpu(), at)
        model.check(cache, r)
        want = model.attention(q, at)
        assert ((o.double().cpu() - want[0]).abs() <= 1.01 * want[2]).all(), r
        eager.append(o.clone())
        start += _i32(*accepted[r])
    last = [t.clone() for t in (cache.table, cache.refs, cache.k_codes, cache.v_scales)]
    cache, start = fresh()
    inputs = [x[:, :, :M].clone() for x in data]
    keep = [t.clone() for t in (cache._data, cache.table, cache.refs, start)]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            out = step(cache, start, *inputs)[0]
        graphs.append((graph, out))
    for t, was in zip((cache._data, cache.table, cache.refs, start), keep):
        t.copy_(was)
    for r in range(rounds):
        for x, y in zip(inputs, data):
            x.copy_(y[:, :, r * M:(r + 1) * M])
        graph, out = graphs[r % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[r]), r
        assert torch.empty(1 << 20, device="cuda").fill_(1.0).sum().item() == 1 << 20
        start += _i32(*accepted[r])
    assert all(torch.equal(a, b) for a, b in zip(last, (cache.table, cache.refs, cache.k_codes, cache.v_scales)))


def test_far_pages(gpu):
    """Offsets past 32 bits: 40000 pages of 256 tokens are 5.2 GB; a sequence on the last pages and one on the first."""
    D, page, capacity = 256, 256, 700
    cache = kv8.Kv8Cache(2, 1, capacity, D, dtype=BF16, pages=40000, page_size=page, layers=1)
    cache.table[0] = _i32(39999, 3, 39998)
    cache.table[1] = _i32(0, 39997, 20000)
    for p in cache.table.flatten().tolist():
        cache.refs[p] = 1
    k, v = (_rand(300 + i, 2, 1, capacity, D, dtype=BF16) for i in range(2))
    held = cache.append(k.cuda(), v.cuda(), _i32(0, 0), return_values=True)
    used = [int(p) for p in cache.table.flatten()]
    codes = cache.k_codes[0, used].cpu()
    values = [x.double().cpu() for x in held]
    for M in (1, 60):
        q = _rand(302, 2, 4, M, D, dtype=BF16).cuda()
        o = flash_atten.sdpa_kv8(q, cache, _i32(capacity - M, 500))
        for b, end in ((0, capacity), (1, 500 + M)):
            s = q[b].double().cpu() @ values[0][b, 0, :end].T * D ** -0.5
            s = s.masked_fill(torch.arange(end)[None, None, :] > (end - M + torch.arange(M))[None, :, None], -math.inf)
            want = torch.softmax(s, -1) @ values[1][b, 0, :end]
            # P and the result are rounded once each: 2 half steps of the sum's largest terms
            bound = 2.2 * 2.0 ** -9 * (torch.softmax(s, -1) @ values[1][b, 0, :end].abs())
            assert ((o[b].double().cpu() - want).abs() <= bound + 2.0 ** -9 * want.abs()).all(), (M, b)
    cache.table[0, 1], cache.refs[3], cache.refs[25000] = 25000, 0, 1
    assert int(cache.compact()) == 6
    assert sorted(cache.table.flatten().tolist()) == list(range(6)) and int(cache.refs.sum()) == 6
    kept = [i for i, p in enumerate(used) if p != 3]
    now = cache.k_codes[0, cache.table.flatten().long()].cpu()
    assert torch.equal(now[kept], codes[kept])


def test_side_stream_alignment_and_layers(gpu):
    B, H, Hk, capacity, D = 2, 4, 2, 600, 64
    cache = _full(80, B, Hk, capacity, D, 64, F16, layers=3)
    q = _rand(81, B, H, 2, D, dtype=F16).cuda()
    want = [flash_atten.sdpa_kv8(q, cache, _i32(500, 10), layer=i) for i in range(3)]
    assert not torch.equal(want[0], want[1])
    odd = torch.empty(q.numel() + 1, dtype=F16, device="cuda")[1:].view_as(q).copy_(q)  # 2-byte aligned: copied first
    side = torch.cuda.Stream()
    start = _i32(500, 10)
    other = start.repeat_interleave(2)[::2]  # int32 with a stride: copied
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [flash_atten.sdpa_kv8(odd, cache, other, layer=i) for i in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    model = Model(cache)
    for i in range(3):
        o, lse = flash_atten.sdpa_kv8(q, cache, start, layer=i, return_lse=True)
        check_attention(o, lse, *model.attention(q, [500, 10], layer=i), i)
    # heads whose keys and values are shared by expansion (a stride of zero) are copied, not misread
    k = _rand(82, B, 1, 3, D, dtype=F16).cuda()
    cache.append(k.expand(B, Hk, 3, D), k.expand(B, Hk, 3, D), start, layer=1)
    model.append(k.expand(B, Hk, 3, D).cpu(), k.expand(B, Hk, 3, D).cpu(), [500, 10], None, 1)
    model.check(cache)


def test_refusals(gpu):
    cache = kv8.Kv8Cache(2, 2, 64, 64, dtype=F16, layers=2)
    k = torch.zeros(2, 2, 3, 64, dtype=F16, device="cuda")
    q, start = k, _i32(0, 0)
    for bad in (k.bfloat16(), k[:1], k[:, :1], k[..., :32], k.cpu(), k[0], None):
        with pytest.raises((ValueError, AttributeError)):
            cache.append(bad, bad, start)
    with pytest.raises(ValueError, match="v must be"):
        cache.append(k, k[:, :, :2], start)
    for bad in (start.long(), start[:1], start.cpu(), [0, 0], None):
        with pytest.raises(ValueError, match="start"):
            cache.append(k, k, bad)
        with pytest.raises(ValueError, match="start"):
            flash_atten.sdpa_kv8(q, cache, bad)
        with pytest.raises(ValueError, match="start"):
            cache.reserve(bad, 1)
        with pytest.raises(ValueError, match="parent"):
            cache.fork(bad)
        with pytest.raises(ValueError, match="length"):
            cache.truncate(bad)
    for rows in (-1, 1.5, None):
        with pytest.raises(ValueError, match="rows"):
            cache.reserve(start, rows)
    for layer in (2, -1, 0.5):
        with pytest.raises(ValueError, match="layer"):
            cache.append(k, k, start, layer=layer)
        with pytest.raises(ValueError, match="layer"):
            flash_atten.sdpa_kv8(q, cache, start, layer=layer)
    with pytest.raises(ValueError, match="count"):
        flash_atten.sdpa_kv8(q, cache, start, count=start.float())
    for bad in (q.bfloat16(), q.cpu()):
        with pytest.raises(ValueError, match="query is"):
            flash_atten.sdpa_kv8(bad, cache, start)
    for bad in (q[:1], q[..., :32], torch.zeros(2, 3, 1, 64, dtype=F16, device="cuda")):
        with pytest.raises(ValueError, match="does not fit"):
            flash_atten.sdpa_kv8(bad, cache, start)
    with pytest.raises(ValueError, match="sm_scale"):
        flash_atten.sdpa_kv8(q, cache, start, scale=0.0)
    assert flash_atten.sdpa_kv8(q[:, :, :0], cache, start).shape == (2, 2, 0, 64)
    assert not flash_atten.sdpa_kv8(q, cache, start).any()  # no page, no token
    with pytest.raises(hip_lib.FaUnsupportedError, match="fork"):
        kv8.Kv8Cache(kv8.MAX_FORK + 1, 1, 1, 64, dtype=F16, pages=1).fork(torch.zeros(kv8.MAX_FORK + 1, dtype=torch.int32, device="cuda"))
