"""Attention over the paged 8-bit cache where its running softmax, its joins and its searches come to their ends."""
from __future__ import annotations

import math

import pytest
import torch

import flash_atten
import kv8
from kv8_model import Model, check_attention
from test_kv8_gpu import BF16, F16, _deal, _full, _i32, _rand

pytestmark = pytest.mark.gpu


def _splits(monkeypatch, n):
    monkeypatch.setattr(kv8, "choose_splits", lambda *a: n)
    monkeypatch.setattr(flash_atten, "_plans", {})


def _scores(dtype, capacity, H, M, q_channels, k_channels, D=64):
    """A cache and queries whose scores (scale 1) are the sum of q_channels[i] * k_channels[i] (a number or one for each
    token), exact in fp32, and random values."""
    cache = kv8.Kv8Cache(1, H, capacity, D, dtype=dtype)
    _deal(cache, [capacity])
    k, v, q = torch.zeros(1, H, capacity, D), _rand(5, 1, H, capacity, D, dtype=dtype), torch.zeros(1, H, M, D)
    for i, (a, b) in enumerate(zip(q_channels, k_channels)):
        q[..., i], k[..., i] = a, b
    held = cache.append(k.to(dtype).cuda(), v.cuda(), _i32(0), return_values=True)[0].cpu()
    assert torch.equal(held.float(), k) and torch.equal(q.to(dtype).float(), q), "exact operands"
    return cache, q.to(dtype).cuda()


def _check_far(cache, q, start, dtype):
    """Scores are exact, so are their differences but for half a step of the difference; an exponent is one times
    fl(log2 e), at most 93 where it counts: 2^-24 x 3 x 93 x ln 2 < 2^-16 on a weight, twice that on a quotient of sums, and
    the sums of 400 terms take 2^-24 x 400 < 2^-15: 2^-14 in all. P and the result are rounded to the type once; a weight
    under the type's normal numbers by 2^-25 of a sum of 2^7 at least."""
    H, M = q.shape[1:3]
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(start), scale=1.0, return_lse=True)
    model = Model(cache)
    want, want_lse, _ = model.attention(q, [start], scale=1.0)
    keys, values, _ = model.line(0, 0)
    u = torch.finfo(dtype).eps / 2
    assert torch.isfinite(o).all()
    for h in range(H):
        s = q[0, h].double().cpu() @ keys[h].t()
        p = torch.softmax(s.masked_fill(torch.arange(s.shape[1])[None] > start + torch.arange(M)[:, None], -math.inf), -1)
        bound = (u + 2.0 ** -14) * (p @ values[h].abs()) + u * want[0, h].abs() + 2.0 ** -32 * values[h].abs().sum(0)
        assert ((o[0, h].double().cpu() - want[0, h]).abs() <= 1.01 * bound).all(), h
    assert ((lse.double().cpu() - want_lse).abs() <= 2e-5 + 2.0 ** -22 * want_lse.abs()).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_a_maximum_that_moves_by_the_spacing_of_the_scores(gpu, monkeypatch, dtype, sign):
    """Scores of 2^26 are 8 apart: the next larger one is further than the maximum may lag behind."""
    _splits(monkeypatch, 1)
    steps = torch.arange(400) // 100 * 8.0
    cache, q = _scores(dtype, 400, 2, 40, (sign * 2.0 ** 13, 1.0), (2.0 ** 13, steps))
    for start in (360, 200, 80):
        _check_far(cache, q, start, dtype)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("M", [1, 20, 40])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("power,spacing", [(12, 2.0), (13, 8.0)])
def test_parts_whose_maxima_are_far_from_zero(gpu, monkeypatch, power, spacing, dtype, M, splits):
    """Parts of a row whose maxima differ by steps of scores of 2^24 and 2^26: they are weighed by the difference of the
    scores, not by that of their rounded products with log2 e."""
    _splits(monkeypatch, splits)
    for sign in (1, -1):
        cache, q = _scores(dtype, 400, 2, M, (sign * 2.0 ** power, 1.0), (2.0 ** power, torch.arange(400) // 50 * spacing))
        for start in (400 - M, 300 - M, 70):
            _check_far(cache, q, start, dtype)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("dtype,near,far", [(F16, (36.0, 0.0), (36.0, 5.0)), (BF16, (30.0, 1.0), (36.0, 0.0))], ids=["f16", "bf16"])
def test_a_maximum_that_leaves_the_reach_of_whole_numbers(gpu, monkeypatch, dtype, near, far, M, splits):
    """Scores round 2^20 / log2 e = 726817.6, where the reference of a chunk's row stops being a whole number: the maximum
    moves by 5, past that border, when 330 tokens of e^-5 have been summed."""
    _splits(monkeypatch, splits)
    late = torch.arange(400) >= 330
    more = [torch.where(late, b, a) for a, b in zip(near, far)]
    cache, q = _scores(dtype, 400, 2, M, (708.0, 1.0, 1.0, 1.0), (1024.0, 1792.0, *more))
    for start in (400 - M, 331):
        _check_far(cache, q, start, dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("splits", [5, 97])
def test_shares_of_many_sequences(gpu, monkeypatch, D, splits):
    """More than 64 row blocks on the line that workgroups share: 70 sequences of unequal lengths, some without rows."""
    _splits(monkeypatch, splits)
    B, H, Hk, M, capacity = 70, 2, 2, 40, 300
    cache = _full(400 + D, B, Hk, capacity, D, 64, BF16)
    q = _rand(401, B, H, M, D, dtype=BF16).cuda()
    starts = [(b * 37) % (capacity - M) - (20 if b % 11 == 0 else 0) for b in range(B)]
    counts = [0 if b % 9 == 4 else M - b % 3 for b in range(B)]
    for causal in (True, False):
        o, lse = flash_atten.sdpa_kv8(q, cache, _i32(*starts), count=_i32(*counts), is_causal=causal, return_lse=True)
        check_attention(o, lse, *Model(cache).attention(q, starts, counts, causal=causal), (D, splits, causal))


@pytest.mark.parametrize("splits", [3, 250])
def test_shares_of_many_row_blocks(gpu, monkeypatch, splits):
    """The same with one sequence: 69 blocks of 128 rows, 8 heads that share 1200 keys."""
    _splits(monkeypatch, splits)
    cache = _full(410, 1, 1, 1200, 64, 64, F16)
    q = _rand(411, 1, 8, 1100, 64, dtype=F16).cuda()
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(100), return_lse=True)
    check_attention(o, lse, *Model(cache).attention(q, [100]), splits)


def test_a_layer_is_a_whole_number(gpu):
    """Also when a call of the same form has been made for the layer that the number is equal to."""
    cache = _full(420, 1, 2, 64, 64, 64, F16, layers=2)
    q, start = _rand(421, 1, 2, 3, 64, dtype=F16).cuda(), _i32(20)
    for layer in (1, 1.0, torch.tensor(1), "1"):
        calls = (lambda: cache.append(q, q, start, layer=layer), lambda: flash_atten.sdpa_kv8(q, cache, start, layer=layer))
        for call in calls:
            if type(layer) is int:
                call()
            else:
                with pytest.raises(ValueError, match="layer"):
                    call()


def test_a_kept_page_waits_for_its_last_copy(gpu):
    """Three holders of a page write and one page is free: the first gets its copy, the second is counted as missing, and the
    last, which keeps the page, cannot write it either until a later call has given the second one a page."""
    cache = kv8.Kv8Cache(4, 1, 64, 64, dtype=F16, pages=3, page_size=64)
    start, three = _i32(10, 10, 10, 0), _i32(1, 1, 1, 0)
    assert int(cache.reserve(_i32(0, 0, 0, 0), 64, count=_i32(10, 0, 0, 64))) == 0
    rows = _rand(430, 4, 1, 10, 64, dtype=F16).cuda()
    cache.append(rows, rows, _i32(0, 0, 0, 0), count=_i32(10, 0, 0, 10))
    cache.fork(_i32(0, 0, 0, 3))
    model = Model(cache)
    new = _rand(431, 4, 1, 1, 64, dtype=F16)

    def both():
        left = int(cache.reserve(start, 1, count=three))
        assert left == model.reserve([10, 10, 10, 0], 1, [1, 1, 1, 0])
        held = cache.append(new.cuda(), new.cuda(), start, count=three, return_values=True)[0]
        want = model.append(new, new, [10, 10, 10, 0], [1, 1, 1, 0])[0]
        model.check(cache)
        assert torch.equal(held.double().cpu(), want)
        return left, [bool(x.any()) for x in held]

    assert both() == (1, [True, False, False, False])
    cache.truncate(_i32(64, 64, 64, 0))
    model.truncate([64, 64, 64, 0])
    assert both() == (0, [True, True, True, False])


def test_results_take_no_part_in_autograd(gpu):
    """They are the bits of a call without gradients, and nothing of a graph."""
    cache = _full(440, 1, 2, 64, 64, 64, BF16)
    q, k = (_rand(441 + i, 1, 2, 3, 64, dtype=BF16).cuda() for i in range(2))
    held = cache.append(k, k, _i32(20), return_values=True)
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(20), return_lse=True)
    q.requires_grad_()
    k.requires_grad_()
    again = (*cache.append(k, k, _i32(20), return_values=True), *flash_atten.sdpa_kv8(q, cache, _i32(20), return_lse=True))
    for a, b in zip((*held, o, lse), again):
        assert torch.equal(a, b) and not b.requires_grad


def test_what_compact_leaves_can_be_moved(gpu):
    """Pages [0, used) of every layer, the table and the counts are the state: a smaller pool that they are copied into answers
    with the same bits."""
    cache = kv8.Kv8Cache(3, 2, 200, 64, dtype=F16, pages=40, page_size=32, layers=2)
    zero, n = _i32(0, 0, 0), _i32(200, 33, 150)
    _deal(cache, [200, 33, 150], 4)
    for layer in range(2):
        k, v = (_rand(450 + 2 * layer + i, 3, 2, 200, 64, dtype=F16).cuda() for i in range(2))
        cache.append(k, v, zero, count=n, layer=layer)
    cache.fork(_i32(0, 1, 0))
    cache.truncate(_i32(200, 0, 97))
    q, start = _rand(460, 3, 4, 2, 64, dtype=F16).cuda(), _i32(198, 0, 95)
    want = [flash_atten.sdpa_kv8(q, cache, start, layer=i) for i in range(2)]
    used = int(cache.compact())
    assert used == 7 == int((cache.refs > 0).sum())
    small = kv8.Kv8Cache(3, 2, 200, 64, dtype=F16, pages=used, page_size=32, layers=2)
    small.table.copy_(cache.table)
    small.refs.copy_(cache.refs[:used])
    for a, b in zip((small.k_codes, small.v_codes, small.k_scales, small.v_scales), (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)):
        a.copy_(b[:, :used])
    for other in (cache, small):
        assert all(torch.equal(a, flash_atten.sdpa_kv8(q, other, start, layer=i)) for i, a in enumerate(want))


@pytest.mark.parametrize("D,H,M", [(64, 2, 1), (128, 2, 1), (256, 2, 1), (128, 8, 5), (64, 8, 8), (256, 8, 8)])
def test_many_tiles_in_one_split(gpu, monkeypatch, D, H, M):
    """9000 tokens by one workgroup: its waves look up their 64 blocks more than once. Pages lie in no order, and some are
    missing, in the first look-up, in the second, and at the border between them."""
    _splits(monkeypatch, 1)
    capacity = 9000
    cache = _full(470 + D, 1, 2, capacity, D, 64, BF16)
    for token in (700, 8160, 8192, 8256, 8900):
        cache.table[0, token // 64] = -1
    q = _rand(471, 1, H, M, D, dtype=BF16).cuda()
    for start in (capacity - M, 8192 - M, 8192):
        o, lse = flash_atten.sdpa_kv8(q, cache, _i32(start), return_lse=True)
        check_attention(o, lse, *Model(cache).attention(q, [start]), (D, M, start))


@pytest.mark.parametrize("splits", [None, 1, 4])
@pytest.mark.parametrize("B,H,M", [(70, 4, 1), (130, 2, 6)])
def test_splits_of_many_sequences(gpu, monkeypatch, B, H, M, splits):
    """More than 64 sequences of unequal lengths, some empty, by single tokens and drafts."""
    if splits is not None:
        _splits(monkeypatch, splits)
    capacity = 1300
    cache = _full(480, B, 2, capacity, 64, 128, F16)
    q = _rand(481, B, H, M, 64, dtype=F16).cuda()
    starts = [(b * 331) % (capacity - M) for b in range(B)]
    counts = [0 if b % 13 == 5 else M for b in range(B)]
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(*starts), count=_i32(*counts), return_lse=True)
    check_attention(o, lse, *Model(cache).attention(q, starts, counts), (B, M, splits))


@pytest.mark.parametrize("D,M", [(128, 33), (256, 65)])
def test_whole_row_blocks_by_the_rule(gpu, D, M):
    """So many row blocks that each workgroup takes a whole one, the longest first, without `choose_splits` being told."""
    B, H, capacity = 128, 8 if M < 64 else 4, 100
    assert kv8.choose_splits(B, H, H, M, D, capacity) == 1
    cache = _full(490, B, H, capacity, D, 32, F16)
    q = _rand(491, B, H, M, D, dtype=F16).cuda()
    starts = [(b * 7) % (capacity - M + 1) for b in range(B)]
    counts = [M - b % 40 if b % 10 else 0 for b in range(B)]
    o, lse = flash_atten.sdpa_kv8(q, cache, _i32(*starts), count=_i32(*counts), return_lse=True)
    check_attention(o, lse, *Model(cache).attention(q, starts, counts), (D, M))


@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_and_missing_pages_in_parts_far_from_zero(gpu, monkeypatch, D, M):
    """Parts whose references are scores, next to one that holds a NaN key and one without a page: rows that see the key are
    NaN, the others' bits stay."""
    _splits(monkeypatch, 3)
    cache, q = _scores(F16, 700, 2, M, (2.0 ** 12, 1.0), (2.0 ** 12, torch.arange(700) // 100 * 2.0), D)
    start, nan = 700 - M, 700 - M // 2 - 1
    for missing in (None, 300 // 64):
        if missing is not None:
            cache.table[0, missing] = -1
        clean, clean_lse = flash_atten.sdpa_kv8(q, cache, _i32(start), scale=1.0, return_lse=True)
        want, want_lse, bound = Model(cache).attention(q, [start], scale=1.0)
        assert torch.isfinite(clean).all()
        assert ((clean.double().cpu() - want).abs() <= 1.01 * bound).all()
        page = cache.table[0, nan // 64].long()
        was = cache.k_codes[0, page, :, nan % 64, 3].clone()
        cache.k_codes[0, page, :, nan % 64, 3] = 127
        o, lse = flash_atten.sdpa_kv8(q, cache, _i32(start), scale=1.0, return_lse=True)
        cache.k_codes[0, page, :, nan % 64, 3] = was
        first = nan - start
        assert torch.equal(o[:, :, :first], clean[:, :, :first]) and torch.equal(lse[:, :, :first], clean_lse[:, :, :first])
        assert torch.isnan(o[:, :, first:]).all() and torch.isnan(lse[:, :, first:]).all()
