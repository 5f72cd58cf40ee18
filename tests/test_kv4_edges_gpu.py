"""The 4-bit cache at its edges: the largest unsplit passes, value blocks that are no numbers in places that a row
does not see, more than 64 sequences to a call, every merge at every head dimension.

Tolerances are those of the other tests of the cache (its `_attention`): the cached values are exact, P and the
result are rounded to the type once each."""
from __future__ import annotations

import math

import pytest
import torch

import flash_atten
import kv4
from test_kv4_gpu import BF16, F16, _attention, _check, _decode, _filled, _held, _i32, _rand

pytestmark = pytest.mark.gpu


def _force_splits(monkeypatch, splits):
    monkeypatch.setattr(kv4, "choose_splits", lambda *a: splits)
    monkeypatch.setattr(flash_atten, "_plans", {})


def test_unsplit_pass_over_more_than_2_28_keys(gpu, monkeypatch):
    """One pass without splits covers every capacity that a cache may have. The keys are zeros but for the last 64,
    which lie behind key 2^28 and whose scores of 38.4 (2 * 6 * 32 * 0.1) outweigh the others together by
    e^(38.4 - ln(2^28)) > e^18: the output is the softmax over those 64, but for e^-16 of the largest value."""
    capacity, D, n = (1 << 28) + 96, 64, 64
    cache = kv4.Kv4Cache(1, 1, capacity, D, dtype=BF16)
    k = torch.zeros(1, 1, n, D, dtype=BF16, device="cuda")
    k[..., :32] = 7.0
    k[..., 32] = torch.linspace(-1, 1, n, device="cuda")
    v = _rand(90, 1, 1, n, D, dtype=BF16).cuda()
    cache.append(k, v, _i32(capacity - n))
    _force_splits(monkeypatch, 1)
    for M in (1, 20):  # 2 rows: shared by the waves; 40 rows: a chunk
        print(f"[kv4] {capacity} keys, M={M}", flush=True)
        q = torch.zeros(1, 2, M, D, dtype=BF16, device="cuda")
        q[..., :32] = 2.0
        o, lse = flash_atten.sdpa_kv4(q, cache, _i32(capacity - M), is_causal=False, scale=0.1, return_lse=True)
        kk, vv = (_decode(s[:, :, -n:].cpu(), c[:, :, -n:].cpu()) for s, c in ((cache.k_scales, cache.k_codes), (cache.v_scales, cache.v_codes)))
        score = 0.1 * (q.double().cpu()[0, :, 0] @ kk[0, 0].T)
        assert float(score.min()) - math.log(capacity) > 16
        want = torch.softmax(score, -1) @ vv[0, 0]
        bound = (2 * 2.0 ** -9 + math.exp(-16)) * vv.abs().amax() + 2.0 ** -9 * want.abs()
        assert ((o[0].double().cpu() - want[:, None]).abs() <= bound[:, None]).all(), M
        # the 64 weights' sum, and e^-16 of it
        top = torch.logsumexp(score, -1)
        assert ((lse[0].double().cpu() - top[:, None]).abs() <= 2e-5 + 2.0 ** -22 * top[:, None] + math.exp(-16)).all(), M


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("H,M", [(2, 5), (10, 5), (14, 40)], ids=["16rows", "32rows", "chunk"])
def test_values_that_are_no_numbers_reach_only_rows_that_see_them(gpu, monkeypatch, H, M, dtype, D, splits):
    """A NaN block of values (and of keys) at a drafted token: the rows before it, and the rows at or behind count,
    come out bit for bit as without it; the rows from it on are NaN in that block's channels, and in no other
    for the values. So does a block whose scale byte, one that append never writes, takes its values past the type."""
    B, Hk, capacity = 2, 2, 1200
    starts, counts = [1100, 517], [M, M - 1]
    _force_splits(monkeypatch, splits)
    cache = _filled(200 + D + M, B, Hk, capacity, D, dtype)
    q = _rand(201, B, H, M, D, dtype=dtype).cuda()
    start, count = _i32(*starts), _i32(*counts)
    call = lambda: flash_atten.sdpa_kv4(q, cache, start, count=count, return_lse=True)  # noqa: E731
    clean, clean_lse = call()
    assert torch.isfinite(clean).all()
    g = H // Hk
    for row in (M - 2, M // 2, 1):  # the draft's row whose token is bad
        for b in range(B):
            at = starts[b] + row
            for block in (0, D // 32 - 1):
                channels = slice(32 * block, 32 * block + 32)
                saved = cache.v_scales[b, 1, at, block].clone(), cache.v_codes[b, 1, at].clone()
                cache.v_scales[b, 1, at, block] = 255
                o, lse = call()
                assert torch.equal(o[:, :g], clean[:, :g]) and torch.equal(lse, clean_lse)
                assert torch.equal(o[1 - b], clean[1 - b])
                assert torch.equal(o[b, g:, :row], clean[b, g:, :row]), (row, b, block)
                seen = o[b, g:, row:counts[b]]
                assert torch.isnan(seen[..., channels]).all()
                others = torch.ones(D, dtype=torch.bool)
                others[channels] = False
                # the same sums, perhaps in another order: P |V| in fp32, then one rounding each
                d = (seen[..., others].double() - clean[b, g:, row:counts[b]][..., others].double()).abs()
                assert (d <= torch.finfo(dtype).eps * (clean[b, g:, row:counts[b]][..., others].double().abs() + 2.0 ** -10)).all()
                assert torch.equal(o[b, :, counts[b]:], clean[b, :, counts[b]:]) and not o[b, :, counts[b]:].any()
                # past the type's range: 4 * 2^23 or 4 * 2^127
                cache.v_scales[b, 1, at, block] = 150 if dtype == F16 else 254
                cache.v_codes[b, 1, at] = 0x66
                o, _ = call()
                assert torch.equal(o[b, g:, :row], clean[b, g:, :row]), (row, b, block)
                assert not o[b, :, counts[b]:].any()
                cache.v_scales[b, 1, at, block], cache.v_codes[b, 1, at] = saved
            saved = cache.k_scales[b, 1, at, 0].clone()
            cache.k_scales[b, 1, at, 0] = 255
            o, lse = call()
            assert torch.equal(o[b, g:, :row], clean[b, g:, :row]) and torch.equal(lse[b, g:, :row], clean_lse[b, g:, :row])
            assert torch.isnan(o[b, g:, row:counts[b]]).all() and torch.isnan(lse[b, g:, row:counts[b]]).all()
            assert not o[b, :, counts[b]:].any() and torch.isinf(lse[b, :, counts[b]:]).all()
            cache.k_scales[b, 1, at, 0] = saved
    # a NaN block that every live row sees: rows at or behind count are zeros all the same
    cache.v_scales[1, 0, 100, 0] = 255
    o, lse = call()
    assert torch.isnan(o[1, :g, :counts[1], :32]).all() and not o[1, :, counts[1]:].any()
    assert torch.equal(o[0], clean[0]) and torch.equal(o[1, g:], clean[1, g:]) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("B", [65, 130])
@pytest.mark.parametrize("M,H", [(1, 4), (12, 4)], ids=["token", "chunk"])
@pytest.mark.parametrize("splits", [2, 7, 40])
def test_more_than_64_sequences(gpu, monkeypatch, B, M, H, splits):
    """The split of a slot is looked up 64 sequences at a time: ragged lengths, with empty sequences first, last,
    and on both sides of a group's border."""
    capacity, D = 1500, 64
    starts = [(37 * b * b + 11) % (capacity - M) for b in range(B)]
    counts = [M] * B
    for b in (0, 63, 64, B - 1):
        counts[b] = 0
    counts[1] = max(1, M // 2)
    starts[2], starts[5] = -5, capacity - 1
    _force_splits(monkeypatch, splits)
    cache = _filled(300 + B, B, 1, capacity, D, F16)
    q = _rand(301, B, H, M, D, dtype=F16).cuda()
    print(f"[kv4] B={B} M={M} splits={splits}", flush=True)
    o, lse = flash_atten.sdpa_kv4(q, cache, _i32(*starts), count=_i32(*counts), return_lse=True)
    _check(o, lse, *_attention(q, *_held(cache), starts, counts, True, D ** -0.5, F16), (B, M, splits))


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("splits", [2, 12, 50])
@pytest.mark.parametrize("M", [1, 6, 40])
def test_every_merge(gpu, monkeypatch, D, dtype, splits, M):
    """One, four and sixteen waves to a row, at the head dimensions beside 128."""
    B, H, Hk, capacity = 2, 8, 2, 13000
    cache = _filled(400 + D, B, Hk, capacity, D, dtype)
    q = _rand(401, B, H, M, D, dtype=dtype).cuda()
    starts = [capacity - M, 4321]
    _force_splits(monkeypatch, splits)
    o, lse = flash_atten.sdpa_kv4(q, cache, _i32(*starts), scale=0.1, return_lse=True)
    _check(o, lse, *_attention(q, *_held(cache), starts, [M] * B, True, 0.1, dtype), (D, splits, M))
