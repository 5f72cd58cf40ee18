"""The 4-bit key/value cache: what append writes against the format's definition in 64 bits (equal), attention
over it against the softmax in 64 bits, and the two together as a decode loop uses them.

Attention's tolerance: the cached values are exact, P is rounded to the type once (u, half a step) and the
result once, the rest is fp32: |error| <= u |o| + (u + e) (P |V|) per element, e covering sums of n terms
(n 2^-24) and the exponent's argument."""
from __future__ import annotations

import math

import pytest
import torch

import flash_atten
import kv4

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
E32 = 2.0 ** -24
CODES = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def _rand(seed, *shape, dtype, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).to(dtype)


def _encode(x):
    """Scale bytes and codes (one a byte) of x by the definition, in 64 bits."""
    f = x.double().unflatten(-1, (-1, 32))
    a = f.abs().amax(-1)
    bad = ~torch.isfinite(a)
    mantissa, exponent = torch.frexp(torch.where(bad, 1.0, a))
    low, high = (104, 140) if x.dtype == F16 else (2, 252)
    e = (exponent - 3 + (mantissa >= 0.875)).clamp(low - 127, high - 127)
    e = torch.where(a > 0, e, low - 127)
    y = (f / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]).nan_to_num(0, 0, 0)
    d = (y.abs()[..., None] - CODES).abs()
    code = d.argmin(-1)
    up = (code + 1).clamp(max=7)
    tie = d.gather(-1, up[..., None])[..., 0] == d.gather(-1, code[..., None])[..., 0]
    code = torch.where(tie & (code % 2 == 1), up, code)
    code = torch.where(bad[..., None], 0, code | torch.signbit(f).long() << 3)
    return torch.where(bad, 255, e + 127).to(torch.uint8), code.flatten(-2)


def _decode(scales, codes):
    """64-bit values of scale bytes and packed codes."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = torch.where(scales == 255, math.nan, torch.pow(2.0, scales.double() - 127))
    return CODES[c & 7] * (1 - 2 * (c >> 3)) * s.repeat_interleave(32, -1)


def _held(cache):
    return (_decode(cache.k_scales.cpu(), cache.k_codes.cpu()), _decode(cache.v_scales.cpu(), cache.v_codes.cpu()))


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _attention(q, keys, values, start, count, causal, scale, dtype):
    """o, lse in 64 bits and o's error bound."""
    q = q.double().cpu()
    B, H, M, D = q.shape
    Hk, N = keys.shape[1], keys.shape[2]
    u = torch.finfo(dtype).eps / 2
    o, lse, bound = torch.zeros(B, H, M, D, dtype=torch.float64), torch.full((B, H, M), -math.inf, dtype=torch.float64), None
    bound = torch.full_like(o, 1e-30)
    for b in range(B):
        n = max(0, min(int(count[b]), M))
        end = max(0, min(int(start[b]) + n, N)) if n else 0
        pos = int(start[b]) + torch.arange(n)
        for h in range(H):
            kk, vv = keys[b, h // (H // Hk), :end], values[b, h // (H // Hk), :end]
            s = scale * (q[b, h, :n] @ kk.t())
            seen = torch.arange(end)[None, :] <= pos[:, None] if causal else torch.ones(n, end, dtype=torch.bool)
            s = s.masked_fill(~seen, -math.inf)
            live = seen.any(1)
            if not live.any():
                continue
            p = torch.softmax(s[live], -1)
            i = torch.arange(n)[live]
            o[b, h, i] = p @ vv
            lse[b, h, i] = torch.logsumexp(s[live], -1)
            arg = E32 * (2 * D * scale * (q[b, h, i].abs() @ kk.abs().t()) + 2 * s[live].abs().nan_to_num(posinf=0) + 8)
            e = 2 * arg.amax(-1, keepdim=True) + E32 * (2 * end + 16)
            bound[b, h, i] = (u + e) * (p @ vv.abs()) + u * o[b, h, i].abs() + 2.0 ** -40 * vv.abs().sum(0) + \
                torch.finfo(dtype).tiny * u
    return o, lse, bound


def _check(got, lse, want, want_lse, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    d = (got - want).abs()
    assert (d <= 1.01 * bound).all(), (what, float((d / bound).max()))
    empty = torch.isinf(want_lse)
    lse = lse.double().cpu()
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all(), what
    # the exponent's argument as above, log and the rounding of lse itself
    assert ((lse - want_lse)[~empty].abs() <= 2e-5 + 2.0 ** -22 * want_lse[~empty].abs()).all(), what


def _filled(seed, B, Hk, capacity, D, dtype):
    """A cache whose every row is written, and tensors behind it."""
    cache = kv4.Kv4Cache(B, Hk, capacity, D, dtype=dtype)
    k, v = (_rand(seed + i, B, Hk, capacity, D, dtype=dtype).cuda() for i in range(2))
    cache.append(k, v, _i32(*[0] * B))
    return cache


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_writes_the_format(gpu, dtype, D):
    B, Hk, rows, capacity = 2, 3, 37, 75
    k = _rand(1, B, rows, Hk, D, dtype=torch.float32)
    v = _rand(2, B, rows, Hk, D, dtype=torch.float32) * torch.logspace(-9, 4, rows)[None, :, None, None]
    k[0, 0] = 0
    k[0, 1] = -0.0
    k[0, 2, 0, :8] = torch.tensor([7.0, 6.99, 5.0, 3.5, 2.5, 1.75, 1.25, 0.25])  # ties and the scale's border
    k[0, 2, 0, 8:32] = 0
    k, v = k.to(dtype), v.to(dtype)
    k[1, 3, 1, 5], k[1, 4, 0, 40], v[1, 5, 2, 0] = math.inf, math.nan, -math.inf
    k[1, 6, 0], v[1, 6, 0] = torch.finfo(dtype).max, torch.finfo(dtype).tiny / 4
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    cache = kv4.Kv4Cache(B, Hk, capacity, D, dtype=dtype)
    for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales):
        t.fill_(0xAB)
    start, count = (5, 38), (37, 20)
    kd, vd = (t.cuda() for t in (k, v))
    values = cache.append(kd, vd, _i32(*start), count=_i32(*count), return_values=True)
    for x, codes, scales, back in ((k, cache.k_codes, cache.k_scales, values[0]), (v, cache.v_codes, cache.v_scales, values[1])):
        e, c = _encode(x)
        packed = (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8)
        codes, scales, back = codes.cpu(), scales.cpu(), back.cpu()
        want = _decode(e, packed)
        for b in range(B):
            s, n = start[b], count[b]
            assert torch.equal(scales[b, :, s:s + n], e[b, :, :n]) and torch.equal(codes[b, :, s:s + n], packed[b, :, :n])
            assert (codes[b, :, :s] == 0xAB).all() and (codes[b, :, s + n:] == 0xAB).all()
            assert (scales[b, :, :s] == 0xAB).all() and (scales[b, :, s + n:] == 0xAB).all()
            assert torch.equal(back[b, :, :n].double().nan_to_num(1e9), want[b, :, :n].nan_to_num(1e9))
            assert not back[b, :, n:].any()
    # without values, from contiguous memory, the same bytes
    other = kv4.Kv4Cache(B, Hk, capacity, D, dtype=dtype)
    assert other.append(kd.contiguous(), vd.contiguous(), _i32(*start), count=_i32(*count)) is None
    for b in range(B):
        rows_b = slice(start[b], start[b] + count[b])
        assert torch.equal(other.k_codes[b, :, rows_b], cache.k_codes[b, :, rows_b])
        assert torch.equal(other.v_scales[b, :, rows_b], cache.v_scales[b, :, rows_b])


def test_append_keeps_inside_the_capacity(gpu):
    cache = kv4.Kv4Cache(3, 1, 40, 64, dtype=F16)
    whole = torch.empty(0)
    k, v = (_rand(i, 3, 1, 10, 64, dtype=F16).cuda() for i in (3, 4))
    values = cache.append(k, v, _i32(-4, 35, 40), return_values=True)
    held = _held(cache)
    for full, x, back in zip(held, (k, v), values):
        e, c = _encode(x.cpu())
        want = _decode(e, (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8))
        assert torch.equal(full[0, 0, :6], want[0, 0, 4:]) and not full[0, 0, 6:].any() and not back[0, 0, :4].any()
        assert torch.equal(full[1, 0, 35:], want[1, 0, :5]) and not full[1, 0, :35].any() and not back[1, 0, 5:].any()
        assert not full[2].any() and not back[2].any()
    before = [t.clone() for t in cache._buffers]
    cache.append(k, v, _i32(2 ** 31 - 3, -2 ** 31, 0), count=_i32(10, 10, 0))
    cache.append(k, v, _i32(0, 0, 0), count=_i32(-1, 0, -7))
    cache.append(k[:, :, :0], v[:, :, :0], _i32(0, 0, 0))
    assert all(torch.equal(a, b) for a, b in zip(before, cache._buffers))
    del whole


CASES = [  # B, H, Hk, M, capacity, D, starts, counts
    (1, 1, 1, 1, 1, 64, [0], None), (2, 4, 4, 1, 40, 64, [39, 0], None), (1, 8, 2, 1, 700, 128, [650], None),
    (3, 6, 2, 1, 300, 128, [-1, 31, 299], None), (1, 8, 1, 1, 1000, 256, [777], None), (2, 7, 1, 4, 333, 64, [100, 329], None),
    (1, 16, 2, 4, 600, 128, [500], None), (2, 4, 2, 5, 90, 256, [60, 3], [5, 2]), (1, 4, 2, 70, 500, 128, [400], None),
    (2, 2, 1, 129, 400, 64, [0, 200], [129, 64]), (2, 6, 2, 100, 260, 128, [-50, 160], [100, 0]),
    (1, 4, 4, 65, 130, 256, [50], None), (1, 32, 8, 1, 9000, 128, [8500], None), (2, 28, 4, 3, 2100, 128, [2000, 513], None),
    (1, 2, 2, 300, 2500, 64, [2100], None), (2, 3, 1, 8, 64, 128, [60, 2 ** 31 - 5], None), (1, 2, 1, 33, 3000, 256, [2900], [30]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])))
def test_attention_over_the_cache(gpu, case, dtype, causal):
    B, H, Hk, M, capacity, D, starts, counts = case
    print(f"[kv4] {case} {dtype} causal={causal}", flush=True)
    cache = _filled(10 + capacity, B, Hk, capacity, D, dtype)
    # what lies behind a sequence is not read: NaN there changes nothing
    for b in range(B):
        n = M if counts is None else max(0, counts[b])
        end = max(0, min(capacity, starts[b] + n)) if n else 0
        for t in (cache.k_scales, cache.v_scales):
            t[b, :, end:] = 255
    q = _rand(20, B, M, H, D, dtype=dtype).cuda().transpose(1, 2)
    count = None if counts is None else _i32(*counts)
    o, lse = flash_atten.sdpa_kv4(q, cache, _i32(*starts), count=count, is_causal=causal, return_lse=True)
    want = _attention(q, *_held(cache), starts, [M] * B if counts is None else counts, causal, D ** -0.5, dtype)
    _check(o, lse, *want, (case, dtype, causal))
    assert torch.equal(o, flash_atten.sdpa_kv4(q.contiguous(), cache, _i32(*starts), count=count, is_causal=causal))


@pytest.mark.parametrize("splits", [1, 2, 5, 33])
@pytest.mark.parametrize("M", [1, 6, 40])
def test_any_number_of_splits(gpu, monkeypatch, splits, M):
    B, H, Hk, capacity, D = 2, 8, 2, 3000, 128
    cache = _filled(40, B, Hk, capacity, D, BF16)
    q = _rand(41, B, H, M, D, dtype=BF16).cuda()
    starts = [capacity - M, 700]
    monkeypatch.setattr(kv4, "choose_splits", lambda *a: splits)
    monkeypatch.setattr(flash_atten, "_plans", {})
    o, lse = flash_atten.sdpa_kv4(q, cache, _i32(*starts), scale=0.2, return_lse=True)
    _check(o, lse, *_attention(q, *_held(cache), starts, [M] * B, True, 0.2, BF16), (splits, M))


def test_large_and_not_finite_scores(gpu):
    """Scores far apart (the running maximum moves), and a NaN block that only its own heads' rows see."""
    B, H, Hk, capacity, D = 1, 4, 2, 500, 64
    for dtype in (F16, BF16):
        k, v = (_rand(50 + i, B, Hk, capacity, D, dtype=torch.float32) for i in range(2))
        k = (k * torch.linspace(0.1, 12, capacity)[None, None, :, None]).to(dtype).cuda()
        cache = kv4.Kv4Cache(B, Hk, capacity, D, dtype=dtype)
        cache.append(k, v.to(dtype).cuda(), _i32(0))
        q = _rand(52, B, H, 1, D, dtype=dtype, sigma=4.0).cuda()
        o, lse = flash_atten.sdpa_kv4(q, cache, _i32(capacity - 1), return_lse=True)
        want = _attention(q, *_held(cache), [capacity - 1], [1], True, D ** -0.5, dtype)
        d = (o.double().cpu() - want[0]).abs()
        assert (d <= 1.01 * want[2]).all()
        cache.k_scales[0, 0, 100, 0] = 255
        bad, bad_lse = flash_atten.sdpa_kv4(q, cache, _i32(capacity - 1), return_lse=True)
        assert torch.isnan(bad[0, :2]).all() and torch.equal(bad[0, 2:], o[0, 2:])
        assert torch.isnan(bad_lse[0, :2]).all() and torch.equal(bad_lse[0, 2:], lse[0, 2:])


def test_decode_loop_eager_and_captured(gpu):
    """A prompt of unequal lengths enters the cache, then tokens one at a time: every step's output against the
    64-bit softmax over what the cache holds; the same steps replayed from one graph give the same bits."""
    B, H, Hk, capacity, D, dtype = 3, 8, 2, 200, 128, BF16
    prompt, steps = 50, 5
    lengths = [50, 17, 1]
    k, v = (_rand(60 + i, B, prompt + steps, Hk, D, dtype=dtype).cuda().transpose(1, 2) for i in range(2))
    q = _rand(62, B, prompt + steps, H, D, dtype=dtype).cuda().transpose(1, 2)
    cache = kv4.Kv4Cache(B, Hk, capacity, D, dtype=dtype)
    zero, count = _i32(0, 0, 0), _i32(*lengths)

    def prefill():
        cache.append(k[:, :, :prompt], v[:, :, :prompt], zero, count=count)
        return flash_atten.sdpa_kv4(q[:, :, :prompt], cache, zero, count=count, return_lse=True)

    o, lse = prefill()
    _check(o, lse, *_attention(q[:, :, :prompt], *_held(cache), [0] * B, lengths, True, D ** -0.5, dtype), "prefill")
    start = count.clone()
    eager = []
    for t in range(prompt, prompt + steps):
        cache.append(k[:, :, t:t + 1], v[:, :, t:t + 1], start)
        o, lse = flash_atten.sdpa_kv4(q[:, :, t:t + 1], cache, start, return_lse=True)
        _check(o, lse, *_attention(q[:, :, t:t + 1], *_held(cache), start.tolist(), [1] * B, True, D ** -0.5, dtype), t)
        start += 1
        eager.append(o.clone())
    tok = [x[:, :, :1].clone() for x in (q, k, v)]
    start = count.clone()
    graph = torch.cuda.CUDAGraph()
    prefill()
    with torch.cuda.graph(graph):
        cache.append(tok[1], tok[2], start)
        out = flash_atten.sdpa_kv4(tok[0], cache, start)
        start += 1
    start.copy_(count)
    for n, t in enumerate(range(prompt, prompt + steps)):
        for x, y in zip(tok, (q, k, v)):
            x.copy_(y[:, :, t:t + 1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[n]), n


def test_training_and_serving_together(gpu):
    """One layer trained a step through the differentiable attention, then served from the 4-bit cache: the
    served output is the full-precision one up to what the cache's format loses."""
    B, S, H, Hk, D, dtype = 1, 96, 4, 2, 64, BF16
    E = H * D
    x = _rand(70, B, S, E, dtype=dtype).cuda()
    w = [(_rand(71 + i, E, n * D, dtype=dtype, sigma=E ** -0.5)).cuda().requires_grad_() for i, n in enumerate((H, Hk, Hk))]

    def heads(n):
        return [(x @ m).view(B, S, -1, D).transpose(1, 2) for m in w][n]

    o = flash_atten.differentiable_attention(heads(0), heads(1), heads(2), causal=True)
    o.float().square().mean().backward()
    for m in w:
        assert m.grad is not None and torch.isfinite(m.grad).all() and m.grad.any()
    with torch.no_grad():
        for m in w:
            m -= 0.1 * m.grad
        q, k, v = (heads(i) for i in range(3))
        full = flash_atten.sdpa(q, k, v, is_causal=True)
        cache = kv4.Kv4Cache(B, Hk, S, D, dtype=dtype)
        kk, vv = cache.append(k, v, _i32(0), return_values=True)
        served = flash_atten.sdpa_kv4(q, cache, _i32(0))
        same = flash_atten.sdpa(q, kk, vv, is_causal=True)  # the forward on what the cache holds
    assert float((served - same).abs().max()) <= 4 * 2.0 ** -8 * float(vv.abs().max())
    # a code is off by at most an eighth of its value or half its smallest step: within a quarter of the norm
    assert float((served - full).float().norm() / full.float().norm()) <= 0.25


def test_far_rows(gpu):
    """Offsets past 32 bits: 70 million cached rows of one head are 4.5 GB of codes. The keys are zeros but for the
    last 64, whose scores of about 40 outweigh all others together by e^20: the output is the softmax over those."""
    capacity, D, n = 70_000_000, 128, 64
    cache = kv4.Kv4Cache(1, 1, capacity, D, dtype=BF16)
    q = torch.zeros(1, 2, 1, D, dtype=BF16, device="cuda")
    q[..., :32] = 2.0
    k = torch.zeros(1, 1, n, D, dtype=BF16, device="cuda")
    k[..., :32] = 7.0  # 2 * 6 * 32 / sqrt(128) = 33.9 as cached
    k[..., 32] = torch.linspace(-1, 1, n, device="cuda")
    v = _rand(90, 1, 1, n, D, dtype=BF16).cuda()
    start = _i32(capacity - n)
    cache.append(k, v, start)
    for M in (1, 40):
        qq = q.expand(1, 2, M, D)
        o = flash_atten.sdpa_kv4(qq, cache, _i32(capacity - M), is_causal=False, scale=0.1)
        kk, vv = (_decode(s[:, :, -n:].cpu(), c[:, :, -n:].cpu()) for s, c in ((cache.k_scales, cache.k_codes), (cache.v_scales, cache.v_codes)))
        score = 0.1 * (q.double().cpu()[0, :, 0] @ kk[0, 0].T)
        assert float(score.min()) - math.log(capacity) > 16  # so the rest weighs under e^-16 of the sum
        want = torch.softmax(score, -1) @ vv[0, 0]
        bound = (2 * 2.0 ** -9 + math.exp(-16)) * vv.abs().amax() + 2.0 ** -9 * want.abs()
        assert ((o[0].double().cpu() - want[:, None]).abs() <= bound[:, None]).all(), M


def test_side_stream_and_alignment(gpu):
    B, H, Hk, capacity, D = 2, 4, 2, 600, 64
    cache = _filled(80, B, Hk, capacity, D, F16)
    q = _rand(81, B, H, 2, D, dtype=F16).cuda()
    want = flash_atten.sdpa_kv4(q, cache, _i32(500, 10))
    odd = torch.empty(q.numel() + 1, dtype=F16, device="cuda")[1:].view_as(q).copy_(q)  # 2-byte aligned: copied first
    side = torch.cuda.Stream()
    start = _i32(500, 10)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = flash_atten.sdpa_kv4(odd, cache, start)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals(gpu):
    cache = kv4.Kv4Cache(2, 2, 64, 64, dtype=F16)
    k = torch.zeros(2, 2, 3, 64, dtype=F16, device="cuda")
    q, start = k, _i32(0, 0)
    for bad in (k.bfloat16(), k[:1], k[:, :1], k[..., :32], k.cpu(), k[0]):
        with pytest.raises(ValueError):
            cache.append(bad, bad, start)
    with pytest.raises(ValueError, match="v must be"):
        cache.append(k, k[:, :, :2], start)
    for bad in (start.long(), start[:1], start.cpu(), [0, 0], None):
        with pytest.raises(ValueError, match="start"):
            cache.append(k, k, bad)
        with pytest.raises(ValueError, match="start"):
            flash_atten.sdpa_kv4(q, cache, bad)
    with pytest.raises(ValueError, match="count"):
        flash_atten.sdpa_kv4(q, cache, start, count=start.float())
    for bad in (q.bfloat16(), q.cpu()):
        with pytest.raises(ValueError, match="query is"):
            flash_atten.sdpa_kv4(bad, cache, start)
    for bad in (q[:1], q[..., :32], torch.zeros(2, 3, 1, 64, dtype=F16, device="cuda")):
        with pytest.raises(ValueError, match="does not fit"):
            flash_atten.sdpa_kv4(bad, cache, start)
    with pytest.raises(ValueError, match="sm_scale"):
        flash_atten.sdpa_kv4(q, cache, start, scale=0.0)
    assert flash_atten.sdpa_kv4(q[:, :, :0], cache, start).shape == (2, 2, 0, 64)
