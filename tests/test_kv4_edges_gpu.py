"""The 4-bit cache at its edges: the largest unsplit passes.

Tolerances are those of the other tests of the cache (its `_attention`): the cached values are exact, P and the
result are rounded to the type once each."""
from __future__ import annotations

import math

import pytest
import torch

import flash_atten
import kv4
from test_kv4_gpu import BF16, _decode, _i32, _rand

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
