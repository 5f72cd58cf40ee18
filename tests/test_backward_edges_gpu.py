"""Attention's backward pass where rows' gradients differ in size by many powers of two: fp16 keeps the small rows'
bits beside the large ones'; rows without keys, which take no part; captures; numbers that are not finite.

Tolerances are those of the other tests of the backward (its `_reference`), but the absolute error of dS is taken
from the rows that share its scale: a row's own for dq, the rows from the key block's first on for causal dk."""
from __future__ import annotations

import math

import pytest
import torch

import flash_atten
from test_backward_gpu import BF16, E32, F16, _check, _forward, _inputs, _rand, _reference

pytestmark = pytest.mark.gpu


def _parts(do, q, k, v, o, lse, causal, scale):
    """64-bit dq, dk, and their bounds' parts: |dS| with its relative errors, and each row's |dO| |V| + |delta|."""
    do, q, k, v, o, lse = (t.double().cpu() for t in (do, q, k, v, o, lse))
    B, H, M, D = q.shape
    Hk, N = k.shape[1], k.shape[2]
    kk, vv = (t.repeat_interleave(H // Hk, dim=1) for t in (k, v))
    p = torch.exp(scale * (q @ kk.transpose(-1, -2)) - lse[..., None])
    if causal:
        p = p * (torch.arange(N)[None, :] <= torch.arange(M)[:, None])
    delta = (do * o).sum(-1)
    ds = p * (do @ vv.transpose(-1, -2) - delta[..., None])
    arg = E32 * (2 * D * scale * (q.abs() @ kk.abs().transpose(-1, -2)) + 3 * lse.abs()[..., None] + 4)
    ddp = E32 * 2 * D * ((do.abs() @ vv.abs().transpose(-1, -2)) + (do * o).abs().sum(-1)[..., None] + delta.abs()[..., None])
    size = do.norm(dim=-1) * v.norm(dim=-1).amax() + delta.abs()
    return q, k, kk, ds, ds.abs() * (2.0 ** -11 + arg) + p * ddp, size


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,H,Hk,N", [(64, 2, 1, 1024), (128, 2, 2, 700), (256, 1, 1, 600)])
def test_small_rows_beside_large_ones(gpu, causal, D, H, Hk, N):
    """Rows of dO of size 2^12 and of size 2^-8 in turn: dq of each is as exact as alone."""
    B, M = 1, N
    scale = D ** -0.5
    q, k, v = (_rand(300 + i, B, h, N, D, dtype=F16, sigma=0.5 if D == 256 else 1.0) for i, h in enumerate((H, Hk, Hk)))
    do = _rand(303, B, H, M, D, dtype=torch.float32)
    do[:, :, 0::2] *= 2.0 ** 12
    do[:, :, 1::2] *= 2.0 ** -8
    do = do.half()
    o, lse = _forward(q, k, v, causal)
    dq, _, _ = flash_atten.attention_backward(do, q, k, v, o, lse, causal=causal)
    _, _, kk, ds, eds, size = _parts(do, q, k, v, o, lse, causal, scale)
    want = scale * (ds @ kk)
    floor = 2.0 ** -40 * 4 * size[..., None]
    bound = 2.0 ** -11 * want.abs() + scale * ((eds + floor + E32 * (N + 8) * ds.abs()) @ kk.abs()) + 2.0 ** -25
    over = (dq.double().cpu() - want).abs() / bound
    assert float(over.max()) <= 1.01, float(over.max())
    # and the small rows as a whole: dS and the result are rounded once each, by at most 2^-11 and independently, so
    # under three of those of the norm; and half a step of subnormal results
    small = (dq.double().cpu() - want)[:, :, 1::2].norm() / want[:, :, 1::2].norm()
    steps = 2.0 ** -25 * want[:, :, 1::2].numel() ** 0.5 / float(want[:, :, 1::2].norm())
    assert float(small) <= 3 * 2.0 ** -11 + steps


@pytest.mark.parametrize("H,Hk,N", [(2, 2, 700), (4, 1, 900)])
def test_causal_keys_behind_large_rows(gpu, H, Hk, N):
    """The first 128 rows' gradients are 2^19 times the others': the keys from 128 on, which those rows do not see,
    have dk as if the others were alone."""
    B, D = 1, 64
    scale = D ** -0.5
    q, k, v = (_rand(310 + i, B, h, N, D, dtype=F16) for i, h in enumerate((H, Hk, Hk)))
    do = _rand(313, B, H, N, D, dtype=torch.float32)
    do[:, :, :128] *= 2.0 ** 11
    do[:, :, 128:] *= 2.0 ** -8
    do = do.half()
    o, lse = _forward(q, k, v, True)
    _, dk, _ = flash_atten.attention_backward(do, q, k, v, o, lse, causal=True)
    qd, _, _, ds, eds, size = _parts(do, q, k, v, o, lse, True, scale)
    fold = lambda t: t.view(B, Hk, H // Hk, *t.shape[2:]).sum(2)  # noqa: E731
    want = scale * fold(ds.transpose(-1, -2) @ qd)
    largest = torch.stack([size[:, :, j // 128 * 128:].amax() for j in range(N)])  # of the rows from the key's block on
    floor = 2.0 ** -40 * 4 * largest[None, None, None, :].expand_as(ds)
    n = E32 * (N * (H // Hk) + 8)
    bound = 2.0 ** -11 * want.abs() + scale * fold((eds + floor + n * ds.abs()).transpose(-1, -2) @ qd.abs()) + 2.0 ** -25
    d = (dk.double().cpu() - want).abs()
    assert float((d / bound).max()) <= 1.01, float((d / bound)[:, :, 128:].max())
    err = d[:, :, 128:].norm() / want[:, :, 128:].norm()
    assert float(err) <= 3 * 2.0 ** -11 + 2.0 ** -25 * want[:, :, 128:].numel() ** 0.5 / float(want[:, :, 128:].norm())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_without_keys_take_no_part(gpu, dtype, causal):
    """Rows whose lse is -inf, with NaN in their O, infinities in their dlse and a large dO: zero dq, and the others'
    gradients are what they are without those rows."""
    B, H, Hk, M, N, D = 1, 2, 1, 70, 50, 128
    q, k, v, do = _inputs(320, B, H, Hk, M, N, D, dtype)
    o, lse = _forward(q, k, v, causal)
    dlse = _rand(325, B, H, M, dtype=torch.float32, sigma=0.1)
    dead = torch.zeros(M, dtype=torch.bool)
    dead[5:40] = dead[M - 1] = True
    clean_do, clean_o, clean_dlse = do.clone(), o.clone(), dlse.clone()
    for t in (clean_do, clean_o, clean_dlse):
        t[:, :, dead.cuda()] = 0
    lse[:, :, dead.cuda()] = -math.inf
    do[:, :, dead.cuda()] = 1e4
    o[:, :, dead.cuda()] = math.nan
    dlse[:, :, dead.cuda()] = math.inf
    grads = flash_atten.attention_backward(do, q, k, v, o, lse, causal=causal, dlse=dlse)
    assert not grads[0][:, :, dead.cuda()].any()
    want, bound = _reference(clean_do, q, k, v, clean_o, lse, causal, D ** -0.5, clean_dlse)
    _check(grads, want, bound, (dtype, causal))


def test_capture_of_an_eager_result_s_backward_is_refused(gpu):
    """The forward ran eagerly on a side stream; its backward inside a capture on that stream raises before it
    launches anything, and works again afterwards."""
    q, k, v, do = _inputs(330, 1, 2, 2, 32, 32, 64, F16)
    q.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = flash_atten.differentiable_attention(q, k, v)
    torch.cuda.synchronize()
    print("[backward] captured", flush=True)
    with pytest.raises(RuntimeError, match="capture attention"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            torch.autograd.grad(o, q, do, retain_graph=True)
    torch.cuda.synchronize()
    print("[backward] eager", flush=True)
    with torch.cuda.stream(side):
        (dq,) = torch.autograd.grad(o, q, do)
    torch.cuda.synchronize()
    want = flash_atten.attention_backward(do, q.detach(), k, v, *_forward(q.detach(), k, v, False))[0]
    assert torch.equal(dq, want)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_causal_numbers_stay_in_their_tile(gpu, D, bad):
    """Causal: what is not finite in key 50 reaches no row before 32, and in row 50's gradient no key from 64 on, bit for
    bit (tiles of 32)."""
    B, H, M = 1, 2, 200
    q, k, v, do = _inputs(340 + D, B, H, H, M, M, D, BF16)
    o, lse = _forward(q, k, v, True)
    clean = flash_atten.attention_backward(do, q, k, v, o, lse, causal=True)
    for t in (k, v):
        held = t[:, :, 50].clone()
        t[:, :, 50] = bad
        dq = flash_atten.attention_backward(do, q, k, v, o, lse, causal=True)[0]
        assert torch.equal(dq[:, :, :32], clean[0][:, :, :32])
        assert not torch.isfinite(dq[:, :, 50:]).any()
        t[:, :, 50] = held
    do[:, :, 50] = bad
    _, dk, dv = flash_atten.attention_backward(do, q, k, v, o, lse, causal=True)
    assert torch.equal(dk[:, :, 64:], clean[1][:, :, 64:]) and torch.equal(dv[:, :, 64:], clean[2][:, :, 64:])
