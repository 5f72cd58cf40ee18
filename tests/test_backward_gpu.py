"""Attention's backward pass against the formula in 64 bits, against differences, and as a user calls it.

Tolerances. With u half a step of the type, the kernels round P and dS to the type once before the second
products, and the results once: |dq error| <= u |dq| + scale (u + e) (|dS| |K|), likewise dk and dv, where
e covers what is done in fp32: sums of n terms (n 2^-24 of the sum of magnitudes) and the exponent's argument
(an absolute error a in it is a relative error a in P). All of it is computed per element below."""
from __future__ import annotations

import math

import pytest
import torch

import flash_atten
import hip_lib

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
E32 = 2.0 ** -24


def _rand(seed, *shape, dtype, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).to(dtype).cuda()


def _inputs(seed, B, H, Hk, M, N, D, dtype, do_sigma=0.02):
    return (_rand(seed, B, H, M, D, dtype=dtype), _rand(seed + 1, B, Hk, N, D, dtype=dtype),
            _rand(seed + 2, B, Hk, N, D, dtype=dtype), _rand(seed + 3, B, H, M, D, dtype=dtype, sigma=do_sigma))


def _reference(do, q, k, v, o, lse, causal, scale, dlse=None):
    """(dq, dk, dv) of the formula in 64 bits, and a bound on each element's error."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * u  # half the step of subnormal results
    do, q, k, v, o, lse = (t.detach().double().cpu() for t in (do, q, k, v, o, lse))
    B, H, M, D = q.shape
    Hk, N = k.shape[1], k.shape[2]
    kk, vv = (t.repeat_interleave(H // Hk, dim=1) for t in (k, v))
    s = scale * (q @ kk.transpose(-1, -2))
    p = torch.exp(s - lse[..., None])
    p = torch.where(torch.isinf(lse)[..., None], 0.0, p)
    if causal:
        p = p * (torch.arange(N)[None, :] <= torch.arange(M)[:, None])
    delta = (do * o).sum(-1)
    if dlse is not None:
        delta = delta - dlse.double().cpu()
    dp = do @ vv.transpose(-1, -2) - delta[..., None]
    ds = p * dp
    dq = scale * (ds @ kk)
    dk = scale * (ds.transpose(-1, -2) @ q).view(B, Hk, H // Hk, N, D).sum(2)
    dv = (p.transpose(-1, -2) @ do).view(B, Hk, H // Hk, N, D).sum(2)
    # fp32 errors: of the exponent's argument, of dP - delta
    arg = E32 * (2 * D * scale * (q.abs() @ kk.abs().transpose(-1, -2)) + 3 * lse.abs().nan_to_num(posinf=0)[..., None] + 4)
    ddp = E32 * 2 * D * ((do.abs() @ vv.abs().transpose(-1, -2)) + (do * o).abs().sum(-1)[..., None] + delta.abs()[..., None])
    # fp16: what lies 2^-29 under the largest weight (or product) has an absolute error instead
    floor_p = 2.0 ** -40 if dtype == F16 else 0.0
    floor_s = floor_p * 4 * (do.norm(dim=-1).amax() * v.norm(dim=-1).amax() + delta.abs().amax()) if M and N else 0.0
    eds = ds.abs() * (u + arg) + p * ddp + floor_s
    ep = p * (u + arg) + floor_p
    n_q, n_k = E32 * (N + 8), E32 * (M * (H // Hk) + 8)
    bq = u * dq.abs() + scale * ((eds + n_q * ds.abs()) @ kk.abs()) + tiny
    bk = scale * ((eds + n_k * ds.abs()).transpose(-1, -2) @ q.abs()).view(B, Hk, H // Hk, N, D).sum(2) + u * dk.abs() + tiny
    bv = ((ep + n_k * p).transpose(-1, -2) @ do.abs()).view(B, Hk, H // Hk, N, D).sum(2) + u * dv.abs() + tiny
    return (dq, dk, dv), (bq, bk, bv)


def _check(grads, want, bound, what):
    for name, got, w, b in zip(("dq", "dk", "dv"), grads, want, bound):
        d = (got.double().cpu() - w).abs()
        assert got.shape == w.shape and torch.isfinite(got).all(), (what, name)
        over = d > b * 1.01
        assert not over.any(), (what, name, int(over.sum()), float((d / b.clamp(min=1e-300)).max()))


def _forward(q, k, v, causal, scale=None):
    return flash_atten.attention(q, k, v, causal=causal, sm_scale=scale, return_lse=True)


SIZES = [  # B, H, Hk, M, N, D
    (1, 1, 1, 1, 1, 64), (1, 2, 2, 33, 65, 64), (2, 4, 2, 127, 129, 64), (1, 3, 1, 128, 128, 64),
    (1, 1, 1, 1, 300, 128), (1, 2, 1, 300, 1, 128), (2, 4, 1, 95, 161, 128), (1, 6, 2, 257, 200, 128),
    (1, 1, 1, 16, 31, 256), (1, 4, 2, 130, 97, 256), (2, 2, 2, 64, 256, 256), (3, 1, 1, 17, 513, 128),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_against_the_formula(gpu, size, dtype, causal):
    B, H, Hk, M, N, D = size
    print(f"[backward] {size} {dtype} causal={causal}", flush=True)
    q, k, v, do = _inputs(100 + M + N, *size, dtype)
    o, lse = _forward(q, k, v, causal)
    grads = flash_atten.attention_backward(do, q, k, v, o, lse, causal=causal)
    _check(grads, *_reference(do, q, k, v, o, lse, causal, D ** -0.5), (size, dtype, causal))
    again = flash_atten.attention_backward(do, q, k, v, o, lse, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_strided_views_scale_and_lse_gradient(gpu, dtype):
    """[B, S, H, D] projections seen as [B, H, S, D], slices of a packed projection, a scale of its own, the
    log-sum-exp's gradient."""
    B, H, Hk, S, D, scale = 2, 6, 2, 150, 128, 0.17
    packed = _rand(7, B, S, H + 2 * Hk, D, dtype=dtype)
    q, k, v = (t.transpose(1, 2) for t in (packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]))
    do = _rand(8, B, S, H, D, dtype=dtype, sigma=0.02).transpose(1, 2)
    dlse = _rand(9, B, S, H, dtype=torch.float32, sigma=0.5).transpose(1, 2)
    o, lse = _forward(q, k, v, True, scale)
    grads = flash_atten.attention_backward(do, q, k, v, o, lse, causal=True, sm_scale=scale, dlse=dlse)
    _check(grads, *_reference(do, q, k, v, o, lse, True, scale, dlse), dtype)
    dense = flash_atten.attention_backward(*(t.contiguous() for t in (do, q, k, v, o, lse)), causal=True, sm_scale=scale,
                                           dlse=dlse.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(grads, dense))
    assert grads[0].stride() == torch.empty(B, S, H, D).transpose(1, 2).stride()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -14, 1.0, 300.0], ids=["small", "one", "large"])
def test_gradients_of_any_size(gpu, dtype, size):
    """fp16 keeps its bits for small and large gradients (dS is scaled into its range)."""
    B, H, Hk, M, N, D = 1, 2, 1, 200, 700, 64
    q, k, v, do = _inputs(31, B, H, Hk, M, N, D, dtype, do_sigma=size)
    o, lse = _forward(q, k, v, False)
    grads = flash_atten.attention_backward(do, q, k, v, o, lse)
    _check(grads, *_reference(do, q, k, v, o, lse, False, D ** -0.5), (dtype, size))


@pytest.mark.parametrize("causal", [False, True])
def test_against_differences(gpu, causal):
    """<gradient, direction> against central differences of sum(o w) + sum(lse z) in 64 bits."""
    B, H, Hk, M, N, D, scale = 1, 4, 2, 70, 90, 64, 64 ** -0.5
    q, k, v, w = _inputs(55, B, H, Hk, M, N, D, F16, do_sigma=1.0)
    z = _rand(60, B, H, M, dtype=torch.float32)
    o, lse = _forward(q, k, v, causal)
    grads = [g.double().cpu() for g in flash_atten.attention_backward(w, q, k, v, o, lse, causal=causal, dlse=z)]

    def loss(q, k, v):
        kk, vv = (t.repeat_interleave(H // Hk, dim=1) for t in (k, v))
        s = scale * (q @ kk.transpose(-1, -2))
        if causal:
            s = s.masked_fill(torch.arange(N)[None, :] > torch.arange(M)[:, None], -math.inf)
        return (torch.softmax(s, -1) @ vv * w.double().cpu()).sum() + (torch.logsumexp(s, -1) * z.double().cpu()).sum()

    x = [t.double().cpu() for t in (q, k, v)]
    h = 1e-5
    for n in range(3):
        d = torch.randn(x[n].shape, generator=torch.Generator().manual_seed(n), dtype=torch.float64)
        hi, lo = list(x), list(x)
        hi[n], lo[n] = x[n] + h * d, x[n] - h * d
        slope = (loss(*hi) - loss(*lo)) / (2 * h)
        # each element of the gradient is off by about the type's rounding (o's enters through delta): their
        # errors are independent, so the sum's is their root sum of squares; 8 of those
        spread = 8 * 2.0 ** -11 * 3 * float((grads[n] * d).norm()) + 1e-6 * abs(float(slope))
        assert abs(float((grads[n] * d).sum() - slope)) <= spread, (n, causal)


def test_autograd(gpu):
    B, H, Hk, M, N, D = 2, 4, 2, 100, 100, 64
    q, k, v, do = (t.requires_grad_(i < 3) for i, t in enumerate(_inputs(70, B, H, Hk, M, N, D, BF16)))
    o, lse = flash_atten.differentiable_attention(q, k, v, causal=True, return_lse=True)
    with torch.no_grad():
        assert torch.equal(o, flash_atten.attention(q, k, v, causal=True))
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    want = flash_atten.attention_backward(do, *(t.detach() for t in (q, k, v, o, lse)), causal=True)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), want))
    # a sum's gradient has zero strides; the log-sum-exp alone; both
    for loss, do_, dlse in ((o.sum(), torch.ones_like(o), None), (lse.sum(), torch.zeros_like(o), torch.ones_like(lse)),
                            (o.sum() + lse.sum(), torch.ones_like(o), torch.ones_like(lse))):
        got = torch.autograd.grad(loss, (q, k, v), retain_graph=True)
        want = flash_atten.attention_backward(do_, *(t.detach() for t in (q, k, v, o, lse)), causal=True, dlse=dlse)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a key/value head broadcast to all query heads gets the sum of its copies' gradients
    k1, v1 = k.detach()[:, :1].requires_grad_(), v.detach()[:, :1].requires_grad_()
    o1 = flash_atten.differentiable_attention(q, k1.expand(B, H, N, D), v1.expand(B, H, N, D), causal=True)
    got = torch.autograd.grad(o1, (k1, v1), do)
    o2, lse2 = flash_atten.attention(q.detach(), k1.detach(), v1.detach(), causal=True, return_lse=True)
    want, bound = _reference(do, q, k1, v1, o2, lse2, True, D ** -0.5)
    u = torch.finfo(BF16).eps / 2
    for g, w, b in zip(got, want[1:], bound[1:]):  # H gradients, each rounded, and their sum rounded H - 1 times
        slack = u * 2 * H * w.abs() + 2 * H * b
        assert ((g.double().cpu() - w).abs() <= slack + u * float(w.abs().max())).all()


def test_empty_problems(gpu):
    for dtype in (F16, BF16):
        q, k, v, do = _inputs(80, 1, 2, 2, 40, 0, 64, dtype)
        lse = torch.full((1, 2, 40), -math.inf, device="cuda")
        dq, dk, dv = flash_atten.attention_backward(do, q, k, v, torch.zeros_like(q), lse)
        assert not dq.any() and dk.numel() == dv.numel() == 0
        q, k, v, do = _inputs(81, 1, 2, 2, 0, 40, 64, dtype)
        dq, dk, dv = flash_atten.attention_backward(do, q, k, v, torch.zeros_like(q), torch.empty(1, 2, 0, device="cuda"))
        assert dq.numel() == 0 and not dk.any() and not dv.any()
        # rows that the forward calls empty have no gradients
        q, k, v, do = _inputs(82, 1, 2, 1, 70, 50, 128, dtype)
        o, lse = _forward(q, k, v, False)
        o[:, :, 5:40] = 0
        lse[:, :, 5:40] = -math.inf
        grads = flash_atten.attention_backward(do, q, k, v, o, lse)
        assert not grads[0][:, :, 5:40].any()
        _check(grads, *_reference(do, q, k, v, o, lse, False, 128 ** -0.5), dtype)


def test_not_finite_rows_stay_their_own(gpu):
    """An infinity in one row's gradient leaves the other rows' dq as they were."""
    for dtype in (F16, BF16):
        q, k, v, do = _inputs(85, 1, 1, 1, 96, 64, 64, dtype)
        o, lse = _forward(q, k, v, False)
        clean = flash_atten.attention_backward(do, q, k, v, o, lse)[0]
        do[0, 0, 50, 3] = math.inf
        dq = flash_atten.attention_backward(do, q, k, v, o, lse)[0]
        keep = torch.arange(96) != 50
        want, bound = _reference(do[:, :, keep], q[:, :, keep], k, v, o[:, :, keep], lse[:, :, keep], False, 0.125)
        assert ((dq[:, :, keep].double().cpu() - want[0]).abs() <= 1.01 * bound[0]).all()
        assert not torch.isfinite(dq[0, 0, 50]).any() and torch.isfinite(clean).all()


def test_graph_replays_and_streams(gpu):
    """Captured once, replayed with other contents between eager calls on the same leaves; and on a side stream."""
    B, H, Hk, M, N, D = 1, 4, 2, 200, 333, 128
    ins = _inputs(90, B, H, Hk, M, N, D, F16)
    q, k, v, do = ins
    o, lse = _forward(q, k, v, True)
    run = lambda: flash_atten.attention_backward(do, q, k, v, o, lse, causal=True)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for rep in range(3):
        for t, n in zip(ins, _inputs(91 + 10 * rep, B, H, Hk, M, N, D, F16)):
            t.copy_(n)
        fresh = _forward(q, k, v, True)
        o.copy_(fresh[0])
        lse.copy_(fresh[1])
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), rep
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_expanded_operands(gpu):
    """Heads, batches and rows with stride zero, sizes of one with any stride, a lse seen through strides."""
    B, H, M, N, D = 2, 3, 40, 50, 64
    q = _rand(110, 1, 1, M, D, dtype=F16).expand(B, H, M, D)
    k = _rand(111, 1, 1, N, D, dtype=F16).expand(B, 1, N, D)
    v = _rand(112, B, 1, 1, D, dtype=F16).expand(B, 1, N, D)
    do = _rand(113, 1, H, 1, D, dtype=F16).expand(B, H, M, D)
    o, lse = _forward(q, k, v, True)
    lse2 = torch.empty(M, H, B, device="cuda").permute(2, 1, 0).copy_(lse)
    grads = flash_atten.attention_backward(do, q, k, v, o, lse2, causal=True)
    _check(grads, *_reference(do, q, k, v, o, lse, True, D ** -0.5), "expanded")
    one = [t[:, :, :1] for t in (do, q, k, v, o)]
    grads = flash_atten.attention_backward(*one, lse[:, :, :1], causal=True)  # one row, one key: P as the lse says
    _check(grads, *_reference(*one, lse[:, :, :1], True, D ** -0.5), "one row")


def test_capture_of_the_differentiable_form_is_refused(gpu):
    q, k, v, _ = _inputs(120, 1, 2, 2, 32, 32, 64, F16)
    flash_atten.differentiable_attention(q, k, v)
    q.requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture attention"):
        with torch.cuda.graph(graph):
            flash_atten.differentiable_attention(q, k, v)
    with torch.no_grad():  # without gradients there is nothing to refuse
        want = flash_atten.differentiable_attention(q, k, v)
        held = torch.cuda.CUDAGraph()
        with torch.cuda.graph(held):
            o = flash_atten.differentiable_attention(q, k, v)
    for _ in range(2):
        held.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)


def test_long_causal_and_many_heads(gpu):
    """A longer call against 32-bit formulas per head: relative error of the whole gradient. P and dS are each
    rounded once, and the result: independent errors of at most u each, so under 3 u of the norm."""
    for dtype, (B, H, Hk, M, N, D, causal) in ((BF16, (1, 12, 2, 1500, 1500, 128, True)), (F16, (2, 4, 4, 1000, 2100, 64, False)),
                                               (BF16, (1, 4, 1, 900, 700, 256, True))):
        q, k, v, do = _inputs(95, B, H, Hk, M, N, D, dtype)
        o, lse = _forward(q, k, v, causal)
        grads = flash_atten.attention_backward(do, q, k, v, o, lse, causal=causal)
        (want, _) = _reference(do, q, k, v, o, lse, causal, D ** -0.5)
        u = torch.finfo(dtype).eps / 2
        for name, g, w in zip(("dq", "dk", "dv"), grads, want):
            assert float((g.double().cpu() - w).norm() / w.norm()) <= 3 * u, (name, dtype)


def test_refusals(gpu):
    q, k, v, do = _inputs(99, 1, 2, 2, 32, 48, 64, F16)
    o, lse = _forward(q, k, v, False)
    bwd = flash_atten.attention_backward
    with pytest.raises(ValueError, match="dtypes differ"):
        bwd(do.bfloat16(), q, k, v, o, lse)
    with pytest.raises(ValueError, match="shapes"):
        bwd(do[:, :, :16], q, k, v, o, lse)
    with pytest.raises(ValueError, match="shapes"):
        bwd(do, q, k, v[:, :, :40], o, lse)
    with pytest.raises(ValueError, match="lse must be"):
        bwd(do, q, k, v, o, lse.double())
    with pytest.raises(ValueError, match="dlse must be"):
        bwd(do, q, k, v, o, lse, dlse=lse[:, :1])
    with pytest.raises(ValueError, match="GPU tensor"):
        bwd(do, q, k.cpu(), v, o, lse)
    with pytest.raises(ValueError, match="lse is on"):
        bwd(do, q, k, v, o, lse.cpu())
    with pytest.raises(ValueError, match="sm_scale"):
        bwd(do, q, k, v, o, lse, sm_scale=-1.0)
    with pytest.raises(ValueError, match="4-D"):
        bwd(do, q[0], k, v, o, lse)
    with pytest.raises(ValueError, match="multiple of kv heads"):
        bwd(do[:, :1], q[:, :1], k, v, o[:, :1], lse[:, :1])
    with pytest.raises(hip_lib.FaUnsupportedError):
        bwd(*(t[..., :32] for t in (do, q, k, v, o)), lse)
    with pytest.raises(hip_lib.FaUnsupportedError):
        bwd(*(t.float() for t in (do, q, k, v, o)), lse)
    g = flash_atten.differentiable_attention(q.requires_grad_(), k, v)
    (first,) = torch.autograd.grad(g.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), q)
