"""The paged 8-bit cache by its definition, in 64 bits on the CPU, token by token: what the tests compare with."""
from __future__ import annotations

import math

import torch

BLOCK = 32
RANGE = {torch.float16: (112, 134), torch.bfloat16: (10, 246)}
E32 = 2.0 ** -24


def _values():
    out = []
    for c in range(256):
        exponent, mantissa = c >> 3 & 15, c & 7
        v = math.ldexp(8 + mantissa, exponent - 10) if exponent else math.ldexp(mantissa, -9)
        out.append(math.nan if c & 127 == 127 else -v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


VALUES = _values()  # of the 256 codes


def power(e):
    """2^e of whole numbers, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def step_of(scales, dtype):
    """What scale bytes stand for: those past the type's largest are read as that."""
    return power(scales.int().clamp(max=RANGE[dtype][1]) - 127)


def decode(scales, codes, dtype):
    """Values of codes [..., tokens, D] with scale bytes [..., tokens / 32]."""
    return VALUES[codes.long()] * step_of(scales, dtype).repeat_interleave(BLOCK, -1)[..., None]


def encode_block(x, dtype):
    """Scale byte and codes of a block [32, D] of 64-bit values."""
    finite = torch.isfinite(x)
    top = float(torch.where(finite, x, 0.0).abs().max())
    low, high = RANGE[dtype]
    if top > 0:
        mantissa, exponent = math.frexp(top)  # top = mantissa 2^exponent, mantissa in [0.5, 1)
        e = min(max(exponent - 1 + (mantissa > 0.875) - 8 + 127, low), high)
    else:
        e = low
    y = torch.where(finite, x, 0.0) / math.ldexp(1.0, e - 127)
    positive = VALUES[:127]  # ascending
    a = y.abs().clamp(max=448.0)
    up = torch.searchsorted(positive, a.contiguous()).clamp(max=126)
    down = (up - 1).clamp(min=0)
    to_up, to_down = positive[up] - a, a - positive[down]
    code = torch.where((to_up < to_down) | ((to_up == to_down) & (up % 2 == 0)), up, down)
    code = torch.where(torch.signbit(x), code | 128, code)
    return e, torch.where(finite, code, 127).to(torch.uint8)


class Model:
    def __init__(self, cache):
        self.page, self.capacity, self.dtype = cache.page_size, cache.capacity, cache.dtype
        self.pull(cache)

    def pull(self, cache):
        self.table, self.refs = cache.table.cpu().clone(), cache.refs.cpu().clone()
        self.codes = [t.cpu().clone() for t in (cache.k_codes, cache.v_codes)]
        self.scales = [t.cpu().clone() for t in (cache.k_scales, cache.v_scales)]

    def check(self, cache, what=""):
        assert torch.equal(cache.table.cpu(), self.table), what
        assert torch.equal(cache.refs.cpu(), self.refs), what
        for mine, theirs in zip(self.codes + self.scales, (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)):
            assert torch.equal(mine, theirs.cpu()), what

    def tokens(self, start, count, rows):
        n = rows if count is None else max(0, min(int(count), rows))
        return max(0, int(start)), min(int(start) + n, self.capacity)

    def _page(self, b, column):
        p = int(self.table[b, column])
        return p if 0 <= p < len(self.refs) else -1

    def append(self, k, v, start, count=None, layer=0):
        """Returns what the rows stand for, in 64 bits."""
        out = [torch.zeros(x.shape, dtype=torch.float64) for x in (k, v)]
        B, H, rows, D = k.shape
        for b in range(B):
            low, high = self.tokens(start[b], None if count is None else count[b], rows)
            for block in range(low // BLOCK, -(-high // BLOCK)) if high > low else ():
                page = self._page(b, block * BLOCK // self.page)
                if page < 0 or int(self.refs[page]) != 1:
                    continue
                at = block * BLOCK
                r0, r1 = max(low, at) - at, min(high, at + BLOCK) - at
                sub = at % self.page // BLOCK
                for x, o, codes, scales in zip((k, v), out, self.codes, self.scales):
                    for h in range(H):
                        where = codes[layer, page, h, sub * BLOCK:(sub + 1) * BLOCK]
                        line = torch.zeros(BLOCK, D, dtype=torch.float64)
                        line[:r0] = (VALUES[where.long()] * step_of(scales[layer, page, h, sub], self.dtype))[:r0]
                        t = at + r0 - int(start[b])
                        line[r0:r1] = x[b, h, t:t + r1 - r0].double()
                        e, c = encode_block(line, self.dtype)
                        where.copy_(c)
                        scales[layer, page, h, sub] = e
                        o[b, h, t:t + r1 - r0] = (VALUES[c.long()] * math.ldexp(1.0, e - 127))[r0:r1]
        return out

    def reserve(self, start, rows, count=None):
        items = []
        for b in range(self.table.shape[0]):
            low, high = self.tokens(start[b], None if count is None else count[b], rows)
            if high > low:
                items += [(b, c) for c in range(low // self.page, -(-high // self.page))]
        by_page = {}
        for item in items:
            page = self._page(*item)
            if page >= 0 and int(self.refs[page]) > 1:
                by_page.setdefault(page, []).append(item)
        keeps = {v[-1] for page, v in by_page.items() if len(v) == int(self.refs[page])}
        copies = {item: page for page, v in by_page.items() for item in v if item not in keeps}
        wants = [item for item in items if item in copies or self._page(*item) < 0]
        free = [p for p, n in enumerate(self.refs.tolist()) if n == 0]
        for (b, c), page in zip(wants, free):
            if (b, c) in copies:
                self.refs[copies[b, c]] -= 1
                for t in self.codes + self.scales:
                    t[:, page] = t[:, copies[b, c]]
            self.table[b, c] = page
            self.refs[page] = 1
        return max(0, len(wants) - len(free))

    def _count(self, entries, by):
        for p in entries.flatten().tolist():
            if 0 <= p < len(self.refs):
                self.refs[p] += by

    def fork(self, parent):
        old = self.table.clone()
        self._count(old, -1)
        for b, p in enumerate(parent):
            self.table[b] = old[p] if 0 <= p < len(old) else -1
        self._count(self.table, 1)

    def truncate(self, length):
        for b, n in enumerate(length):
            c = max(0, -(-n // self.page))
            self._count(self.table[b, c:], -1)
            self.table[b, c:] = -1

    def compact(self):
        used = [p for p, n in enumerate(self.refs.tolist()) if n]
        live = len(used)
        to = dict(zip([p for p in used if p >= live], [p for p in range(live) if not int(self.refs[p])]))
        for a, b in to.items():
            for t in self.codes + self.scales:
                t[:, b] = t[:, a]
            self.refs[b], self.refs[a] = self.refs[a].clone(), 0
            self.table[self.table == a] = b
        return live

    def line(self, b, layer=0):
        """Keys, values [heads, capacity, D] and which of sequence b's tokens are there."""
        out = []
        pages = [self._page(b, c) for c in range(self.table.shape[1])]
        for codes, scales in zip(self.codes, self.scales):
            x = [decode(scales[layer, max(p, 0)], codes[layer, max(p, 0)], self.dtype) for p in pages]
            out.append(torch.cat(x, 1)[:, :self.capacity])
        there = torch.tensor([p >= 0 for p in pages]).repeat_interleave(self.page)[:self.capacity]
        return *out, there

    def attention(self, q, start, count=None, layer=0, causal=True, scale=None):
        """o, lse in 64 bits, and o's error bound: the cached values are exact, P is rounded to the type once (u, half a
        step) and the result once, the rest is fp32: |error| <= u |o| + (u + e) (P |V|) per element, e covering sums of n
        terms (n 2^-24) and the exponent's argument."""
        q = q.double().cpu()
        B, H, M, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        u = torch.finfo(self.dtype).eps / 2
        o, lse = torch.zeros(B, H, M, D, dtype=torch.float64), torch.full((B, H, M), -math.inf, dtype=torch.float64)
        bound = torch.full_like(o, 1e-30)
        for b in range(B):
            n = M if count is None else max(0, min(int(count[b]), M))
            end = max(0, min(int(start[b]) + n, self.capacity)) if n else 0
            keys, values, there = self.line(b, layer)
            pos = int(start[b]) + torch.arange(n)
            for h in range(H):
                g = h // (H // keys.shape[0])
                kk, vv = keys[g, :end], values[g, :end]
                seen = torch.arange(end)[None, :] <= pos[:, None] if causal else torch.ones(n, end, dtype=torch.bool)
                seen = seen & there[None, :end]
                live = seen.any(1)
                if not live.any():
                    continue
                i = torch.arange(n)[live]
                s = scale * (q[b, h, i] @ kk.t())
                s = s.masked_fill(~seen[live], -math.inf)
                p = torch.softmax(s, -1)
                vs = torch.where(there[:end, None], vv, 0.0)
                o[b, h, i] = p @ vs
                lse[b, h, i] = torch.logsumexp(s, -1)
                kk = torch.where(there[:end, None], kk, 0.0)
                arg = E32 * (2 * D * scale * (q[b, h, i].abs() @ kk.abs().t()) + 2 * s.abs().nan_to_num(posinf=0) + 8)
                e = 2 * arg.amax(-1, keepdim=True) + E32 * (2 * end + 16)
                bound[b, h, i] = (u + e) * (p @ vs.abs()) + u * o[b, h, i].abs() + 2.0 ** -40 * vs.abs().sum(0) + \
                    torch.finfo(self.dtype).tiny * u
        return o, lse, bound


def check_attention(got, lse, want, want_lse, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    d = (got - want).abs()
    assert (d <= 1.01 * bound).all(), (what, float((d / bound).max()))
    empty = torch.isinf(want_lse)
    lse = lse.double().cpu()
    assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all(), what
    # the exponent's argument as above, log and the rounding of lse itself
    assert ((lse - want_lse)[~empty].abs() <= 2e-5 + 2.0 ** -22 * want_lse[~empty].abs()).all(), what
