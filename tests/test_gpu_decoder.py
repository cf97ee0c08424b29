"""GPU tests of the decoder-layer operators against plain 64-bit formulas on the host.

Tolerances, elementwise, with h = eps / 2 the largest relative rounding of the output's type and
u = 2^-23 (one fp32 step; tensor-core sums may truncate):
  rotary     h |y| + 10 * 2^-24 m (|a| + |b|): angle off by pi 2^-24 (the top bits of the phase in fp32),
             sincospif by 2 * 2^-24, then four fp32 roundings of terms of at most m (|a| + |b|).
  linear_w4  h |y| + (80 + K / 512) u A, A = sum |x w| + |bias|: codes, products and scales are exact or one
             rounding; a block's sums chain at most 4 steps of 17 terms, a warp adds K / 512 blocks, then
             8 warps and the bias.
  attention  h |o| + (h + 2 d + (L / 16 + 32) u) A, A = sum p |v| with normalised p: each weight is rounded to
             the 16-bit type (h) and off by the error d = (D + 4) u max_j scale sum |q k_j| of its logit (as
             much again for the normaliser), L / 16 steps of the second product, and the joins.
"""
import math

import numpy as np
import pytest
import torch

from shorokoo_b200 import B200ArgumentError, B200NotSupportedError, decoder

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -23


def half(dtype):
    return torch.finfo(dtype).eps / 2


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float32) * scale).to(dtype)


def within(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= tol)   # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max())} x tolerance"


# ---- rotary ----------------------------------------------------------------------------------

def turned(x, positions, table, sign=1.0):
    """The formula in 64 bits, and the tolerance."""
    f = torch.tensor(table.frequencies, dtype=torch.float64)
    n = f.numel()
    ang = sign * positions.double()[:, None, None] * f
    c, s = torch.cos(ang) * table.magnitude, torch.sin(ang) * table.magnitude
    y = x.double().clone()
    sl = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if table.interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = y[..., sl[0]].clone(), y[..., sl[1]].clone()
    slack = torch.zeros_like(y)
    y[..., sl[0]], y[..., sl[1]] = a * c - b * s, a * s + b * c
    slack[..., sl[0]] = slack[..., sl[1]] = 10 * 2.0 ** -24 * abs(table.magnitude) * (a.abs() + b.abs())
    return y, slack + half(x.dtype) * (y.abs() + slack)


@pytest.mark.parametrize("tokens,heads,dim,r,dtype,inter,kw", [
    (1, 1, 64, 64, BF16, False, {}),
    (7, 32, 128, 128, FP16, False, dict(scaling="linear", factor=4.0)),
    (3, 5, 80, 80, BF16, True, dict(scaling="ntk", factor=4.0)),
    (2500, 12, 64, 32, FP32, True, {}),
    (2500, 3, 64, 32, FP32, False, dict(scaling="by_parts", factor=8.0, original_context=4096)),
    (33, 2, 96, 48, FP16, True, {}),
    (5, 3, 66, 30, BF16, False, {}),       # half of 30 pairs: no 16-byte pieces
    (5, 3, 66, 22, FP32, True, {}),
    (4, 2, 7, 6, FP16, False, {}),         # odd head
    (2, 96, 256, 256, BF16, False, {}),    # more pieces than a CTA has threads
])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(tokens, heads, dim, r, dtype, inter, kw, inverse):
    gen = torch.Generator().manual_seed(tokens * 131 + dim)
    x = normal(gen, (tokens, heads, dim), dtype)
    pos = torch.randint(-1000000, 1000000, (tokens,), generator=gen)
    pos[0] = 0
    table = decoder.RotaryTable(r, interleaved=inter, device="cuda", **kw)
    want, tol = turned(x, pos, table, -1.0 if inverse else 1.0)
    xg = x.cuda()
    got = decoder.rotary(xg, pos.cuda(), table, inverse=inverse)
    within(got, want, tol, "rotary")
    assert torch.equal(got[..., r:].cpu(), x[..., r:])
    assert torch.equal(xg.cpu(), x)
    assert torch.equal(decoder.rotary(xg, pos.int().cuda(), table, inverse=inverse), got)   # int32 positions
    decoder.rotary(xg, pos.cuda(), table, inverse=inverse, out=xg)                           # in place
    assert torch.equal(xg, got)


@pytest.mark.parametrize("shift", [0, 1])
def test_rotary_strides_and_alignment(shift):
    gen = torch.Generator().manual_seed(5)
    whole = normal(gen, (9, 3 * 4 * 64 + 8), BF16)
    table = decoder.RotaryTable(64, device="cuda")
    pos = torch.arange(9)
    part = whole[:, shift: shift + 256].view(9, 4, 64)          # a slice of a wider projection
    want, tol = turned(part, pos, table)
    g = whole.cuda()
    out = torch.full((4, 9, 64 + 8), 7.0, dtype=BF16, device="cuda")
    view = out[:, :, :64].transpose(0, 1)                         # heads outermost
    decoder.rotary(g[:, shift: shift + 256].view(9, 4, 64), pos.cuda(), table, out=view)
    within(view, want, tol, "strided")
    assert (out[:, :, 64:] == 7.0).all()


def test_rotary_inverse_is_the_gradient():
    """Against a difference quotient of f(x) = <rotary(x), g> along d. f is linear, so the quotient's only
    error is rounding: 2^-24 relative of sums of 20 x 64 products, over the step 1."""
    gen = torch.Generator().manual_seed(9)
    x, g, d = (normal(gen, (10, 2, 64), FP32).cuda() for _ in range(3))
    pos = torch.randint(0, 100000, (10,), generator=gen).cuda()
    table = decoder.RotaryTable(48, interleaved=True, scaling="by_parts", factor=4.0, original_context=2048, device="cuda")
    f = lambda z: (decoder.rotary(z, pos, table).double() * g.double()).sum()
    quotient = f(x + d) - f(x - d)
    grad = decoder.rotary(g, pos, table, inverse=True)
    direct = 2 * (grad.double() * d.double()).sum()
    scale = (x.abs() + d.abs()).double().sum() * float(g.abs().max()) * table.magnitude * 2
    assert abs(float(quotient - direct)) <= 16 * 2.0 ** -24 * float(scale)


def test_rotary_keeps_nan_and_inf_in_their_pair():
    x = torch.zeros(2, 2, 16, dtype=FP32)
    x[0, 0, 3], x[1, 1, 12] = math.inf, math.nan      # the latter behind the rotated part
    table = decoder.RotaryTable(8, device="cuda")
    y = decoder.rotary(x.cuda(), torch.tensor([1, 2]).cuda(), table).cpu()
    finite = torch.ones_like(x, dtype=torch.bool)
    finite[0, 0, 3] = finite[0, 0, 7] = finite[1, 1, 12] = False
    assert torch.equal(torch.isfinite(y), finite) and torch.isnan(y[1, 1, 12])


def test_rotary_refuses_on_the_gpu():
    x = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    t = decoder.RotaryTable(64, device="cuda")
    bad = [(x, pos[:1], t, {}), (x, pos.float(), t, {}), (x, pos.cpu(), t, {}), (x[0], pos, t, {}), (x, pos, None, {}),
           (x.transpose(1, 2), pos, t, {}), (x, pos, decoder.RotaryTable(64, device="cpu"), {}),
           (x, pos, decoder.RotaryTable(66, device="cuda"), {}), (x, pos, t, dict(out=x[:, :2])), (x, pos, t, dict(out=x.float()))]
    for a in bad:
        with pytest.raises(B200ArgumentError):
            decoder.rotary(a[0], a[1], a[2], **a[3])
    with pytest.raises(B200NotSupportedError):
        decoder.rotary(x.double(), pos, t)
    with pytest.raises(B200NotSupportedError):
        decoder.rotary(x.float().requires_grad_(), pos, t)
    assert decoder.rotary(x[:0], pos[:0], t).shape == (0, 4, 64)


# ---- paged cache -----------------------------------------------------------------------------

class Paged:
    """A cache with random pages in a random order, slots that no position has filled with NaN."""

    def __init__(self, new, context, kv, dim, page, dtype, seed=0, width=None, layout="pthd", poison=True):
        gen = torch.Generator().manual_seed(seed)
        self.new, self.context, self.kv, self.dim, self.page, self.dtype = new, context, kv, dim, page, dtype
        need = [-(-c // page) for c in context]
        self.width = max(need + [1]) + 2 if width is None else width
        self.pages = sum(need) + 5
        order = torch.randperm(self.pages, generator=gen).int()
        self.table = torch.full((len(new), self.width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, : min(n, self.width)] = order[at: at + min(n, self.width)]
            at += n
        shape = (self.pages, page, kv, dim)
        self.k, self.v = normal(gen, shape, dtype), normal(gen, shape, dtype)
        if poison:
            used = torch.zeros(self.pages, page, dtype=torch.bool)
            for b, c in enumerate(context):
                for j in range(min(c, self.width * page)):
                    used[self.table[b, j // page], j % page] = True
            self.k[~used], self.v[~used] = math.nan, math.nan
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
        self.layout = layout

    def gpu(self):
        if self.layout == "phtd":     # heads before tokens
            k, v = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (self.k, self.v))
        elif self.layout == "one":    # keys and values of a page in one buffer, padded heads
            both = torch.full((self.pages, 2, self.page, self.kv, self.dim + 8), math.nan, dtype=self.dtype)
            both[:, 0, :, :, : self.dim], both[:, 1, :, :, : self.dim] = self.k, self.v
            both = both.cuda()
            k, v = both[:, 0, :, :, : self.dim], both[:, 1, :, :, : self.dim]
        else:
            k, v = self.k.cuda(), self.v.cuda()
        return decoder.PagedCache(k, v, self.table.cuda(), torch.tensor(self.context, dtype=torch.int32).cuda())

    def gather(self, b):
        """Keys and values of a sequence's positions, and which of them are there."""
        c = self.context[b]
        j = torch.arange(c)
        ok = j < self.width * self.page
        page = torch.where(ok, self.table[b][(j // self.page).clamp(max=self.width - 1)].long(), -1)
        ok &= (page >= 0) & (page < self.pages)
        page = page.clamp(0, self.pages - 1)
        return self.k[page, j % self.page].double(), self.v[page, j % self.page].double(), ok


def attended(p, q, window=0, scale=None):
    """The formula in 64 bits, and the tolerance; rows that see nothing are zero."""
    heads, d = q.shape[1], q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    want, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    h = half(q.dtype)
    for b, n in enumerate(p.new):
        k, v, ok = p.gather(b)
        r0 = int(p.starts[b])
        for i in range(n):
            pos = p.context[b] - n + i
            j = torch.arange(p.context[b])
            see = ok & (j <= pos)
            if window:
                see &= j > pos - window
            if not see.any():
                continue
            for x in range(heads):
                kk, vv = k[see, x // (heads // p.kv)], v[see, x // (heads // p.kv)]
                s = (kk @ q[r0 + i, x].double()) * scale
                w = torch.softmax(s, 0)
                want[r0 + i, x] = w @ vv
                delta = (d + 4) * U * float((kk.abs() @ q[r0 + i, x].double().abs()).max()) * scale
                tol[r0 + i, x] = h * want[r0 + i, x].abs() + (h + 2 * delta + (len(s) / 16 + 32) * U) * (w @ vv.abs())
    return want, tol


CASES = [
    # new, context, heads, kv_heads, dim, page, dtype, window, layout
    ([1], [1], 1, 1, 64, 16, BF16, 0, "pthd"),
    ([1], [1500], 32, 8, 128, 16, BF16, 0, "pthd"),
    ([1, 1, 1], [1, 64, 65], 4, 2, 128, 16, FP16, 0, "pthd"),
    ([1] * 9, [0, 3, 700, 16, 17, 129, 64, 1, 300], 8, 1, 64, 16, BF16, 0, "phtd"),
    ([1, 1], [333, 90], 40, 2, 128, 64, FP16, 0, "one"),              # 20 rows of a key head: two row tiles
    ([1, 0, 1], [200, 50, 31], 6, 2, 80, 24, BF16, 0, "pthd"),        # pages that end inside a tile
    ([3, 5, 1], [100, 5, 700], 12, 4, 96, 8, FP16, 0, "pthd"),        # a few tokens, a whole prompt of 5
    ([2, 1], [257, 1000], 8, 8, 72, 1, BF16, 0, "pthd"),              # pages of one position
    ([1, 4], [600, 300], 8, 2, 64, 7, BF16, 33, "pthd"),              # windows
    ([1, 3], [600, 300], 5, 5, 128, 128, FP16, 1, "phtd"),
    ([20, 37], [20, 150], 4, 4, 64, 16, BF16, 0, "pthd"),
    ([130, 3, 65], [130, 700, 400], 8, 2, 128, 16, FP16, 0, "pthd"),
    ([70, 200], [300, 200], 6, 6, 64, 32, BF16, 50, "one"),
    ([129], [1000], 8, 4, 88, 24, BF16, 0, "phtd"),
    ([64, 1], [40, 5], 4, 2, 128, 16, BF16, 0, "pthd"),               # more new tokens than context: rows that see nothing
    ([257, 0, 1, 300], [513, 9, 0, 2000], 16, 2, 128, 64, BF16, 0, "pthd"),
    ([190, 140], [190, 640], 10, 2, 64, 16, FP16, 100, "pthd"),       # 5 heads per key head: rows of a token over two tiles
    ([300], [2500], 3, 1, 128, 16, FP16, 700, "pthd"),
    ([200], [333], 2, 2, 64, 8, BF16, 0, "phtd"),                     # the smallest pages that are copied whole
    ([150, 60], [700, 60], 4, 2, 128, 256, FP16, 0, "one"),           # pages longer than a tile
    ([100, 100], [100, 900], 8, 2, 104, 128, BF16, 333, "phtd"),
    ([90, 40], [95, 300], 16, 2, 128, 4, FP16, 0, "pthd"),            # pages too small for that: gathered
    ([1] * 600, [1 + i % 70 for i in range(600)], 2, 1, 64, 16, BF16, 0, "pthd"),     # more sequences than are counted at once
    ([3] * 520, [3 + i % 40 for i in range(520)], 16, 1, 64, 16, FP16, 0, "pthd"),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(case):
    new, context, heads, kv, dim, page, dtype, window, layout = case
    p = Paged(new, context, kv, dim, page, dtype, seed=len(context) + dim, layout=layout)
    q = normal(torch.Generator().manual_seed(3), (sum(new) + 3, heads, dim), dtype)
    want, tol = attended(p, q, window)
    cache = p.gpu()
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    got = decoder.paged_attention(cache, q.cuda(), p.starts.cuda(), window=window, out=out)
    assert got is out
    n = sum(new)
    within(out[:n], want[:n], tol[:n], "attention")
    assert (out[n:] == 5.0).all()      # rows behind the last sequence
    again = decoder.paged_attention(cache, q.cuda(), p.starts.cuda(), window=window)
    assert torch.equal(again[:n], out[:n])


@pytest.mark.parametrize("new,group", [(1, 4), (3, 1), (40, 4), (150, 2)])
def test_attention_leaves_out_what_is_not_there(new, group):
    """Table entries outside the pool, a context longer than its table, and pages of infinities."""
    p = Paged([new, new], [500, 400], 2, 64, 16, BF16, seed=4)
    p.table[0, 3], p.table[0, 7], p.table[1, 0] = -7, p.pages, 1 << 30
    p.context[1] = 900                       # the table holds (25 + 2 + ..) x 16 positions at most
    p.table[1, 25:] = -1
    p.k[~torch.isfinite(p.k)], p.v[~torch.isfinite(p.v)] = math.inf, -math.inf
    q = normal(torch.Generator().manual_seed(3), (2 * new, 2 * group, 64), BF16)
    want, tol = attended(p, q)
    got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda())
    within(got, want, tol, "missing pages")


@pytest.mark.parametrize("new,context,window", [(4, 40, 0), (4, 40, 3), (16, 16, 0), (100, 150, 0), (300, 700, 60)])
def test_attention_hides_nonfinite_later_positions(new, context, window):
    """NaN and infinities in the keys and values of a position reach the tokens that see it, no other."""
    p = Paged([new], [context], 1, 64, 16, BF16, seed=8)
    at = context - new // 2                  # a position among the new tokens' own
    early = max(0, context - new - 1)        # one that a window takes from the later tokens
    q = normal(torch.Generator().manual_seed(3), (new, 2, 64), BF16)
    page = lambda j: (p.table[0, j // 16].item(), j % 16)
    for what in ("v", "k"):
        x = getattr(p, what)
        keep = x.clone()
        x[page(at)][0, 5] = math.nan
        x[page(at)][0, 9] = math.inf
        x[page(early)][0, 11] = -math.inf
        if what == "v":
            clean, tol = attended(p, q, window)     # torch's sums keep unseen positions out altogether
            got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda(), window=window).double().cpu()
            ok = torch.isfinite(clean)
            assert torch.equal(torch.isfinite(got), ok)
            within(got[ok], clean[ok], tol[ok], "v")
            assert torch.equal(torch.isnan(got), torch.isnan(clean))
        else:
            x[page(early)] = keep[page(early)]
            got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda(), window=window).double().cpu()
            pos = torch.arange(context - new, context)
            sees = (at <= pos) & ((at > pos - window) if window else torch.tensor(True))
            setattr(p, what, keep)
            clean, tol = attended(p, q, window)
            within(got[~sees], clean[~sees], tol[~sees], "k")
            assert torch.isnan(got[sees]).all()
        setattr(p, what, keep)


def test_attention_scale_peaks_and_large_logits():
    """A scale that makes the softmax one-hot, and logits of thousands: the running maximum has to hold."""
    p = Paged([1, 200], [900, 600], 2, 128, 16, BF16, seed=6)
    q = normal(torch.Generator().manual_seed(3), (201, 8, 128), BF16, 8.0)
    for scale in (1e-6, 1.0, 30.0):
        want, tol = attended(p, q, 0, scale)
        got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda(), scale=scale)
        within(got, want, tol, f"scale {scale}")


def test_attention_rising_logits():
    """Keys whose logits rise along the context, so that the maximum grows at every step."""
    p = Paged([1, 140], [1200, 700], 1, 64, 16, FP16, seed=6)
    for b in range(2):
        for j in range(p.context[b]):
            p.k[p.table[b, j // 16], j % 16, 0] = 0.01 * j
    q = torch.full((141, 4, 64), 0.5, dtype=FP16) + normal(torch.Generator().manual_seed(3), (141, 4, 64), FP16, 0.1)
    want, tol = attended(p, q)
    within(decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda()), want, tol, "rising")


def test_attention_strided_queries():
    p = Paged([5, 90], [50, 300], 2, 64, 16, BF16, seed=2)
    qkv = normal(torch.Generator().manual_seed(3), (95, (8 + 2 + 2) * 64), BF16)
    q = qkv[:, : 8 * 64].view(95, 8, 64)
    want, tol = attended(p, q)
    g = qkv.cuda()
    out = torch.empty(8, 95, 64, dtype=BF16, device="cuda")
    decoder.paged_attention(p.gpu(), g[:, : 8 * 64].view(95, 8, 64), p.starts.cuda(), out=out.transpose(0, 1))
    within(out.transpose(0, 1), want, tol, "strided")


def test_attention_window_longer_than_the_context():
    p = Paged([3, 100], [50, 300], 2, 64, 16, BF16, seed=2)
    q = normal(torch.Generator().manual_seed(3), (103, 4, 64), BF16).cuda()
    want = decoder.paged_attention(p.gpu(), q, p.starts.cuda())
    for window in (300, 1 << 30, 1 << 31, (1 << 32) + 5):
        assert torch.equal(decoder.paged_attention(p.gpu(), q, p.starts.cuda(), window=window), want)


def test_attention_refuses_on_the_gpu():
    p = Paged([1], [20], 2, 64, 16, BF16)
    cache, q, s = p.gpu(), torch.zeros(1, 4, 64, dtype=BF16, device="cuda"), p.starts.cuda()
    for a, kw in [((q[..., :56], s), {}), ((q.half(), s), {}), ((q[:, :3], s), {}), ((q, s[:1]), {}), ((q, s.long()), {}),
                  ((q, s), dict(window=-1)), ((q, s), dict(scale=0.0)), ((q, s), dict(out=q[:, :2])), ((q.cpu(), s), {})]:
        with pytest.raises(B200ArgumentError):
            decoder.paged_attention(cache, *a, **kw)
    wide = torch.zeros(1, 4 * 64 + 1, dtype=BF16, device="cuda")[:, 1:].view(1, 4, 64)
    with pytest.raises(B200NotSupportedError):
        decoder.paged_attention(cache, wide, s)
    big = torch.zeros(2, 16, 2, 136, dtype=BF16, device="cuda")
    with pytest.raises(B200NotSupportedError):
        decoder.paged_attention(decoder.PagedCache(big, big, cache.page_table, cache.context_lengths),
                                torch.zeros(1, 4, 136, dtype=BF16, device="cuda"), s)
    for bad in [(cache.k_pages, cache.v_pages[:1]), (cache.k_pages, cache.v_pages.half()), (cache.k_pages[0], cache.v_pages[0])]:
        with pytest.raises(B200ArgumentError):
            decoder.PagedCache(*bad, cache.page_table, cache.context_lengths)
    with pytest.raises(B200ArgumentError):
        decoder.PagedCache(cache.k_pages, cache.v_pages, cache.page_table.long(), cache.context_lengths)
    with pytest.raises(B200ArgumentError):
        decoder.PagedCache(cache.k_pages, cache.v_pages, cache.page_table, cache.context_lengths.repeat(2))
    assert decoder.paged_attention(cache, q[:0], s).shape == (0, 4, 64)


@pytest.mark.parametrize("new,context,heads,kv,dim,r,page,dtype,inter,layout", [
    ([1, 1, 1], [1, 50, 33], 8, 2, 64, 64, 16, BF16, False, "pthd"),
    ([1] * 40, list(range(1, 41)), 32, 8, 128, 128, 16, FP16, False, "phtd"),
    ([5, 0, 70, 1], [5, 9, 100, 0], 4, 4, 80, 40, 24, BF16, True, "one"),
    ([3, 900], [2, 1000], 6, 1, 66, 30, 7, FP16, False, "pthd"),        # no 16-byte pieces; more tokens than context
    ([300], [300], 1, 1, 128, 64, 1, BF16, True, "pthd"),
    ([1500, 2500], [1500, 2600], 2, 1, 64, 64, 16, BF16, False, "pthd"),   # several tokens to a CTA
])
def test_append(new, context, heads, kv, dim, r, page, dtype, inter, layout):
    p = Paged(new, context, kv, dim, page, dtype, seed=dim, layout=layout, poison=False)
    if len(new) > 2:
        p.table[2, context[2] // (2 * page)] = p.pages        # a page that is not there
    gen = torch.Generator().manual_seed(11)
    n = sum(new)
    q, k, v = (normal(gen, (n + 2, x, dim), dtype) for x in (heads, kv, kv))
    table = decoder.RotaryTable(r, interleaved=inter, device="cuda")
    pos = torch.cat([torch.arange(c - m, c) for m, c in zip(new, context)] + [torch.zeros(2, dtype=torch.int64)])
    wq, tq = turned(q, pos, table)
    wk, tk = turned(k, pos, table)
    for turn in (True, False):
        cache = p.gpu()
        if turn:
            out = torch.full(q.shape, 3.0, dtype=dtype, device="cuda")
            got = decoder.paged_append(cache, k.cuda(), v.cuda(), p.starts.cuda(), q=q.cuda(), table=table, out=out)
            assert got is out
            within(got[:n], wq[:n], tq[:n], "q")
            assert (got[n:] == 3.0).all()
        else:
            assert decoder.paged_append(cache, k.cuda(), v.cuda(), p.starts.cuda()) is None
        kg, vg = cache.k_pages.cpu(), cache.v_pages.cpu()
        touched = torch.zeros(p.pages, page, dtype=torch.bool)
        row = 0
        for b, (m, c) in enumerate(zip(new, context)):
            for j in range(c - m, c):
                if 0 <= j < p.width * page:
                    pg = int(p.table[b, j // page])
                    if 0 <= pg < p.pages:
                        touched[pg, j % page] = True
                        assert torch.equal(vg[pg, j % page], v[row])
                        if turn:
                            within(kg[pg, j % page], wk[row], tk[row], "k")
                        else:
                            assert torch.equal(kg[pg, j % page], k[row])
                row += 1
        assert touched.any()
        assert torch.equal(kg[~touched], p.k[~touched]) and torch.equal(vg[~touched], p.v[~touched])


def test_append_in_place_and_keys_alone():
    p = Paged([2, 1], [9, 4], 2, 64, 4, BF16, poison=False)
    gen = torch.Generator().manual_seed(1)
    qkv = normal(gen, (3, 8 * 64), BF16).cuda()
    q, k, v = qkv[:, :256].view(3, 4, 64), qkv[:, 256:384].view(3, 2, 64), qkv[:, 384:].view(3, 2, 64)
    table = decoder.RotaryTable(64, device="cuda")
    one, two = p.gpu(), p.gpu()
    want = decoder.paged_append(one, k, v, p.starts.cuda(), q=q.clone(), table=table)
    assert decoder.paged_append(two, k, v, p.starts.cuda(), table=table) is None
    assert torch.equal(one.k_pages, two.k_pages) and torch.equal(one.v_pages, two.v_pages)
    got = decoder.paged_append(two, k, v, p.starts.cuda(), q=q, table=table, out=q)
    assert torch.equal(got, want) and torch.equal(one.k_pages, two.k_pages)
    with pytest.raises(B200ArgumentError):
        decoder.paged_append(one, k, v, p.starts.cuda(), q=q)
    with pytest.raises(B200ArgumentError):
        decoder.paged_append(one, k, v[:2], p.starts.cuda())


@pytest.mark.parametrize("starts", [[0, -5, 3], [2, 0, 1], [0, 100, 2], [3, 3, 3], [5, 1, 3]])
def test_index_arrays_out_of_order_stay_in_bounds(starts):
    """Row starts that no caller should pass: the kernels clamp them, touch nothing outside, and return."""
    p = Paged([2, 1], [40, 30], 2, 64, 16, BF16, poison=False)
    cache, s = p.gpu(), torch.tensor(starts, dtype=torch.int32).cuda()
    q = torch.ones(3, 4, 64, dtype=BF16, device="cuda")
    decoder.paged_append(cache, q[:, :2].contiguous(), q[:, :2].contiguous(), s, q=q, table=decoder.RotaryTable(64, device="cuda"))
    decoder.paged_attention(cache, q, s)
    torch.cuda.synchronize()


# ---- 4-bit linear ----------------------------------------------------------------------------

def linear(x, packed, scales, zeros, bias, k, group):
    """The formula in 64 bits, and the tolerance."""
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(1)[:, :k].double()
    spread = lambda t: t.double().repeat_interleave(group, 1)[:, :k]
    w = (codes - (8.0 if zeros is None else spread(zeros))) * spread(scales)
    y, a = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    if bias is not None:
        y, a = y + bias.double(), a + bias.double().abs()
    return y, half(x.dtype) * y.abs() + (80 + k / 512) * U * a


@pytest.mark.parametrize("rows,n,k,group,dtype,zeros,bias", [
    (1, 1, 1, 32, BF16, False, False),
    (1, 16, 64, 32, FP16, True, False),
    (1, 4096, 4096, 128, BF16, False, True),
    (2, 37, 130, 32, BF16, True, True),        # a last block of two inputs
    (3, 100, 255, 64, FP16, True, False),      # odd inputs: a half-used byte
    (8, 48, 96, 96, BF16, True, False),        # a group that ends inside a block
    (9, 500, 1000, 128, FP16, False, True),
    (16, 33, 2048, 256, BF16, True, True),
    (17, 129, 640, 64, FP16, True, False),
    (33, 50, 192, 32, BF16, False, False),
    (100, 80, 320, 64, BF16, True, True),
    (5, 1000, 9000, 32, FP16, True, False),
    (4, 64, 100, 4096, FP16, True, False),     # one group longer than the row
    (1, 100, 1000, 64, FP16, True, True),      # one row: each group size, ragged ends, odd inputs
    (1, 50, 2050, 32, BF16, True, False),
    (1, 33, 777, 256, FP16, True, False),
    (1, 20, 300, 96, BF16, True, True),
    (1, 70, 5000, 1024, BF16, True, False),
    (1, 2500, 8192, 32, FP16, True, False),
    (1, 19000, 128, 128, BF16, False, False),  # enough outputs for the smaller CTAs
    (7, 19100, 320, 64, FP16, True, False),    # two tiles of outputs per CTA, the last one alone
    (12, 9500, 256, 32, BF16, True, True),
])
def test_linear_w4(rows, n, k, group, dtype, zeros, bias):
    gen = torch.Generator().manual_seed(n + k)
    packed = torch.randint(0, 256, (n, (k + 1) // 2), generator=gen, dtype=torch.uint8)
    groups = -(-k // group)
    scales = ((torch.rand((n, groups), generator=gen) + 0.5) / math.sqrt(k)).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=gen, dtype=torch.uint8) if zeros else None
    b = normal(gen, (n,), dtype) if bias else None
    x = normal(gen, (rows, k), dtype)
    want, tol = linear(x, packed, scales, z, b, k, group)
    g = lambda t: None if t is None else t.cuda()
    w = decoder.W4Weights(packed.cuda(), scales.cuda(), g(z), in_features=k, group_size=group)
    within(decoder.linear_w4(x.cuda(), w, g(b)), want, tol, "linear_w4")
    # a slice of wider rows, into a slice of wider rows
    wide = torch.full((rows, k + 13), math.nan, dtype=dtype)
    wide[:, 3: 3 + k] = x
    out = torch.full((rows, n + 5), 9.0, dtype=dtype, device="cuda")
    decoder.linear_w4(wide.cuda()[:, 3: 3 + k], w, g(b), out=out[:, 2: 2 + n])
    within(out[:, 2: 2 + n], want, tol, "strided")
    assert (out[:, :2] == 9.0).all() and (out[:, 2 + n:] == 9.0).all()


def test_linear_w4_many_rows():
    """More row blocks than one launch's second grid dimension holds, the last one ragged."""
    rows, n, k = 65535 * 32 + 5, 16, 32
    packed = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8)
    scales = torch.ones(n, 1, dtype=BF16)
    w = decoder.W4Weights(packed.cuda(), scales.cuda(), in_features=k, group_size=32)
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    x[[0, -1, 65535 * 32], [3, 4, 5]] = 1.0
    y = decoder.linear_w4(x, w).cpu()
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(1).double() - 8
    assert torch.equal(y[0].double(), codes[:, 3]) and torch.equal(y[-1].double(), codes[:, 4])
    assert torch.equal(y[65535 * 32].double(), codes[:, 5]) and int((y != 0).any(1).sum()) <= 3


def test_linear_w4_row_stays_with_its_row():
    """A row of NaN and one of infinities leave the other rows as they are."""
    gen = torch.Generator().manual_seed(2)
    packed = torch.randint(0, 256, (40, 64), generator=gen, dtype=torch.uint8)
    scales = (torch.rand((40, 2), generator=gen) + 0.5).half()
    w = decoder.W4Weights(packed.cuda(), scales.cuda(), in_features=128, group_size=64)
    x = normal(gen, (6, 128), FP16)
    clean = decoder.linear_w4(x.cuda(), w)
    x[2], x[4, 7] = math.nan, math.inf
    y = decoder.linear_w4(x.cuda(), w)
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[2]).all() and not torch.isfinite(y[4]).any()


def test_w4_refuses_on_the_gpu():
    packed = torch.zeros(8, 32, dtype=torch.uint8, device="cuda")
    s = torch.ones(8, 1, dtype=BF16, device="cuda")
    ok = decoder.W4Weights(packed, s, in_features=64, group_size=64)
    for a, kw in [((packed, s), dict(in_features=66, group_size=64)), ((packed, s), dict(in_features=64, group_size=32)),
                  ((packed, s, s), dict(in_features=64, group_size=64)), ((packed.int(), s), dict(in_features=64, group_size=64)),
                  ((packed, s.cpu()), dict(in_features=64, group_size=64)), ((packed, s), dict(in_features=64, group_size=0))]:
        with pytest.raises(B200ArgumentError):
            decoder.W4Weights(*a, **kw)
    with pytest.raises(B200NotSupportedError):
        decoder.W4Weights(packed, s.float(), in_features=64, group_size=64)
    with pytest.raises(B200NotSupportedError):
        decoder.W4Weights(packed, torch.ones(8, 2, dtype=BF16, device="cuda"), in_features=64, group_size=40)
    x = torch.zeros(2, 64, dtype=BF16, device="cuda")
    for a, kw in [((x[:, :32], ok), {}), ((x.half(), ok), {}), ((x[0], ok), {}), ((x, ok, s), {}), ((x, ok), dict(out=x)),
                  ((x.t().contiguous().t(), ok), {}), ((x, ok, torch.zeros(7, dtype=BF16, device="cuda")), {})]:
        with pytest.raises(B200ArgumentError):
            decoder.linear_w4(*a, **kw)
    assert decoder.linear_w4(x[:0], ok).shape == (0, 8)


# ---- together --------------------------------------------------------------------------------

def test_a_layer_from_prompt_to_single_tokens():
    """One layer as it is used: 4-bit projections, rotary positions into the cache, attention, 4-bit
    output, for prompts in two chunks and then single tokens. Every stage is held to its own tolerance on
    the inputs it got, and the cache that grew step by step to the one of the whole text at once."""
    gen = torch.Generator().manual_seed(21)
    width, heads, kv, d, page, lengths = 256, 8, 2, 64, 16, [150, 41]
    pack = lambda n, k: (torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8),
                         ((torch.rand((n, k // 32), generator=gen) + 0.5) * 0.25 / math.sqrt(k)).to(BF16))
    pin, pout = pack((heads + 2 * kv) * d, width), pack(width, heads * d)
    win = decoder.W4Weights(pin[0].cuda(), pin[1].cuda(), in_features=width, group_size=32)
    wout = decoder.W4Weights(pout[0].cuda(), pout[1].cuda(), in_features=heads * d, group_size=32)
    table = decoder.RotaryTable(d, device="cuda")
    p = Paged([0, 0], lengths, kv, d, page, BF16, seed=1)
    whole = Paged([0, 0], lengths, kv, d, page, BF16, seed=1)
    text = [normal(gen, (n, width), BF16) for n in lengths]

    def step(book, cache, spans):
        x = torch.cat([t[a:b] for t, (a, b) in zip(text, spans)])
        new = [b - a for a, b in spans]
        book.new, book.context = new, [b for _, b in spans]
        book.starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32)
        cache.context_lengths.copy_(torch.tensor(book.context, dtype=torch.int32))
        starts, n = book.starts.cuda(), sum(new)
        qkv = decoder.linear_w4(x.cuda(), win)
        within(qkv, *linear(x, pin[0], pin[1], None, None, width, 32), "in")
        q, k, v = (t.view(n, -1, d) for t in qkv.split([heads * d, kv * d, kv * d], 1))
        qr = decoder.paged_append(cache, k, v, starts, q=q, table=table)
        pos = torch.cat([torch.arange(a, b) for a, b in spans])
        within(qr, *turned(q.cpu(), pos, table), "q")
        book.k, book.v = cache.k_pages.cpu(), cache.v_pages.cpu()
        o = decoder.paged_attention(cache, qr, starts)
        within(o, *attended(book, qr.cpu()), "attention")
        y = decoder.linear_w4(o.view(n, -1), wout)
        within(y, *linear(o.view(n, -1).cpu(), pout[0], pout[1], None, None, heads * d, 32), "out")
        return o

    cache, once = p.gpu(), whole.gpu()
    outs = [[], []]
    for spans in [((0, 100), (0, 30)), ((100, 146), (30, 37))] + [((a, a + 1), (c, c + 1)) for a, c in zip(range(146, 150), range(37, 41))]:
        o = step(p, cache, spans)
        n = spans[0][1] - spans[0][0]
        outs[0].append(o[:n])
        outs[1].append(o[n:])
    o = step(whole, once, ((0, 150), (0, 41)))
    used = torch.isfinite(once.k_pages)
    # qkv rounds once from sums whose order does not depend on the batch, so the caches agree exactly
    assert torch.equal(cache.k_pages[used], once.k_pages[used]) and torch.equal(cache.v_pages[used], once.v_pages[used])
    both = torch.cat(outs[0] + outs[1])
    # two results within h |o| + (h + small) A of the same value, |o| <= A <= max |v|
    assert (both.double() - o.double()).abs().max() <= 5 * half(BF16) * float(once.v_pages[used].abs().max())


def test_graph_replay_follows_the_lengths():
    """A captured step, replayed after the context lengths, tables and rows changed in place."""
    p = Paged([1, 1, 1], [40, 700, 5], 2, 64, 16, BF16, seed=3, width=60, poison=False)
    cache, table = p.gpu(), decoder.RotaryTable(64, device="cuda")
    gen = torch.Generator().manual_seed(4)
    q, k, v = (normal(gen, (3, x, 64), BF16).cuda() for x in (8, 2, 2))
    starts = p.starts.cuda()

    def step():
        qr = decoder.paged_append(cache, k, v, starts, q=q, table=table)
        return decoder.paged_attention(cache, qr, starts)

    step()
    torch.cuda.synchronize()
    graph, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(two):
        out2 = step()
    for lengths in ([41, 701, 6], [1, 16, 17], [0, 704, 3]):
        cache.context_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        q.copy_(normal(gen, (3, 8, 64), BF16))
        graph.replay()
        two.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want)


def test_attention_reports_no_wait_errors():
    decoder.check()
    p = Paged([200], [1500], 2, 64, 16, BF16)
    decoder.paged_attention(p.gpu(), torch.zeros(200, 4, 64, dtype=BF16, device="cuda"), p.starts.cuda())
    decoder.check()


def test_calls_on_two_streams():
    """Decode and chunk calls on two streams at once give what they give alone."""
    cases = [Paged([1] * 8, [900] * 8, 2, 128, 16, BF16, seed=1), Paged([200, 100], [1500, 700], 2, 64, 16, FP16, seed=2)]
    caches = [c.gpu() for c in cases]
    qs = [normal(torch.Generator().manual_seed(5), (sum(c.new), 8, c.dim), c.dtype).cuda() for c in cases]
    starts = [c.starts.cuda() for c in cases]
    alone = [decoder.paged_attention(c, q, s) for c, q, s in zip(caches, qs, starts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(decoder.paged_attention(caches[i], qs[i], starts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, alone[i]) for g in got[i])
