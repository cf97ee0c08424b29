"""GPU tests of the operators between attention and the next token (residual norms, mixture-of-experts layers,
sampling) against plain 64-bit formulas on the host.

Tolerances, elementwise, with h = eps / 2 the largest relative rounding of the output's type, v = 2^-24 that of fp32 and
u = 2^-23 (tensor-core sums may truncate):
  residual_norm  errors carried through the formula to first order: a sum of squares or values chains at most 32 terms per
                 thread and 10 steps of shuffles (45 v with the division), rsqrtf 4 v, each product or sum v; then h |y|.
                 The first order is taken 1.25 times, for the products of errors.
  moe            gate and up off by d = (width / 16 + 8) u sum |w x|, hidden by 1.1 |up| d_gate + |act| d_up + 8 v |hidden| and its
                 rounding h |hidden| (at least half the type's smallest step), y by the shares' and the products' (inner / 16 + 16) u sum share |D hidden| on top, and
                 h |y|; |act'| is below 1.13.
  sample         none: the same token. Weights are off by 2^-41 of a row's largest and u times their sum falls that near to a border
                 with a chance of about 10^-8 a row.
"""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from shorokoo_b200 import B200ArgumentError, B200NotSupportedError, decoder

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
V, U = 2.0 ** -24, 2.0 ** -23


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(y, dy, dtype):
    """dy and the rounding of values within it of y to the type: half a step, which is eps / 2 of the value, and eps / 2 of the
    smallest normal number below that, where the steps stay as they are (fp16: 2^-25)."""
    return dy + half(dtype) * (y.abs() + dy) + half(dtype) * torch.finfo(dtype).smallest_normal


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float32) * scale).to(dtype)


def within(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= tol)   # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max())} x tolerance"


# ---- residual norms --------------------------------------------------------------------------

def normed(z, dz, w, b, kind, eps):
    """norm(z) w + b in 64 bits, and how far fp32 may be off where z is off by dz."""
    mean = z.mean(1, keepdim=True) if kind == "layer" else torch.zeros(z.shape[0], 1, dtype=torch.float64)
    dm = dz.mean(1, keepdim=True) + 45 * V * z.abs().mean(1, keepdim=True) if kind == "layer" else 0.0
    e = z - mean
    de = dz + dm + V * e.abs()
    q = (e * e).mean(1, keepdim=True)
    dq = 2 * (e.abs() * de).mean(1, keepdim=True) + (de * de).mean(1, keepdim=True) + 45 * V * q
    r = 1 / torch.sqrt(q + eps)
    dr = dq / (2 * (q + eps)) + 4 * V
    y = e * r * w
    dy = 1.25 * w.abs() * r * (de + e.abs() * (dr + 4 * V))
    if b is not None:
        y = y + b
        dy = dy + V * y.abs()
    return y, dy


def norm_reference(x, weight, *, bias=None, residual=None, post_weight=None, post_bias=None, gate=None, scale=1.0, kind="rms", eps=1e-6,
                   weight_offset=0.0):
    wide = lambda t: None if t is None else t.double()
    scale, eps, weight_offset = (float(np.float32(v)) for v in (scale, eps, weight_offset))
    t, dt = x.double(), torch.zeros(x.shape, dtype=torch.float64)
    if post_weight is not None:
        w = wide(post_weight) + weight_offset
        t, dt = normed(t, dt, w, wide(post_bias), kind, eps)
    g = torch.ones((), dtype=torch.float64) if gate is None else gate.double()
    add = scale * g * t
    h = add if residual is None else residual.double() + add
    dh = (scale * g).abs() * dt + 3 * V * add.abs() + V * h.abs()
    if weight is None:
        return None, None, h, dh
    y, dy = normed(h, dh, wide(weight) + weight_offset, wide(bias), kind, eps)
    return y, dy, h, dh


def check_norm(x, weight, out=None, residual_out=None, **kw):
    y, dy, h, dh = norm_reference(x, weight, **kw)
    gpu = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t
    got_y, got_h = decoder.residual_norm(gpu(x), gpu(weight), **{k: gpu(v) for k, v in kw.items()})
    if weight is None:
        assert got_y is None
    else:
        assert got_y.dtype is x.dtype
        within(got_y, y, rounded(y, dy, x.dtype), "y")
    within(got_h, h, rounded(h, dh, got_h.dtype), "h")
    return got_y, got_h


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 8), (2, 64), (400, 40), (1, 768), (613, 768), (9, 1000), (301, 1001), (1, 4096),
                                        (310, 4096), (2, 8200), (3, 11001), (300, 11001), (1, 16384), (301, 16392), (2, 32767),
                                        (298, 32768), (2, 32768)])
def test_residual_norm_sizes(rows, width, dtype):
    gen = torch.Generator().manual_seed(rows * 7 + width)
    x, r, g = (normal(gen, (rows, width), dtype) for _ in range(3))
    w, b, p = (normal(gen, (width,), dtype) for _ in range(3))
    check_norm(x, w, residual=r, eps=1e-5)
    check_norm(x, w, bias=b, residual=r, post_weight=p, gate=g, scale=0.3, kind="layer")


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [72, 75, 5000])
def test_residual_norm_forms(width, kind):
    gen = torch.Generator().manual_seed(width)
    x, r, g = (normal(gen, (6, width), BF16) for _ in range(3))
    w, b, p, c, v = (normal(gen, (width,), BF16) for _ in range(5))
    y, h = check_norm(x, w, kind=kind)
    assert torch.equal(h.cpu(), x)                                    # nothing was to be done to it
    check_norm(x, w, bias=b, kind=kind)
    check_norm(x, w, residual=r, gate=v, kind=kind)
    check_norm(x, w, gate=g, kind=kind)
    check_norm(x, w, scale=-2.0, residual=r, kind=kind)
    check_norm(x, None, post_weight=p, post_bias=c, residual=r, gate=g, scale=0.5, kind=kind)
    check_norm(x, None, residual=r, kind=kind)
    check_norm(x, w, post_weight=p, weight_offset=1.0, residual=r, kind=kind)
    f = lambda t: t.float() * 1.001
    check_norm(x, f(w), bias=f(b), post_weight=f(p), post_bias=f(c), residual=r, kind=kind)   # weights in 32 bits
    y, h = check_norm(x, w, residual=f(r), gate=g, kind=kind)         # the stream in 32 bits
    assert h.dtype is FP32


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,width,pitch", [(4800, 1024, 1024), (1300, 4104, 4112), (1300, 2050, 2050), (2500, 1033, 1033), (640, 11001, 11001),
                                              (620, 16392, 16392), (900, 5000, 5001), (610, 14001, 14003), (5000, 130, 131)])
def test_residual_norm_of_many_rows(rows, width, pitch, dtype):
    """Rows enough for every CTA to take several, from aligned ones to those that begin anywhere, and in place."""
    gen = torch.Generator().manual_seed(rows + width)
    x, r, g = (normal(gen, (rows, pitch), dtype)[:, pitch - width:].cuda() for _ in range(3))
    w, b, p = (normal(gen, (width,), dtype).cuda() for _ in range(3))
    some = sorted({0, 1, 5, rows // 2, rows - 2, rows - 1})
    kw = dict(bias=b, post_weight=p, scale=0.3, kind="layer")
    y, h = decoder.residual_norm(x, w, residual=r, gate=g, **kw)
    small = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    wy, dy, wh, dh = norm_reference(x[some].cpu(), w.cpu(), residual=r[some].cpu(), gate=g[some].cpu(), **small)
    within(y[some], wy, rounded(wy, dy, dtype), "y")
    within(h[some], wh, rounded(wh, dh, dtype), "h")
    for i in range(0, rows, 97):                      # a few rows at a time, the same results to rounding of sums
        part = slice(i, min(i + 3, rows))
        a, c = decoder.residual_norm(x[part], w, residual=r[part], gate=g[part], **kw)
        scale = float(w.abs().max()) * 8
        assert (a.float() - y[part].float()).abs().max() <= scale * torch.finfo(dtype).eps + 1e-4
        assert (c.float() - h[part].float()).abs().max() <= scale * torch.finfo(dtype).eps + 1e-4
    wide = normal(gen, (rows, width), FP32).cuda()
    y2, h2 = decoder.residual_norm(x, w, residual=wide, gate=b)
    wy, dy, wh, dh = norm_reference(x[some].cpu(), w.cpu(), residual=wide[some].cpu(), gate=b.cpu())
    within(y2[some], wy, rounded(wy, dy, dtype), "y, stream in 32 bits")
    within(h2[some], wh, rounded(wh, dh, FP32), "h, stream in 32 bits")
    some_of = lambda t: t[some].cpu()
    for more in (dict(residual=r, gate=g), dict(gate=g), dict(residual=r), dict(residual=wide, gate=g, scale=-0.5)):   # h alone
        none, h3 = decoder.residual_norm(x, None, **more)
        _, _, wh, dh = norm_reference(some_of(x), None, **{k: some_of(v) if isinstance(v, torch.Tensor) else v for k, v in more.items()})
        assert none is None
        within(h3[some], wh, rounded(wh, dh, h3.dtype), "h alone")
    y4, h4 = decoder.residual_norm(x, w.float(), bias=b.float(), weight_offset=1.0)
    wy, dy, _, _ = norm_reference(some_of(x), w.float().cpu(), bias=b.float().cpu(), weight_offset=1.0)
    within(y4[some], wy, rounded(wy, dy, dtype), "weights in 32 bits")
    decoder.residual_norm(x, w, residual=r, gate=g, out=x, residual_out=r, **kw)
    assert torch.equal(x, y) and torch.equal(r, h)


def test_residual_norm_of_a_loud_mean():
    """The variance is taken of differences from the mean: values 1000 off zero keep theirs."""
    gen = torch.Generator().manual_seed(3)
    x = 1000 + torch.randn((4, 4096), generator=gen)
    check_norm(x, torch.ones(4096), kind="layer", eps=1e-5)
    check_norm((x * 10).half(), torch.ones(4096).half(), kind="layer", residual=normal(gen, (4, 4096), FP32), eps=1e-5)


@pytest.mark.parametrize("shift", [0, 1, 8])
@pytest.mark.parametrize("width", [64, 136, 1024])
def test_residual_norm_strides_places_and_streams(width, shift):
    gen = torch.Generator().manual_seed(width + shift)
    wide = normal(gen, (5, 3 * width + 16), FP16)
    x, r, w = wide[:, shift: shift + width], wide[:, width + 2 * shift: 2 * width + 2 * shift], normal(gen, (width,), FP16)
    want_y, dy, want_h, dh = norm_reference(x, w, residual=r)
    buf = torch.full((5, 2 * width + 24), 7.0, dtype=FP16, device="cuda")
    y, h = buf[:, shift: shift + width], buf[:, width + 8 + shift: 2 * width + 8 + shift]
    g, gw = wide.cuda(), w.cuda()
    gx, gr = g[:, shift: shift + width], g[:, width + 2 * shift: 2 * width + 2 * shift]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = decoder.residual_norm(gx, gw, residual=gr, out=y, residual_out=h)
    side.synchronize()
    assert got[0] is y and got[1] is h
    within(y, want_y, rounded(want_y, dy, FP16), "y")
    within(h, want_h, rounded(want_h, dh, FP16), "h")
    used = torch.zeros(buf.shape, dtype=torch.bool)
    used[:, shift: shift + width] = used[:, width + 8 + shift: 2 * width + 8 + shift] = True
    assert (buf.cpu()[~used] == 7.0).all()
    first = y.clone(), h.clone()
    a, b = gx.clone(), gr.clone()
    decoder.residual_norm(a, gw, residual=b, out=a, residual_out=b)       # in place
    assert torch.equal(a, first[0]) and torch.equal(b, first[1])
    b = gr.clone()
    one = decoder.residual_norm(gx, gw, residual=b[:1].expand(5, width))   # a row for all
    within(one[1], (x.double() + r[:1].double()), half(FP16) * 2 * (x.double().abs() + r[:1].double().abs()), "shared row")


def test_residual_norm_keeps_rows_apart():
    gen = torch.Generator().manual_seed(8)
    x, w = normal(gen, (9, 264), BF16), normal(gen, (264,), BF16)
    clean = decoder.residual_norm(x.cuda(), w.cuda())[0].cpu()
    x[2, 5], x[4, 0], x[6] = math.nan, math.inf, 0.0
    y = decoder.residual_norm(x.cuda(), w.cuda())[0].cpu()
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[2]).all() and torch.isnan(y[4, 0]) and (y[4, 1:] == 0).all() and (y[6] == 0).all()
    assert decoder.residual_norm(x[:0].cuda(), w.cuda())[0].shape == (0, 264)


def test_residual_norm_refuses():
    x, w = torch.zeros(2, 64, dtype=BF16, device="cuda"), torch.ones(64, dtype=BF16, device="cuda")
    f = decoder.residual_norm
    bad = [lambda: f(x, w[:32]), lambda: f(x, w.half()), lambda: f(x, w.cpu()), lambda: f(x[0], w), lambda: f(x.t(), w[:2]),
           lambda: f(x, w, residual=x[:1]), lambda: f(x, w, residual=x.half()), lambda: f(x, w, gate=x.float()), lambda: f(x, w, gate=w[:3]),
           lambda: f(x, w, kind="other"), lambda: f(x, w, eps=-1.0), lambda: f(x, w, scale=math.inf), lambda: f(x, None),
           lambda: f(x, None, residual=x, bias=w), lambda: f(x, w, post_bias=w), lambda: f(x, w, bias=w.float()),
           lambda: f(x, w, out=x[:1]), lambda: f(x, w, out=x.float()), lambda: f(x, w, residual=x, residual_out=x.float()),
           lambda: f(x, w, residual=x, out=x, residual_out=x), lambda: f(x, w, out=x[:1].expand(2, 64)), lambda: f(None, w),
           lambda: f(x.double(), w)]
    for i, call in enumerate(bad):
        with pytest.raises((B200ArgumentError, B200NotSupportedError)):
            call()
            pytest.fail(f"call {i} was accepted")
    with pytest.raises(B200NotSupportedError, match="32768"):
        f(torch.zeros(1, 32776, dtype=BF16, device="cuda"), torch.zeros(32776, dtype=BF16, device="cuda"))
    for name in ("weight", "residual", "gate", "post_weight"):
        given = dict(weight=w, residual=x, gate=x, post_weight=w)
        given[name] = given[name].clone().requires_grad_()
        with pytest.raises(B200NotSupportedError, match="gradient"):
            f(x, given.pop("weight"), **given)
        with torch.no_grad():
            given = dict(weight=w, residual=x, gate=x, post_weight=w)
            given[name] = given[name].clone().requires_grad_()
            f(x, given.pop("weight"), **given)


# ---- mixture of experts ----------------------------------------------------------------------

def layer(gen, experts, width, inner, dtype, router_type=None, spread=2.0):
    return (normal(gen, (experts, width), router_type or dtype, spread / math.sqrt(width)),
            normal(gen, (experts, 2 * inner, width), dtype, 1 / math.sqrt(width)), normal(gen, (experts, width, inner), dtype, 1 / math.sqrt(inner)))


def moe_reference(x, router, gate_up, down, *, top_k, scoring="softmax", normalize=True, scale=1.0, selection_bias=None, activation="silu",
                  gap=1e-6):
    """y and its tolerance; the choice must not hang on rounding (scores nearer than `gap` at its border, unless equal)."""
    dtype, inner = x.dtype, down.shape[2]
    xd = x.double()
    logits = xd @ router.double().t()
    scores = torch.softmax(logits, 1) if scoring == "softmax" else torch.sigmoid(logits)
    by = scores if selection_bias is None else scores + selection_bias.double()
    ranked, order = torch.sort(by, dim=1, descending=True, stable=True)
    if top_k < by.shape[1]:
        near = ranked[:, top_k - 1] - ranked[:, top_k]
        assert ((near > gap * ranked[:, top_k - 1].abs()) | (near == 0)).all(), "the inputs' choice is too near"
    chosen = order[:, :top_k]
    share = scores.gather(1, chosen)
    if normalize:
        share = share / share.sum(1, keepdim=True)
    share = share * float(np.float32(scale))
    y, slack = torch.zeros_like(xd), torch.zeros_like(xd)
    step = torch.finfo(dtype).smallest_normal * half(dtype)
    for e in range(router.shape[0]):
        who, rank = torch.nonzero(chosen == e, as_tuple=True)
        if who.numel() == 0:
            continue
        w, d = gate_up[e].double(), down[e].double()
        both, size = xd[who] @ w.t(), (x.shape[1] / 16 + 8) * U * (xd[who].abs() @ w.abs().t())
        g, up, dg, du = both[:, :inner], both[:, inner:], size[:, :inner], size[:, inner:]
        act = g * torch.sigmoid(g) if activation == "silu" else 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
        dact = 1.13 * dg + 6 * V * (g.abs() if activation == "gelu" else act.abs())
        hidden = act * up
        dh = up.abs() * dact + act.abs() * du + dact * du + 3 * V * hidden.abs()
        dh = dh + half(dtype) * (hidden.abs() + dh) + step
        s = share[who, rank][:, None]
        y[who] += s * (hidden @ d.t())
        slack[who] += s.abs() * (dh @ d.abs().t() + ((inner / 16 + 16) * U + 8 * V) * (hidden.abs() @ d.abs().t()))
    return y, rounded(y, slack, dtype)


def check_moe(x, weights, **kw):
    want, tol = moe_reference(x, *weights, **kw)
    kw.pop("gap", None)
    if kw.get("selection_bias") is not None:
        kw["selection_bias"] = kw["selection_bias"].cuda()
    w = decoder.MoEWeights(*(t.cuda() for t in weights), **kw)
    xg = x.cuda()
    got = decoder.moe(xg, w)
    within(got, want, tol, "moe")
    assert torch.equal(decoder.moe(xg, w), got)   # no order of arrival in the results
    assert torch.equal(xg.cpu(), x)
    return got, w


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,experts,top_k,width,inner", [
    (1, 1, 1, 8, 8), (1, 8, 2, 64, 24), (2, 5, 5, 72, 40), (3, 16, 4, 256, 136), (8, 33, 7, 128, 64), (9, 33, 7, 128, 64), (1, 128, 8, 512, 96),
    (13, 60, 6, 264, 200), (17, 4, 1, 2048, 16), (33, 8, 2, 64, 520), (40, 2, 2, 200, 72), (1, 512, 32, 64, 32), (7, 512, 32, 64, 32),
    (70, 512, 32, 64, 32), (257, 6, 3, 64, 48), (600, 3, 1, 72, 64), (130, 40, 20, 64, 24), (4, 4, 2, 4096, 1032), (1, 2, 1, 1024, 4096),
    (40, 4, 2, 200, 2056), (260, 32, 4, 136, 1544), (50, 5, 1, 1032, 64),   # columns shared by a CTA, parts of k, ragged tiles
])
def test_moe_sizes(tokens, experts, top_k, width, inner, dtype):
    gen = torch.Generator().manual_seed(tokens * 1009 + experts * 31 + width)
    check_moe(normal(gen, (tokens, width), dtype), layer(gen, experts, width, inner, dtype), top_k=top_k)


@pytest.mark.parametrize("tokens", [1, 5, 21])
@pytest.mark.parametrize("kw", [
    dict(scoring="sigmoid"), dict(scoring="sigmoid", normalize=False, scale=2.5), dict(normalize=False), dict(scale=-0.7), dict(activation="gelu"),
    dict(bias=True), dict(bias=True, scoring="sigmoid", scale=1.5), dict(bias=True, normalize=False), dict(router_type=FP32),
    dict(router_type=FP32, scoring="sigmoid")])
def test_moe_scoring(tokens, kw):
    gen = torch.Generator().manual_seed(tokens * 17 + len(str(kw)))
    kw = dict(kw)
    x = normal(gen, (tokens, 136), BF16)
    weights = layer(gen, 24, 136, 56, BF16, kw.pop("router_type", None))
    if kw.pop("bias", False):
        kw["selection_bias"] = 0.1 * torch.randn(24, generator=gen)
    check_moe(x, weights, top_k=3, **kw)


@pytest.mark.parametrize("tokens", [3, 40])
def test_moe_equal_scores_go_to_the_lower_expert(tokens):
    gen = torch.Generator().manual_seed(2)
    x = normal(gen, (tokens, 64), BF16)
    router, gate_up, down = layer(gen, 70, 64, 32, BF16)
    router[:] = router[:1]                        # all of them
    check_moe(x, (router, gate_up, down), top_k=5)
    router[3:] = 0.5 * router[:1]                 # a few ahead or behind, by the logit's sign
    check_moe(x, (router, gate_up, down), top_k=5)


@pytest.mark.parametrize("tokens", [2, 12])
def test_moe_all_tokens_on_one_expert(tokens):
    """Other experts' weights are not touched: they hold NaN."""
    gen = torch.Generator().manual_seed(4)
    x = normal(gen, (tokens * 9, 64), FP16)
    router, gate_up, down = layer(gen, 9, 64, 40, FP16)
    bias = torch.zeros(9)
    bias[6] = 100.0
    for e in range(9):
        if e != 6:
            gate_up[e], down[e] = math.nan, math.nan
    check_moe(x, (router, gate_up, down), top_k=1, selection_bias=bias, scoring="sigmoid")


def test_moe_strides_place_and_more_streams():
    gen = torch.Generator().manual_seed(5)
    width, inner, experts = 128, 72, 6
    router, gate_up, down = layer(gen, experts, width, inner, BF16)
    x = normal(gen, (11, width), BF16)
    want, w = check_moe(x, (router, gate_up, down), top_k=2)
    big = torch.zeros(experts + 1, 2 * inner + 3, width + 8, dtype=BF16, device="cuda")
    big[1:, 3:, 8:] = gate_up.cuda()
    low = torch.zeros(width, experts, inner + 16, dtype=BF16, device="cuda")    # experts inside
    low[:, :, :inner] = down.cuda().transpose(0, 1)
    rt = torch.zeros(experts, 2 * width, dtype=BF16, device="cuda")
    rt[:, width:] = router.cuda()
    other = decoder.MoEWeights(rt[:, width:], big[1:, 3:, 8:], low[:, :, :inner].transpose(0, 1), top_k=2)
    wide = torch.full((11, 3 * width), 7.0, dtype=BF16, device="cuda")
    wide[:, width: 2 * width] = x.cuda()
    out = torch.full((11, 2 * width), 7.0, dtype=BF16, device="cuda")
    assert torch.equal(decoder.moe(wide[:, width: 2 * width], other, out=out[:, width:]), want)
    assert (out[:, :width] == 7.0).all() and (wide[:, :width] == 7.0).all()
    xg = x.cuda()
    decoder.moe(xg, other, out=xg)
    assert torch.equal(xg, want)
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    xg = x.cuda()
    torch.cuda.synchronize()
    for i in range(12):                                                           # calls that may overlap
        with torch.cuda.stream(streams[i % 3]):
            results.append(decoder.moe(xg, w))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


@pytest.mark.parametrize("tokens", [4, 30])
def test_moe_keeps_tokens_apart(tokens):
    gen = torch.Generator().manual_seed(6)
    weights = layer(gen, 8, 64, 32, FP16)
    x = normal(gen, (tokens, 64), FP16)
    clean, w = check_moe(x, weights, top_k=2)
    x[1, 7], x[2] = math.nan, 0.0
    y = decoder.moe(x.cuda(), w).cpu()
    keep = [i for i in range(tokens) if i not in (1, 2)]
    assert torch.equal(y[keep], clean.cpu()[keep]) and torch.isnan(y[1]).all() and (y[2] == 0).all()
    assert decoder.moe(x[:0].cuda(), w).shape == (0, 64)
    assert torch.equal(decoder.moe(x[keep[:1]].cuda(), w).cpu(), clean.cpu()[keep[:1]])   # a token by itself


def test_moe_refuses():
    gen = torch.Generator().manual_seed(1)
    r, g, d = (t.cuda() for t in layer(gen, 4, 64, 32, BF16))
    x = torch.zeros(3, 64, dtype=BF16, device="cuda")
    make = decoder.MoEWeights
    w = make(r, g, d, top_k=2)
    bad = [lambda: make(r, g, d, top_k=0), lambda: make(r, g, d, top_k=5), lambda: make(r[:3], g, d, top_k=2), lambda: make(r, g[:, :63], d, top_k=2),
           lambda: make(r, g, d.half(), top_k=2), lambda: make(r.half(), g, d, top_k=2), lambda: make(r, g, d.transpose(1, 2), top_k=2),
           lambda: make(r, g, d, top_k=2, scoring="x"), lambda: make(r, g, d, top_k=2, activation="x"),
           lambda: make(r, g, d, top_k=2, scale=math.nan), lambda: make(r, g, d, top_k=2, selection_bias=r[0]),
           lambda: make(r, g, d, top_k=2, selection_bias=torch.zeros(3, device="cuda")), lambda: make(r.float(), g.float(), d.float(), top_k=2),
           lambda: make(r[:, :60], g[:, :, :60], d[:, :60], top_k=2), lambda: make(r, g.transpose(0, 1).contiguous().transpose(1, 0)[:, :, :], d[..., :4], top_k=2),
           lambda: decoder.moe(x, None), lambda: decoder.moe(x.half(), w), lambda: decoder.moe(x[:, :32], w), lambda: decoder.moe(x[0], w),
           lambda: decoder.moe(x.cpu(), w), lambda: decoder.moe(x, w, out=x[:2]), lambda: decoder.moe(x, w, out=x[:1].expand(3, 64)),
           lambda: decoder.moe(torch.zeros(3, 65, dtype=BF16, device="cuda")[:, 1:], w)]
    for i, call in enumerate(bad):
        with pytest.raises((B200ArgumentError, B200NotSupportedError)):
            call()
            pytest.fail(f"call {i} was accepted")
    for i in range(3):
        t = [r, g, d]
        t[i] = t[i].clone().requires_grad_()
        with pytest.raises(B200NotSupportedError, match="gradient"):
            make(*t, top_k=2)
        with torch.no_grad():
            late = make(*t, top_k=2)
            decoder.moe(x, late)
        with pytest.raises(B200NotSupportedError, match="gradient"):
            decoder.moe(x, late)


# ---- sampling --------------------------------------------------------------------------------

def chosen(row, u, temperature, top_k, top_p, min_p):
    """The definition, in 64 bits, of one row."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    n, best = row.size, row.max()
    if best == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.flatnonzero(row == best)[0])
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        w = np.where(row == best, 1.0, np.exp(np.where(row == -np.inf, -np.inf, (row - best) / temperature)))
    order = np.lexsort((np.arange(n), -row))
    order = order[w[order] > 0]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    if 0 < top_k < n:
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order])
        order = order[: max(1, int((mass < top_p * mass[-1]).sum()) + 1)]
    order = np.sort(order)
    mass, u = np.cumsum(w[order]), min(max(u, 0.0), 1.0)
    at = min(int((mass <= u * mass[-1]).sum()), order.size - 1)
    kinds = np.unique(w[order])
    if kinds.size <= 4:   # sums of few different weights may equal u times theirs, which rounded sums do not show: exact ones
        counts = [np.cumsum(w[order] == v) for v in kinds]
        upto = lambda i: sum(Fraction(float(v)) * int(c[i]) for v, c in zip(kinds, counts)) if i >= 0 else 0
        target = Fraction(u) * upto(order.size - 1)
        while at > 0 and upto(at - 1) > target:
            at -= 1
        while at < order.size - 1 and upto(at) <= target:
            at += 1
    return int(order[at])


def check_sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    each = lambda v: v.tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * logits.shape[0]
    gpu = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v
    got = decoder.sample(logits.cuda(), u.cuda(), temperature=gpu(temperature), top_k=gpu(top_k), top_p=gpu(top_p), min_p=gpu(min_p)).cpu()
    assert got.dtype is torch.int64
    rows = logits.float().numpy()
    want = [chosen(rows[i], *v) for i, v in enumerate(zip(u.tolist(), each(temperature), map(int, each(top_k)), each(top_p), each(min_p)))]
    assert got.tolist() == want
    return got


SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.5, top_k=40, top_p=0.7, min_p=0.001),
            dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(top_p=1e-7), dict(min_p=1.0), dict(top_k=1000, top_p=0.999)]


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 513), (40, 1000), (7, 4097), (160, 3001), (1, 32000), (3, 65537), (80, 20011)])
def test_sample(rows, vocab, dtype):
    gen = torch.Generator().manual_seed(rows * 131 + vocab)
    logits = (torch.randn((rows, vocab), generator=gen) * (0.5 + 3 * torch.rand((rows, 1), generator=gen))).to(dtype)
    for kw in SETTINGS:
        check_sample(logits, torch.rand(rows, generator=gen), **kw)


@pytest.mark.parametrize("vocab,dtype", [(262144, FP32), (380001, FP32), (500001, FP32), (900013, BF16)])
def test_sample_wide(vocab, dtype):
    """Slices beyond shared memory (the last two) and near its limit."""
    gen = torch.Generator().manual_seed(vocab)
    logits = (2 * torch.randn((3, vocab), generator=gen)).to(dtype)
    for kw in (dict(), dict(top_p=0.8), dict(top_k=300, temperature=0.9), dict(temperature=0.0)):
        check_sample(logits, torch.rand(3, generator=gen), **kw)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_sample_equal_logits(dtype):
    """Rows of few distinct values: the border is a tie, cut in the order of the index."""
    gen = torch.Generator().manual_seed(11)
    logits = torch.randint(0, 4, (40, 9001), generator=gen).to(dtype)
    logits[:8] = 1.5                 # all the same
    logits[8] = -logits[8] * 0.0     # zeros of both signs
    logits[9] = 0.0
    logits[9, ::2] = -0.0
    logits[10] = -1e30 if dtype is FP32 else -1e4
    u = torch.rand(40, generator=gen)
    for kw in (dict(), dict(top_k=1), dict(top_k=700), dict(top_k=3000), dict(top_p=0.3), dict(top_p=0.77), dict(top_k=4000, top_p=0.4), dict(min_p=0.2),
               dict(temperature=0.0), dict(top_k=8999), dict(top_p=0.99999)):
        check_sample(logits, u, **kw)


def test_sample_of_the_widest_rows():
    """2^21 equal logits (their weights sum to 2^61), and few above the others."""
    logits = torch.zeros((3, 1 << 21), dtype=BF16)
    logits[1, 1234567] = 9.0
    logits[2, ::4097] = 3.5
    for kw in (dict(), dict(top_p=0.5), dict(top_k=100000)):
        check_sample(logits, torch.tensor([0.75, 0.999, 0.5]), **kw)


def test_sample_every_part_of_the_unit_interval():
    gen = torch.Generator().manual_seed(12)
    row = torch.randn(300, generator=gen) * 2
    u = torch.cat((torch.linspace(0, 1, 1000), torch.tensor([1.0 - 2.0 ** -24, 0.0, 1e-30])))
    got = check_sample(row.expand(u.numel(), 300), u, top_k=60)
    assert got.unique().numel() > 40 and (got[1:1000] >= got[:999]).all()
    odd = torch.tensor([math.nan, -1.0, 2.0, math.inf])
    got = decoder.sample(row.expand(4, 300).cuda(), odd.cuda()).cpu()
    ends = decoder.sample(row.expand(4, 300).cuda(), torch.tensor([0.0, 0.0, 1.0, 1.0]).cuda()).cpu()
    assert torch.equal(got, ends) and ends[0] == 0 and ends[2] == 299


def test_sample_of_infinities_and_nan():
    gen = torch.Generator().manual_seed(13)
    n = 5000
    logits = torch.randn((12, n), generator=gen)
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 1:] = -math.inf
    logits[3, :-1] = -math.inf
    logits[4, 100:] = math.nan
    logits[5, [7, 90, 4000]] = math.inf
    logits[6, ::2] = -math.inf
    logits[7] = torch.finfo(FP32).min
    logits[7, 17] = torch.finfo(FP32).max
    logits[8, 5:] = torch.finfo(FP32).min            # a mask by the lowest value
    logits[9] = math.nan
    logits[9, 4321] = -math.inf
    logits[10] = math.inf
    logits[11] *= 1e38
    for kw in SETTINGS + [dict(temperature=math.inf), dict(temperature=1e-40), dict(temperature=math.inf, top_k=9, top_p=0.5)]:
        got = check_sample(logits, torch.rand(12, generator=gen), **kw)
        assert got[[0, 1, 9]].tolist() == [-1] * 3
    check_sample(logits.half(), torch.rand(12, generator=gen), top_p=0.8)


def test_sample_settings_of_each_row():
    gen = torch.Generator().manual_seed(14)
    rows, vocab = 200, 2500
    logits = torch.randn((rows, vocab), generator=gen) * 3
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=gen)]
    kw = dict(temperature=pick(0.0, 0.5, 1.0, 2.0, -1.0), top_k=pick(0, 1, 7, 5000, -3, 2500).int(), top_p=pick(1.0, 0.9, 0.2, 2.0, 0.0),
              min_p=pick(0.0, 0.1, -1.0))
    u = torch.rand(rows, generator=gen)
    check_sample(logits, u, **kw)
    nan = torch.full((rows,), math.nan)
    got = decoder.sample(logits.cuda(), u.cuda(), temperature=nan.cuda())
    assert torch.equal(got, logits.cuda().argmax(1))
    plain = decoder.sample(logits.cuda(), u.cuda())
    assert torch.equal(decoder.sample(logits.cuda(), u.cuda(), top_p=nan.cuda(), min_p=nan.cuda()), plain)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_sample_strides_and_what_lies_beside(dtype, shift):
    gen = torch.Generator().manual_seed(15)
    wide = torch.full((6, 5011), math.inf, dtype=dtype)       # beside the rows, larger than all of them
    wide[:, shift: shift + 4999] = torch.randn((6, 4999), generator=gen).to(dtype)
    u = torch.rand(6, generator=gen)
    want = check_sample(wide[:, shift: shift + 4999].contiguous(), u, top_p=0.9)
    out = torch.full((8,), 77, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g, ug = wide.cuda(), u.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        decoder.sample(g[:, shift: shift + 4999], ug, top_p=0.9, out=out[1:7])
    side.synchronize()
    assert out.tolist() == [77] + want.tolist() + [77]
    assert decoder.sample(g[:0, :9], ug[:0]).shape == (0,)
    assert torch.equal(decoder.sample(g[:1, shift: shift + 4999].expand(6, 4999), ug, top_p=0.9)[:1].cpu(), want[:1])


def test_sample_refuses():
    x, u = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda")
    f = decoder.sample
    bad = [lambda: f(x[0], u), lambda: f(x, u[:2]), lambda: f(x, u.double()), lambda: f(x, u.cpu()), lambda: f(x.t(), u), lambda: f(x.double(), u),
           lambda: f(x.cpu(), u), lambda: f(x, u, temperature=u[:2]), lambda: f(x, u, top_k=u), lambda: f(x, u, top_p=u.half()),
           lambda: f(x, u, min_p=u.cpu()), lambda: f(x, u, temperature=math.nan), lambda: f(x, u, top_p=math.nan), lambda: f(x, u, min_p=math.nan),
           lambda: f(x, u, out=u.int()), lambda: f(x, u, out=torch.zeros(2, dtype=torch.int64, device="cuda")), lambda: f(x[:, :0], u), lambda: f(None, u),
           lambda: f(x, None), lambda: f(x, torch.zeros(6, device="cuda")[::2])]
    for i, call in enumerate(bad):
        with pytest.raises((B200ArgumentError, B200NotSupportedError)):
            call()
            pytest.fail(f"call {i} was accepted")
    with pytest.raises(B200NotSupportedError, match="gradient"):
        f(x.clone().requires_grad_(), u)


# ---- together --------------------------------------------------------------------------------

def test_a_decoder_step_eager_and_replayed():
    """From the hidden states to the next tokens, on the library's operators alone; then the same step captured into a
    graph and replayed on other hidden states and numbers."""
    gen = torch.Generator().manual_seed(21)
    batch, width, heads, kv, dim, vocab, page = 5, 256, 4, 2, 64, 3000, 16
    rand = lambda *shape, scale=1.0: normal(gen, shape, BF16, scale).cuda()

    def linear(out, inp):
        packed = torch.randint(0, 256, (out, inp // 2), generator=gen, dtype=torch.uint8).cuda()
        return decoder.W4Weights(packed, torch.full((out, inp // 64), 0.2 / math.sqrt(inp), dtype=BF16, device="cuda"), in_features=inp, group_size=64)

    qkv_w, proj, head = linear((heads + 2 * kv) * dim, width), linear(width, heads * dim), linear(vocab, width)
    experts = tuple(t.cuda() for t in layer(gen, 8, width, 128, BF16))
    moe_w = decoder.MoEWeights(*experts, top_k=2)
    norms = [(1 + rand(width, scale=0.1)) for _ in range(4)]
    table = decoder.RotaryTable(dim, device="cuda")
    context = torch.tensor([20, 33, 1, 16, 50], dtype=torch.int32, device="cuda")
    pages = torch.arange(5 * 4, dtype=torch.int32, device="cuda").view(5, 4)
    cache = decoder.PagedCache(rand(20, page, kv, dim), rand(20, page, kv, dim), pages, context)
    starts = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    hidden, uniform = rand(batch, width), torch.rand(batch, generator=gen).cuda()

    def step():
        seen = {}
        y, h = decoder.residual_norm(hidden, norms[0])
        qkv = decoder.linear_w4(y, qkv_w).view(batch, -1, dim)
        q = decoder.paged_append(cache, qkv[:, heads: heads + kv], qkv[:, heads + kv:], starts, q=qkv[:, :heads], table=table)
        o = decoder.linear_w4(decoder.paged_attention(cache, q, starts).flatten(1), proj)
        seen["o"], seen["h0"] = o, h
        y, h = decoder.residual_norm(o, norms[1], residual=h)
        seen["y1"], seen["h1"] = y, h
        m = decoder.moe(y, moe_w)
        seen["m"] = m
        y, h = decoder.residual_norm(m, norms[2], residual=h, post_weight=norms[3])
        seen["y2"], seen["h2"] = y, h
        seen["logits"] = decoder.linear_w4(y, head)
        seen["tokens"] = decoder.sample(seen["logits"], uniform, temperature=0.8, top_k=50, top_p=0.95)
        return seen

    def check(seen):
        c = {k: v.cpu() for k, v in seen.items()}
        n = [w.cpu() for w in norms]
        for x, r, w, post, y, h in ((c["o"], c["h0"], n[1], None, "y1", "h1"), (c["m"], c["h1"], n[2], n[3], "y2", "h2")):
            wy, dy, wh, dh = norm_reference(x, w, residual=r, post_weight=post)
            within(c[y], wy, rounded(wy, dy, BF16), y)
            within(c[h], wh, rounded(wh, dh, BF16), h)
        want, tol = moe_reference(c["y1"], *(t.cpu() for t in experts), top_k=2)
        within(c["m"], want, tol, "moe")
        rows, f = c["logits"].float().numpy(), lambda v: float(np.float32(v))
        assert c["tokens"].tolist() == [chosen(rows[i], float(uniform[i]), f(0.8), 50, f(0.95), 0.0) for i in range(batch)]

    eager = step()
    check(eager)
    again = step()                                     # the cache holds the same step: the same results
    for k in eager:
        assert torch.equal(eager[k], again[k]), k
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        replayed = step()
    graph.replay()
    for k in eager:
        assert torch.equal(eager[k], replayed[k]), k
    for _ in range(3):
        hidden.copy_(normal(gen, (batch, width), BF16))
        uniform.copy_(torch.rand(batch, generator=gen))
        graph.replay()
        check(replayed)
        fresh = step()
        for k in fresh:
            assert torch.equal(fresh[k], replayed[k]), k
    decoder.check()
