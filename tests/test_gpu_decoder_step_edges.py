"""More GPU tests of the residual norms, mixture-of-experts layers and sampling: routers with logits far apart, scores
next to each other, hidden values that cancel, draws in a row's flat tail, the streaming forms of the norms. Tolerances
as in the tests beside these (h, v, u there), and with what each test says.
"""
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from shorokoo_b200 import B200ArgumentError, B200NotSupportedError, decoder
from test_gpu_decoder_step import BF16, FP16, FP32, U, V, check_moe, check_sample, half, layer, norm_reference, normal, rounded, within

pytestmark = pytest.mark.gpu


# ---- mixture of experts ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,experts,top_k,width,inner", [(1, 4, 2, 16, 64), (3, 4, 2, 16, 64), (40, 2, 1, 16, 64), (90, 5, 3, 24, 72),
                                                              (2, 3, 2, 16, 1032), (50, 2, 2, 16, 1032), (2, 3, 2, 16, 2056), (50, 2, 2, 16, 2056)])
def test_moe_keeps_hidden_values_that_cancel(tokens, experts, top_k, width, inner, dtype):
    """Pairs of features with nearly the same hidden value and opposite weights behind them. What a rounding of hidden values to the
    type would lose (h of each) is many times what is left of a pair; two values of the type hold them to h^2 (fp16: of values
    and remainders that are normal numbers; the remainders are held 2^11 times as large, so 2^-36 and h 2^-25 below that)."""
    gen = torch.Generator().manual_seed(tokens * 31 + inner)
    router, gate_up, down = layer(gen, experts, width, inner, dtype)
    gate_up[:, 1:inner:2] = gate_up[:, 0:inner:2]
    gate_up[:, inner + 1::2] = (gate_up[:, inner::2].float() * (1 + 0.1 * torch.randn((experts, inner // 2, 1), generator=gen))).to(dtype)
    down[:, :, 1::2] = -down[:, :, 0::2]
    x = normal(gen, (tokens, width), dtype)
    xd = x.double()
    share, chosen = torch.softmax(xd @ router.double().t(), 1).topk(top_k, dim=1)
    share = share / share.sum(1, keepdim=True)
    want, slack = torch.zeros_like(xd), torch.zeros_like(xd)
    for t in range(tokens):
        for s, e in zip(share[t], chosen[t]):
            w, d = gate_up[e].double(), down[e].double()
            both, size = w @ xd[t], (width / 16 + 8) * U * (w.abs() @ xd[t].abs())
            act, up = both[:inner] * torch.sigmoid(both[:inner]), both[inner:]
            hidden = act * up
            dact = 1.13 * size[:inner] + 6 * V * act.abs()
            dh = up.abs() * dact + act.abs() * size[inner:] + dact * size[inner:] + 3 * V * hidden.abs()
            dh = dh + half(dtype) ** 2 * (hidden.abs() + dh) + (half(dtype) * 2.0 ** -25 + 2.0 ** -36 if dtype is FP16 else 0.0)
            want[t] += s * (d @ hidden)
            slack[t] += s * (d.abs() @ dh + ((inner / 16 + 16) * U + 8 * V) * (d.abs() @ hidden.abs()))
    w = decoder.MoEWeights(router.cuda(), gate_up.cuda(), down.cuda(), top_k=top_k)
    within(decoder.moe(x.cuda(), w), want, rounded(want, slack, dtype), "moe")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,experts", [(1, 3), (40, 2)])
def test_moe_of_infinite_weights(tokens, experts, dtype):
    """One infinite weight behind a hidden value makes its output infinite, of the value's sign, and no other."""
    gen = torch.Generator().manual_seed(tokens)
    router, gate_up, down = layer(gen, experts, 64, 40, dtype)
    x = normal(gen, (tokens, 64), dtype)
    down[:, 17, 5] = math.inf
    hidden = lambda e: (lambda g, u: g * torch.sigmoid(g) * u)(x.double() @ gate_up[e, 5].double(), x.double() @ gate_up[e, 45].double())
    first = (x.double() @ router.double().t()).argmax(1)
    sign = torch.stack([hidden(e) for e in range(experts)], 1)[torch.arange(tokens), first].sign()
    y = decoder.moe(x.cuda(), decoder.MoEWeights(router.cuda(), gate_up.cuda(), down.cuda(), top_k=1)).cpu().double()
    assert torch.equal(y[:, 17], sign * math.inf)
    assert torch.isfinite(y[:, :17]).all() and torch.isfinite(y[:, 18:]).all()


def by_logits(gen, logits, tokens, dtype, width=32, inner=40, router_type=None):
    """x and a layer whose experts have these logits for every token, from the first input alone; the others are the tokens' own."""
    router, gate_up, down = layer(gen, len(logits), width, inner, dtype, router_type)
    router[:] = 0
    router[:, 0] = torch.tensor(logits)
    x = normal(gen, (tokens, width), dtype)
    x[:, 0] = 1.0
    return x, (router, gate_up, down)


@pytest.mark.parametrize("tokens", [1, 30])
@pytest.mark.parametrize("logits,bias,top_k", [
    ((-100.0, 0.0), (2.0, 0.0), 2), ((45.0, -50.0, 1.0, 2.0), (0.0, 10.0, 0.0, 0.0), 2), ((-300.0, -200.0, 0.0, -1.0, 5.0), (9.0, 8.0, 0.0, 0.0, 7.0), 3),
    ((-300.0, -200.0, 0.0, -1.0, 5.0), (9.0, 8.0, 0.0, 0.0, 7.0), 5), ((0.0, -200.0, -201.0), (0.0, 5.0, 4.0), 2)])
def test_moe_softmax_shares_of_experts_chosen_by_their_bias(logits, bias, top_k, tokens):
    """The first chosen has a logit far below another's, or all chosen are far below the rest."""
    gen = torch.Generator().manual_seed(tokens + len(logits))
    for dtype in (BF16, FP16):
        x, weights = by_logits(gen, logits, tokens, dtype)
        check_moe(x, weights, top_k=top_k, selection_bias=torch.tensor(bias))


@pytest.mark.parametrize("tokens", [1, 30])
@pytest.mark.parametrize("logits,bias,top_k", [
    ((-91.0, -92.0, -95.0), None, 2), ((-91.0,), None, 1), ((-300.0, -120.0, -119.0, -118.0), None, 3), ((-300.0, -120.0, -119.0, 3.0), None, 3),
    ((-100.0, -101.0, 60.0, 61.0), (5.0, 4.0, 0.0, 0.0), 2), ((-100.0, -101.0, 60.0, 61.0), (5.0, 4.0, 0.0, 3.5), 3)])
def test_moe_sigmoid_shares_of_scores_next_to_nothing(logits, bias, top_k, tokens):
    """Scores of 10^-40 and less have their ratios all the same."""
    gen = torch.Generator().manual_seed(tokens + len(logits))
    for dtype in (BF16, FP16):
        x, weights = by_logits(gen, logits, tokens, dtype)
        check_moe(x, weights, top_k=top_k, scoring="sigmoid", selection_bias=None if bias is None else torch.tensor(bias))


def test_moe_sigmoid_share_of_a_single_expert():
    """All of it, at any score, also at those that are none in 64 bits."""
    gen = torch.Generator().manual_seed(1)
    x, (router, gate_up, down) = by_logits(gen, (0.0, -1.0), 3, BF16)
    run = lambda: decoder.moe(x.cuda(), decoder.MoEWeights(router.cuda(), gate_up.cuda(), down.cuda(), top_k=1, scoring="sigmoid"))
    want = run()
    for logit in (-50.0, -1000.0, -1e30, 1000.0):
        router[:, 0] = torch.tensor([logit, 2 * logit if logit < 0 else -logit])
        assert torch.equal(run(), want)


@pytest.mark.parametrize("experts", [6, 300])
@pytest.mark.parametrize("kw", [dict(), dict(scoring="sigmoid"), dict(selection_bias=0.0), dict(selection_bias=1000.0),
                                dict(selection_bias=-3.0, scoring="sigmoid"), dict(normalize=False)])
def test_moe_orders_experts_by_scores_in_64_bits(kw, experts):
    """Two logits 2^-30 apart (with a bias of 1000 2^-20, where fp32 has steps of 2^-14): the larger is chosen, not the lower expert."""
    gen = torch.Generator().manual_seed(experts)
    for tokens in (1, 20):
        x, weights = by_logits(gen, [0.0] * experts, tokens, BF16, router_type=FP32)
        bias = kw.get("selection_bias")
        x[:, 8] = 2.0 ** -10 if bias == 1000.0 else 2.0 ** -15
        weights[0][[1, 4], 0] = 1.0
        weights[0][4, 8] = x[0, 8].float()
        given = dict(kw)
        if bias is not None:
            given["selection_bias"] = torch.zeros(experts)
            given["selection_bias"][[1, 4]] = bias if bias > 0 else 0.0
            if bias < 0:
                given["selection_bias"] += bias
        check_moe(x, weights, top_k=1, gap=0.0, **given)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens", [1, 20])
def test_moe_sums_a_16_bit_router_in_64_bits(tokens, dtype):
    """Products of one piece of eight inputs, of 1 and of 2^-26, and such as cancel: 32 bits would lose the small ones."""
    gen = torch.Generator().manual_seed(tokens)
    x, weights = by_logits(gen, [0.0] * 5, tokens, dtype)
    x[:, 1], x[:, 2] = 2.0 ** -13, -1.0
    weights[0][[1, 4], 0] = 1.0
    weights[0][4, 1] = 2.0 ** -13
    check_moe(x, weights, top_k=1, gap=0.0)
    weights[0][:, 2] = 1.0 - 2.0 ** -6          # 0 in place of 1, 2^-6 in place of 0
    weights[0][[1, 4], 2] = 1.0 - 2.0 ** -5
    check_moe(x, weights, top_k=1, gap=0.0)


# ---- sampling --------------------------------------------------------------------------------

def check_draws(row, u, temperature=1.0):
    """The tokens of one row for many u, against sums in long double. Weights are off by half a unit of 2^-42 of the largest and
    by 2^-27.9 of themselves (a number of 2^29 to 2^30, off by half from a table, times one off by 2^-30, the product cut off to a
    whole number: 2^-30 + 2^-30 + 2^-29, and 2^-32 of what is rounded before), so that a running sum and u times all of
    them differ by at most n units and 2^-26.9 of all from what they are; a token whose border is nearer than that to the target
    may be its neighbour."""
    row = row.double().numpy().astype(np.longdouble)
    w = np.exp((row - row.max()) / np.longdouble(np.float32(temperature)))
    mass = np.concatenate((np.zeros(1, np.longdouble), np.cumsum(w)))
    off = row.size * np.longdouble(2) ** -42 + np.longdouble(2) ** np.longdouble(-26.9) * mass[-1] + np.longdouble(2) ** -41
    target = u.numpy().astype(np.longdouble) * mass[-1]
    def check(got):
        got = got.cpu().numpy()
        wrong = (target < mass[got] - off) | (target >= mass[got + 1] + off)
        assert not wrong.any(), f"{int(wrong.sum())} of {wrong.size} draws are off"
    return check


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("vocab", [150001, 200000])
def test_sample_in_the_tail_of_a_peaked_row(vocab, dtype):
    """One token with nearly all the mass and a tail of weights of some 10^-9, where nearly all the u of this test point: roundings of the
    weights that go one way add up along it."""
    gen = torch.Generator().manual_seed(vocab)
    row = (0.3 * torch.randn(vocab, generator=gen)).to(dtype)
    row[100] = 19.0
    tail = float(torch.exp(row.double() - 19.0).sum()) - 1.0
    u = torch.cat((torch.rand(100, generator=gen), 1 - tail / (1 + tail) * torch.rand(3000, generator=gen).double())).float().clamp(max=1 - 2.0 ** -24)
    check = check_draws(row, u)
    logits = row.cuda().expand(u.numel(), vocab)
    check(decoder.sample(logits, u.cuda()))
    check(torch.cat([decoder.sample(logits[i: i + 10], u[i: i + 10].cuda()) for i in range(0, 400, 10)] + [decoder.sample(logits[400:], u[400:].cuda())]))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_sample_of_tiny_logits_below_a_large_one(dtype):
    """What the difference from the largest loses in fp32 is the same for all of them, and as much as some tokens weigh."""
    gen = torch.Generator().manual_seed(5)
    row = torch.full((150001,), 7 * 2.0 ** -24).to(dtype)
    row[::1000] = torch.randn(151, generator=gen).to(dtype)
    row[100000] = 10.0
    u = torch.rand(20000, generator=gen)
    check_draws(row, u)(decoder.sample(row.cuda().expand(u.numel(), row.numel()), u.cuda()))


@pytest.mark.parametrize("temperature", [1e-2, 1e-3, 1e-4, 1e-6])
def test_sample_at_low_temperatures(temperature):
    """Quotients of logit and temperature from thousands to millions, and tokens near enough to count all the same."""
    gen = torch.Generator().manual_seed(6)
    for top in (30.0, -50.0, 1000.0):
        row = top - 10 * max(temperature, abs(top) * 2.0 ** -22) * torch.rand(50001, generator=gen)
        u = torch.rand(4000, generator=gen)
        check_draws(row, u, temperature)(decoder.sample(row.cuda().expand(u.numel(), row.numel()), u.cuda(), temperature=temperature))


@pytest.mark.parametrize("temperature", [1e-3, 1e-4, 1e-5])
def test_sample_filters_at_low_temperatures(temperature):
    gen = torch.Generator().manual_seed(8)
    logits = 30 + max(3 * temperature, 1e-4) * torch.randn((20, 5001), generator=gen)
    for kw in (dict(), dict(top_k=40), dict(top_k=1000), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.05), dict(top_k=400, top_p=0.8, min_p=0.001)):
        check_sample(logits, torch.rand(20, generator=gen), temperature=temperature, **kw)


# ---- residual norms --------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width,dtype", [(3, 64, BF16), (700, 4096, BF16), (5, 75, FP32)])
def test_residual_norm_over_x_leaves_h(rows, width, dtype):
    """Where h is x itself and y goes over x, h is a tensor of its own."""
    gen = torch.Generator().manual_seed(rows)
    x, w = normal(gen, (rows, width), dtype).cuda(), normal(gen, (width,), dtype).cuda()
    before = x.clone()
    want, h = decoder.residual_norm(x, w)
    assert h is x and torch.equal(x, before)
    y, h = decoder.residual_norm(x, w, out=x)
    assert y is x and torch.equal(y, want) and torch.equal(h, before)
    x = before.clone()
    y, h = decoder.residual_norm(x, w, out=x.view(rows, width))          # the same memory by another name
    assert torch.equal(x, want) and torch.equal(h, before)


def test_settings_that_are_no_numbers_of_their_type_are_refused():
    gen = torch.Generator().manual_seed(1)
    r, g, d = (t.cuda() for t in layer(gen, 4, 64, 32, BF16))
    for top_k in (2 ** 32 + 2, -2 ** 32 + 2, 2 ** 31, math.nan, math.inf, None, "two"):
        with pytest.raises(B200ArgumentError):
            decoder.MoEWeights(r, g, d, top_k=top_k)
    with pytest.raises(B200ArgumentError):
        decoder.MoEWeights(r, g, d, top_k=2, scale="one")
    x, u = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda")
    for kw in (dict(top_k=math.nan), dict(top_k=None), dict(top_k="two"), dict(top_p=None), dict(temperature="hot"), dict(top_k=math.inf)):
        with pytest.raises(B200ArgumentError):
            decoder.sample(x, u, **kw)
    assert decoder.sample(x, u, top_k=2 ** 40).tolist() == [0, 0, 0]     # more than there are


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,width,pitch", [(6100, 1024, 1024), (6100, 1033, 1033), (6000, 1500, 1501), (3100, 2048, 2056), (3100, 2050, 2050), (1600, 4096, 4096),
                                              (1600, 4099, 4099), (1600, 4095, 4100), (950, 5003, 5003), (950, 6000, 6000), (620, 11001, 11001)])
def test_residual_norm_of_rows_that_stream(rows, width, pitch, dtype):
    """More than two rows for each of as many CTAs as 148 multiprocessors hold (20 of the shortest rows here), in every type, aligned or not;
    rows spread over all of them against the formula, in the forms that differ in what streams beside x."""
    gen = torch.Generator(device="cuda").manual_seed(rows + width)
    rand = lambda *shape, kind=dtype: torch.randn(shape, device="cuda", generator=gen).to(kind)
    x, r, g = (rand(rows, pitch)[:, pitch - width:] for _ in range(3))
    wide = rand(rows, pitch, kind=FP32)[:, pitch - width:]
    w, b, p, c, v = (rand(width) for _ in range(5))
    f = lambda t: t.float() * 1.001
    room = lambda kind: torch.empty((rows, pitch), dtype=kind, device="cuda")[:, pitch - width:]     # rows that begin as x's do
    some = sorted({i * (rows - 1) // 60 for i in range(61)} | {i for i in (1, 2, 147, 148, 739, 740, rows - 2) if i < rows})
    host = lambda t: t if not isinstance(t, torch.Tensor) else t[some].cpu() if t.dim() == 2 else t.cpu()
    for given in (dict(residual=r), dict(bias=b, residual=r, post_weight=p, post_bias=c, gate=g, scale=0.3, kind="layer"),
                  dict(residual=wide, gate=v, kind="layer", eps=1e-5), dict(residual=wide, post_weight=p, gate=g, weight_offset=1.0), dict(gate=g, bias=b)):
        for weight in (w, f(w)):
            if weight.dtype is FP32:
                given = {k: f(t) if k in ("bias", "post_weight", "post_bias") else t for k, t in given.items()}
            stream = given["residual"].dtype if "residual" in given else dtype
            y, h = decoder.residual_norm(x, weight, out=room(dtype), residual_out=room(stream), **given)
            wy, dy, wh, dh = norm_reference(host(x), weight.cpu(), **{k: host(t) for k, t in given.items()})
            within(y[some], wy, rounded(wy, dy, dtype), "y")
            within(h[some], wh, rounded(wh, dh, h.dtype), "h")
    given = dict(gate=g, post_weight=p)
    a, d = room(dtype).copy_(x), room(FP32).copy_(wide)
    y, h = decoder.residual_norm(x, w, residual=wide, out=room(dtype), residual_out=room(FP32), **given)
    decoder.residual_norm(a, w, residual=d, out=a, residual_out=d, **given)
    assert torch.equal(a, y) and torch.equal(d, h)

@pytest.mark.parametrize("rows,width", [(3, 3), (5, 48), (2, 768), (700, 768), (400, 1001), (1300, 4100), (2, 6000), (300, 11001), (2, 20000)])
def test_residual_norm_of_equal_values(rows, width):
    """A layer norm of equal values of 8 bits: their sums and mean are exact, so nothing is left but the bias."""
    gen = torch.Generator().manual_seed(width)
    w, b = normal(gen, (width,), FP32).cuda(), normal(gen, (width,), FP32).cuda()
    value = torch.tensor([1000.0, -3.5, 1.0078125, 253.0, 30000.0, 1e-3, 0.0, 44032.0]).bfloat16().float()
    x = value[torch.arange(rows) % 8][:, None].expand(rows, width).cuda()
    for kind in (BF16, FP32):
        y, h = decoder.residual_norm(x.to(kind), w.to(kind), bias=b.to(kind), kind="layer", residual=torch.zeros_like(x, dtype=kind))
        assert torch.equal(h, x.to(kind)) and torch.equal(y, b.to(kind).expand(rows, width))


# ---- what is refused -------------------------------------------------------------------------

def test_tensors_with_a_gradient_or_a_tangent_are_refused():
    gen = torch.Generator().manual_seed(1)
    r, g, d = (t.cuda() for t in layer(gen, 4, 64, 32, BF16))
    x, w, bias = normal(gen, (3, 64), BF16).cuda(), torch.ones(64, dtype=BF16, device="cuda"), torch.zeros(4, device="cuda")
    logits, u, k = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda"), torch.ones(3, device="cuda")
    experts = decoder.MoEWeights(r, g, d, top_k=2)
    norm = lambda **t: decoder.residual_norm(**dict(dict(x=x, weight=w, bias=w, residual=x, post_weight=w, post_bias=w, gate=x), **t))
    calls = [(lambda t, n=n: norm(**{n: t}), s) for n, s in (("x", x), ("weight", w), ("bias", w), ("residual", x), ("post_weight", w), ("post_bias", w), ("gate", x),
                                                             ("gate", w), ("out", x), ("residual_out", x))]
    calls += [(lambda t: decoder.moe(t, experts), x), (lambda t: decoder.moe(x, experts, out=t), x), (lambda t: decoder.MoEWeights(r, g, d, top_k=2, selection_bias=t), bias),
              (lambda t: decoder.MoEWeights(t, g, d, top_k=2), r), (lambda t: decoder.MoEWeights(r, t, d, top_k=2), g), (lambda t: decoder.MoEWeights(r, g, t, top_k=2), d)]
    calls += [(lambda t: decoder.sample(t, u), logits), (lambda t: decoder.sample(logits, t), u)]
    calls += [(lambda t, n=n: decoder.sample(logits, u, **{n: t}), k) for n in ("temperature", "top_p", "min_p")]
    for i, (call, t) in enumerate(calls):
        call(t.clone())
        with pytest.raises(B200NotSupportedError, match="gradient"):
            call(t.clone().requires_grad_())
            pytest.fail(f"call {i} was accepted")
        with torch.no_grad():
            call(t.clone().requires_grad_())
        with forward_ad.dual_level(), pytest.raises(B200NotSupportedError, match="tangent"):
            call(forward_ad.make_dual(t.clone(), torch.ones_like(t)))
            pytest.fail(f"call {i} was accepted")
    with torch.no_grad():
        late = decoder.MoEWeights(r, g, d, top_k=2, selection_bias=bias.clone().requires_grad_())
    with pytest.raises(B200NotSupportedError, match="gradient"):
        decoder.moe(x, late)
