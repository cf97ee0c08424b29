"""GPU tests of the decoder-layer operators where they can go wrong at the edges: weights far below a
row's largest, non-finite values over long walks, waits that run out, gradients
that the operators do not record, index arrays that no caller should pass. Formulas, caches and tolerances are those of test_gpu_decoder.py."""
import math
import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from shorokoo_b200 import B200ArgumentError, B200NotSupportedError, decoder
from test_gpu_decoder import BF16, FP16, U, Paged, attended, half, normal, within

pytestmark = pytest.mark.gpu


# ---- softmax weights far below the largest -----------------------------------------------------

def given_logits(logits, values, new, dtype, page=16):
    """A cache of one key head of 64 whose keys give logit j at scale 1 for queries (1, 0, 0, ..), and the queries
    of its last `new` tokens."""
    p = Paged([new], [len(logits)], 1, 64, page, dtype, poison=False)
    j = torch.arange(len(logits))
    at = p.table[0][j // page].long(), j % page
    p.k.zero_()
    p.k[at[0], at[1], 0, 0] = logits.to(dtype)
    p.v[at[0], at[1], 0] = values.to(dtype)
    q = torch.zeros(new, 1, 64, dtype=dtype)
    q[:, :, 0] = 1
    return p, q


def fp16_weights(p, q, block):
    """What fp16 weights add to the tolerance of `attended` at scale 1. A block of positions is weighted against
    one reference, by which its largest weight becomes 2^-2 or more, and 2^11 or more where it is the largest of
    the row; fp16 below 2^-14 is off by up to 2^-25."""
    c, n = p.context[0], p.new[0]
    k, v, _ = p.gather(0)
    s = k[:, 0] @ q[0, 0].double()
    more = torch.zeros(n, 1, 64, dtype=torch.float64)
    for i in range(n):
        w = torch.softmax(s[: c - n + i + 1], 0)
        mass = v[: len(w), 0].abs()
        for a in range(0, len(w), block):
            top = w[a: a + block].max()
            off = 2.0 ** -25 / (2.0 ** 11 if top == w.max() else 2.0 ** -2)
            more[i, 0] += off * top * mass[a: a + block].sum(0)
    return more


@pytest.mark.parametrize("new", [1, 40])          # the 16-row kernel's, the tensor core's
@pytest.mark.parametrize("gap,length", [(8, 8000), (14, 8000), (15, 8000), (17, 8000), (19, 30000)])
def test_attention_keeps_a_long_tail_of_small_weights(gap, length, new):
    """A leading position with nothing in its value, as the first of a text often is, and thousands of equal
    ones `gap` nats below it: the result is theirs."""
    gen = torch.Generator().manual_seed(gap)
    logits, values = torch.zeros(length), 1 + 0.25 * torch.randn((length, 64), generator=gen)
    logits[0], values[0] = gap, 0
    p, q = given_logits(logits, values, new, FP16)
    want, tol = attended(p, q, 0, 1.0)
    got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda(), scale=1.0)
    within(got, want, tol + fp16_weights(p, q, 16 if new == 1 else 64), f"gap {gap}")


@pytest.mark.parametrize("new,dtype", [(1, FP16), (40, FP16), (1, BF16), (40, BF16)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_attention_follows_levels_up_and_down(seed, new, dtype):
    """Stretches of positions at four levels down to 19 nats, in a random order, with values that make each
    level's share of the result alike."""
    gen = torch.Generator().manual_seed(seed)
    level = torch.tensor([0.0, -5.0, -12.0, -19.0])[torch.randint(0, 4, (40,), generator=gen)]
    level = level.repeat_interleave(100)
    logits = level + 0.25 * torch.randn(4000, generator=gen)
    values = torch.exp(-level).clamp(max=30000)[:, None] * 2 ** -8 * torch.randn((4000, 64), generator=gen)
    p, q = given_logits(logits, values, new, dtype)
    want, tol = attended(p, q, 0, 1.0)
    if dtype is FP16:
        tol = tol + fp16_weights(p, q, 16 if new == 1 else 64)
    got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda(), scale=1.0)
    within(got, want, tol, f"levels {seed}")


@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_a_split_context_with_a_leading_position(new):
    """The same over a context that is cut over the whole card, so that most pieces do not hold the leader."""
    length = 100003
    gen = torch.Generator().manual_seed(7)
    logits, values = torch.zeros(length), 1 + 0.25 * torch.randn((length, 64), generator=gen)
    logits[5], values[5] = 17.5, 0
    p, q = given_logits(logits, values, new, FP16, page=64)
    want, tol = attended(p, q, 0, 1.0)
    got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda(), scale=1.0)
    within(got, want, tol + fp16_weights(p, q, 16 if new == 1 else 64), "split")


# ---- many items to a CTA -------------------------------------------------------------------------

def attended_in_order(p, q):
    """`attended` without window or missing pages, whole sequences at a time."""
    want, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    h, d = half(q.dtype), q.shape[2]
    for b, n in enumerate(p.new):
        k, v, _ = p.gather(b)
        rows, c = slice(int(p.starts[b]), int(p.starts[b]) + n), p.context[b]
        seen = torch.arange(c) <= torch.arange(c - n, c)[:, None]
        for x in range(q.shape[1]):
            qx, kx, vx = (y.double() for y in (q[rows, x], k[:, x * p.kv // q.shape[1]], v[:, x * p.kv // q.shape[1]]))
            w = torch.softmax((qx @ kx.t() * d ** -0.5).masked_fill(~seen, -math.inf), 1)
            delta = (d + 4) * U * (qx.abs() @ kx.abs().t()).amax(1, keepdim=True) * d ** -0.5
            want[rows, x] = w @ vx
            tol[rows, x] = h * want[rows, x].abs() + (h + 2 * delta + (c / 16 + 32) * U) * (w @ vx.abs())
    return want, tol


@pytest.mark.parametrize("page", [16, 24])      # copied whole, gathered
def test_nonfinite_values_in_some_of_many_short_items(page):
    """About ten items per CTA, most of which leave its second row tile without keys, every third with a NaN among
    the new tokens' own values: it reaches the tokens after it in its sequence, no other row."""
    new = [150 if b % 9 == 0 else 40 for b in range(1500)]
    p = Paged(new, new, 1, 64, page, BF16, seed=5, poison=False)
    q = normal(torch.Generator().manual_seed(6), (sum(new), 1, 64), BF16)
    want, tol = attended_in_order(p, q)
    lost = torch.zeros(q.shape, dtype=torch.bool)
    for b in range(0, len(new), 3):
        at = new[b] // 2
        p.v[p.table[b, at // page], at % page, 0, 3] = math.nan
        lost[int(p.starts[b]) + at: int(p.starts[b]) + new[b], 0, 3] = True
    got = decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda()).double().cpu()
    assert torch.equal(torch.isnan(got), lost)
    within(got[~lost], want[~lost], tol[~lost], "items")


# ---- waits that run out --------------------------------------------------------------------------

RUN_OUT = """
import torch
from shorokoo_b200 import B200InvalidOperationError, decoder
from test_gpu_decoder import BF16, Paged, attended, normal, within
for page in (16, 24):                     # copied whole, gathered
    for new, context in (([300, 40, 200], [3000, 40, 900]), ([600], [20000])):
        p = Paged(new, context, 2, 128, page, BF16, seed=1)
        q = normal(torch.Generator().manual_seed(2), (sum(new) + 2, 4, 128), BF16).cuda()
        cache, starts = p.gpu(), p.starts.cuda()
        out = torch.full(q.shape, 5.0, dtype=BF16, device="cuda")
        decoder.paged_attention(cache, q, starts, out=out)
        try:
            decoder.check()
            raise SystemExit("no wait ran out")
        except B200InvalidOperationError as e:
            assert "timed out" in str(e), e
        decoder.check()                   # reported once
        rows = out[: sum(new)]
        lost = torch.isnan(rows).any(2) | (rows == 5.0).all(2)
        assert lost.any() and (out[sum(new):] == 5.0).all()
        if sum(context) < 10000:          # rows that were done before are right
            want, tol = attended(p, q.cpu())
            keep = ~lost.cpu()
            within(rows.cpu()[keep], want[: sum(new)][keep], tol[: sum(new)][keep], "kept")
p = Paged([1, 1], [900, 70], 2, 128, 16, BF16)      # the device goes on
q = normal(torch.Generator().manual_seed(2), (2, 4, 128), BF16)
want, tol = attended(p, q)
within(decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda()), want, tol, "after")
decoder.check()
print("ran out and went on")
"""


def test_waits_that_run_out_are_reported_and_end():
    """With a limit of a nanosecond every wait that is not over at once runs out: the call returns, its rows are NaN
    or not written, and the status says so once."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, SHOROKOO_B200_WAIT_NS="1", PYTHONPATH=os.pathsep.join([os.path.dirname(here), here]))
    r = subprocess.run([sys.executable, "-c", RUN_OUT], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ran out and went on" in r.stdout, r.stdout + r.stderr


# ---- gradients that are not recorded ------------------------------------------------------------

def small_layer():
    packed = torch.zeros(8, 32, dtype=torch.uint8, device="cuda")
    w = decoder.W4Weights(packed, torch.ones(8, 1, dtype=BF16, device="cuda"), in_features=64, group_size=64)
    p = Paged([2], [20], 2, 64, 16, BF16, poison=False)
    zeros = lambda *shape: torch.zeros(*shape, dtype=BF16, device="cuda")
    return dict(w=w, cache=p.gpu(), starts=p.starts.cuda(), table=decoder.RotaryTable(64, device="cuda"), x=zeros(2, 64),
                bias=zeros(8), q=zeros(2, 4, 64), k=zeros(2, 2, 64), v=zeros(2, 2, 64), pos=torch.zeros(2, dtype=torch.int64, device="cuda"))


CALLS = {
    "linear_w4 x": ("x", lambda s, t: decoder.linear_w4(t, s["w"])),
    "linear_w4 bias": ("bias", lambda s, t: decoder.linear_w4(s["x"], s["w"], t)),
    "linear_w4 out": ("y", lambda s, t: decoder.linear_w4(s["x"], s["w"], out=t)),
    "rotary x": ("q", lambda s, t: decoder.rotary(t, s["pos"], s["table"])),
    "rotary out": ("q", lambda s, t: decoder.rotary(s["q"], s["pos"], s["table"], out=t)),
    "append k": ("k", lambda s, t: decoder.paged_append(s["cache"], t, s["v"], s["starts"])),
    "append v": ("v", lambda s, t: decoder.paged_append(s["cache"], s["k"], t, s["starts"])),
    "append q": ("q", lambda s, t: decoder.paged_append(s["cache"], s["k"], s["v"], s["starts"], q=t, table=s["table"])),
    "append out": ("q", lambda s, t: decoder.paged_append(s["cache"], s["k"], s["v"], s["starts"], q=s["q"], table=s["table"], out=t)),
    "attention q": ("q", lambda s, t: decoder.paged_attention(s["cache"], t, s["starts"])),
    "attention out": ("q", lambda s, t: decoder.paged_attention(s["cache"], s["q"], s["starts"], out=t)),
}


@pytest.mark.parametrize("name", CALLS)
def test_tensors_that_require_a_gradient_are_refused(name):
    """Every tensor argument, and the same call without recording, which has to pass."""
    s = small_layer()
    s["y"] = torch.zeros(2, 8, dtype=BF16, device="cuda")
    which, call = CALLS[name]
    t = s[which].clone().requires_grad_()
    with pytest.raises(B200NotSupportedError, match="gradient"):
        call(s, t)
    with torch.no_grad():
        call(s, t)
    call(s, t.detach())


@pytest.mark.parametrize("name", [n for n in CALLS if not n.endswith("out")])
def test_arguments_that_are_no_tensors_are_refused(name):
    s = small_layer()
    for t in (1.0, [0.0] * 8):
        with pytest.raises(B200ArgumentError):
            CALLS[name][1](s, t)


@pytest.mark.parametrize("name", CALLS)
def test_tensors_with_a_tangent_are_refused(name):
    """Forward-mode derivatives, by a dual tensor and by torch.func.jvp."""
    s = small_layer()
    s["y"] = torch.zeros(2, 8, dtype=BF16, device="cuda")
    which, call = CALLS[name]
    t = s[which]
    with forward_ad.dual_level():
        with pytest.raises(B200NotSupportedError, match="tangent"):
            call(s, forward_ad.make_dual(t.clone(), torch.ones_like(t)))
        call(s, t)
    with pytest.raises(B200NotSupportedError, match="tangent"):
        torch.func.jvp(lambda z: call(s, z), (t.clone(),), (torch.ones_like(t),))


@pytest.mark.parametrize("which", ["k_pages", "v_pages"])
def test_pages_that_require_a_gradient_later_are_refused(which):
    s = small_layer()
    getattr(s["cache"], which).requires_grad_()
    calls = (lambda: decoder.paged_attention(s["cache"], s["q"], s["starts"]),
             lambda: decoder.paged_append(s["cache"], s["k"], s["v"], s["starts"]))
    for call in calls:
        with pytest.raises(B200NotSupportedError, match="gradient"):
            call()
        with torch.no_grad():
            call()


def test_objects_of_another_kind_are_refused():
    s = small_layer()
    for call in (lambda: decoder.linear_w4(s["x"], s["x"]), lambda: decoder.paged_attention(s["w"], s["q"], s["starts"]),
                 lambda: decoder.paged_append(None, s["k"], s["v"], s["starts"]), lambda: decoder.rotary(s["q"], s["pos"], s["w"])):
        with pytest.raises(B200ArgumentError):
            call()


# ---- sequences of many row tiles -----------------------------------------------------------------

@pytest.mark.parametrize("new,heads,kv", [
    ([1] * 60 + [600] + [1] * 60, 2, 2),      # 38 row tiles in the 16-row kernel
    ([4200, 30], 4, 2),                       # 33 in the tensor core's
])
def test_attention_of_sequences_with_more_row_tiles_than_a_warp_has_lanes(new, heads, kv):
    context = [n + 37 for n in new]
    p = Paged(new, context, kv, 64, 16, BF16, seed=9)
    q = normal(torch.Generator().manual_seed(6), (sum(new), heads, 64), BF16)
    want, tol = attended_in_order(p, q)
    within(decoder.paged_attention(p.gpu(), q.cuda(), p.starts.cuda()), want, tol, "tiles")


# ---- index arrays that no caller should pass ------------------------------------------------------

GUARD = 1 << 16    # bytes on either side


def guarded(shape, dtype, fill):
    """A tensor in the middle of a buffer, and a check that the buffer around it is as it was."""
    n = math.prod(shape) * dtype.itemsize
    whole = torch.full((n + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
    inner = whole[GUARD: GUARD + n].view(dtype).view(shape)
    if fill is not None:
        inner.copy_(fill)

    def untouched():
        assert (whole[:GUARD] == 0xA5).all() and (whole[GUARD + n:] == 0xA5).all()
    return inner, untouched


@pytest.mark.parametrize("tokens", [3, 200])          # the 16-row kernel's, the tensor core's
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("starts,context", [
    ((0, -5, 1.0), (40, 30)), ((0.7, 0, 0.3), (300, 30)), ((0, 100, 0.5), (40, 400)), ((1.0, 1.0, 1.0), (40, 30)),
    ((5, 1, 1.0), (40, 30)), ((0, 0.5, 1.0), (-3, (1 << 31) - 1)), ((-(1 << 31), (1 << 31) - 1, 7), (1 << 30, 1)),
])
def test_index_arrays_out_of_order_write_nothing_outside(tokens, page, starts, context):
    """Row starts that decrease or leave the rows, contexts that no table holds, table entries of any value: what
    surrounds the result, the pages and the workspace stays as it was, and so does a page that no entry names."""
    p = Paged([1, 1], [40, 30], 2, 64, page, BF16, poison=False, width=6)
    p.table[0, 4], p.table[1, 4:] = 1 << 30, -(1 << 31)
    named = set(int(x) for x in p.table.flatten() if 0 <= x < p.pages)
    gen = torch.Generator().manual_seed(3)
    q, k, v = (normal(gen, (tokens, x, 64), BF16).cuda() for x in (4, 2, 2))
    s = torch.tensor([int(x * tokens) if isinstance(x, float) else x for x in starts], dtype=torch.int32).cuda()
    kp, k_untouched = guarded(p.k.shape, BF16, p.k)
    vp, v_untouched = guarded(p.v.shape, BF16, p.v)
    out, out_untouched = guarded(q.shape, BF16, torch.zeros(q.shape))
    cache = decoder.PagedCache(kp, vp, p.table.cuda(), torch.tensor(context, dtype=torch.int32).cuda())
    decoder.paged_append(cache, k, v, s, q=q, table=decoder.RotaryTable(64, device="cuda"), out=out)
    n = cache._workspace(4, tokens)
    space, space_untouched = guarded((n,), torch.uint8, None)
    qh, oh = (cache._rows(x, "rows", 4, tokens)[2] for x in (q, out))
    for window in (0, 20):
        decoder._call("sb_paged_attention", cache.device, cache._ref, qh, oh, 4, tokens, s.data_ptr(), 0.125, window,
                      space.data_ptr(), n)
    for check in (k_untouched, v_untouched, out_untouched, space_untouched):
        check()
    for page_no in set(range(p.pages)) - named:
        assert torch.equal(kp[page_no].cpu(), p.k[page_no]) and torch.equal(vp[page_no].cpu(), p.v[page_no])
    decoder.check()
