"""Host side of the decoder-layer operators (no GPU needed): the rotary frequency tables against their
formulas, the phases' exactness, and every refusal of the C entry points that is decided before a
device is touched."""
import ctypes as C
import math

import numpy as np
import pytest

from shorokoo_b200 import B200ArgumentError, _native
from shorokoo_b200 import decoder

L = _native.lib()
PTR = 1 << 20   # an address that the checks look at and nothing reads


def _frequencies(r, base, scaling, factor=1.0, context=0.0, fast=32.0, slow=1.0):
    out, mag = (C.c_double * max(1, r // 2))(), C.c_double()
    st = L.sb_rotary_frequencies(r, base, scaling, factor, context, fast, slow, out, C.byref(mag))
    return st, list(out), mag.value


def test_frequencies_follow_their_formulas():
    r, base = 64, 10000.0
    plain = [base ** (-2 * i / r) for i in range(r // 2)]
    st, f, m = _frequencies(r, base, 0)
    assert st == 0 and m == 1.0
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    np.testing.assert_allclose(_frequencies(r, base, 1, 4.0)[1], np.array(plain) / 4, rtol=1e-14)
    np.testing.assert_allclose(_frequencies(r, base, 2, 4.0)[1],
                               [(base * 4.0 ** (r / (r - 2))) ** (-2 * i / r) for i in range(r // 2)], rtol=1e-13)
    st, f, m = _frequencies(r, base, 3, 8.0, 4096.0)
    assert math.isclose(m, 0.1 * math.log(8.0) + 1)
    turns = 4096 * np.array(plain) / (2 * math.pi)
    assert turns[0] > 32 and turns[-1] < 1
    for fi, p, t in zip(f, plain, turns):
        if t >= 32:
            assert math.isclose(fi, p, rel_tol=1e-14)
        elif t <= 1:
            assert math.isclose(fi, p / 8, rel_tol=1e-14)
        else:
            share = (t - 1) / 31
            assert math.isclose(fi, p * share + p / 8 * (1 - share), rel_tol=1e-13)


@pytest.mark.parametrize("args", [
    (0, 1e4, 0), (7, 1e4, 0), (-2, 1e4, 0), (8, 0.0, 0), (8, math.inf, 0), (8, 1e4, 4), (8, 1e4, 1, 0.0), (2, 1e4, 2, 4.0),
    (8, 1e4, 3, 8.0, 0.0), (8, 1e4, 3, 0.5, 4096.0), (8, 1e4, 3, 8.0, 4096.0, 1.0, 2.0), (8, 1e4, 1, math.nan)])
def test_frequencies_refuse(args):
    assert _frequencies(*args)[0] == 1
    assert "sb_rotary_frequencies" in L.sb_last_error().decode()


def test_phases_keep_far_angles():
    """phase * position modulo 2^64 is the angle in turns: off by at most half a unit of the phase per
    position plus the frequency's own rounding (2^-53 relative), here against exact integers."""
    from fractions import Fraction
    freqs = [1.0, 0.37, 1e-4, 5e-7, 2 * math.pi * 0.75, -0.37]
    ph = (C.c_uint64 * len(freqs))()
    assert L.sb_rotary_phases((C.c_double * len(freqs))(*freqs), len(freqs), ph) == 0
    # 2 pi to 40 digits, as a fraction
    two_pi = 2 * Fraction(31415926535897932384626433832795028841972, 10 ** 40)
    for f, p in zip(freqs, ph):
        for pos in (1, 4095, 1_000_000, (1 << 31) - 1):
            want = Fraction(f) * pos / two_pi
            got = Fraction(int(p) * pos, 1 << 64)
            d = (got - want) % 1
            assert min(d, 1 - d) <= pos * Fraction(1, 1 << 63), (f, pos)
    for bad in (math.nan, math.inf):
        assert L.sb_rotary_phases((C.c_double * 1)(bad), 1, ph) == 1
    assert L.sb_rotary_phases(None, 1, ph) == 1 and L.sb_rotary_phases((C.c_double * 1)(1.0), 0, ph) == 1


def test_table_object_on_the_host():
    t = decoder.RotaryTable(8, 10000.0, device="cpu", interleaved=True)
    assert t.frequencies == [1.0, 0.1, 0.01, 0.001] and t._c.pairs == 4 and t._c.interleaved == 1
    f = decoder.RotaryTable.from_frequencies([0.5, 0.25], magnitude=1.5, device="cpu")
    assert f._c.magnitude == 1.5 and f._c.pairs == 2
    with pytest.raises(B200ArgumentError):
        decoder.RotaryTable(8, scaling="other", device="cpu")
    with pytest.raises(B200ArgumentError):
        decoder.RotaryTable(7, device="cpu")
    with pytest.raises(B200ArgumentError):
        decoder.RotaryTable.from_frequencies([], device="cpu")


def _heads(ptr=PTR, ts=512, hs=64):
    return _native.Heads(ptr, ts, hs)


def _cache(**kw):
    d = dict(k=PTR, v=PTR, k_page_stride=4096, k_token_stride=256, k_head_stride=64, v_page_stride=4096, v_token_stride=256,
             v_head_stride=64, page_table=PTR, context_lengths=PTR, page_table_stride=8, pages=16, elem_type=16, page_size=16,
             max_pages=8, batch=2, kv_heads=4, head_dim=64)
    d.update(kw)
    return _native.PagedCache(**d)


def _table(**kw):
    d = dict(phases=PTR, pairs=32, interleaved=0, magnitude=1.0)
    d.update(kw)
    return _native.RotaryTable(**d)


def _rotary(x=None, y=None, elem=16, tokens=3, heads=8, dim=64, pos=PTR, table=None):
    x, y, table = x or _heads(), y or _heads(), table or _table()
    return L.sb_rotary(C.byref(x), C.byref(y), elem, tokens, heads, dim, pos, 1, C.byref(table), 0, None)


@pytest.mark.parametrize("kw,status", [
    (dict(elem=11), 2), (dict(elem=6), 2), (dict(tokens=-1), 1), (dict(tokens=(1 << 30) + 1), 1), (dict(dim=62), 1),
    (dict(heads=-1), 1), (dict(pos=None), 1), (dict(pos=PTR + 4), 1), (dict(x=_heads(0)), 1), (dict(y=_heads(PTR + 1)), 1),
    (dict(table=_table(phases=0)), 1), (dict(table=_table(pairs=0)), 1), (dict(table=_table(interleaved=2)), 1),
    (dict(x=_heads(ts=1 << 41)), 1), (dict(table=_table(pairs=5000), dim=10000), 2)])
def test_rotary_refuses(kw, status):
    assert _rotary(**kw) == status, L.sb_last_error()
    assert L.sb_last_error().decode().startswith("sb_rotary:")


def test_rotary_of_nothing_is_fine():
    assert _rotary(tokens=0) == 0 and _rotary(heads=0) == 0


BAD_CACHES = [(dict(elem_type=1), 2), (dict(elem_type=0), 2), (dict(page_size=0), 1), (dict(kv_heads=0), 1), (dict(head_dim=0), 1),
              (dict(batch=-1), 1), (dict(pages=-1), 1), (dict(max_pages=-1), 1), (dict(max_pages=1 << 28), 1), (dict(k=None), 1),
              (dict(page_table=None), 1), (dict(context_lengths=None), 1), (dict(context_lengths=PTR + 2), 1),
              (dict(k_page_stride=1 << 41), 1), (dict(pages=1 << 31), 1)]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_cache_is_checked_by_both(kw, status):
    c, h, t = _cache(**kw), _heads(), _table()
    assert L.sb_paged_append(C.byref(c), C.byref(h), C.byref(h), C.byref(h), C.byref(h), 8, 3, PTR, C.byref(t), None) == status
    assert L.sb_paged_attention(C.byref(c), C.byref(h), C.byref(h), 8, 3, PTR, 0.125, 0, PTR, 1 << 40, None) == status


def test_append_refuses():
    c, h, t = _cache(), _heads(), _table()
    def append(c=c, k=h, v=h, q=h, o=h, heads=8, tokens=3, starts=PTR, table=t):
        r = lambda x: None if x is None else C.byref(x)
        return L.sb_paged_append(r(c), r(k), r(v), r(q), r(o), heads, tokens, starts, r(table), None)
    assert append(c=None) == 1 and append(k=None) == 1 and append(v=_heads(0)) == 1
    assert append(q=None) == 1 and append(o=None) == 1            # they go together
    assert append(table=None) == 1 and append(heads=0) == 1       # q needs both
    assert append(starts=None) == 1 and append(tokens=-1) == 1
    assert append(table=_table(pairs=33)) == 1
    assert append(k=_heads(PTR + 1)) == 1
    assert append(tokens=0) == 0 and append(c=_cache(batch=0)) == 0


def test_attention_refuses():
    c, h = _cache(), _heads()
    def attend(c=c, q=h, o=h, heads=8, tokens=3, starts=PTR, scale=0.125, window=0, ws=PTR, n=1 << 40):
        return L.sb_paged_attention(C.byref(c), C.byref(q), C.byref(o), heads, tokens, starts, scale, window, ws, n, None)
    assert attend(heads=6) == 1 and attend(heads=0) == 1
    assert attend(c=_cache(head_dim=136)) == 2 and attend(c=_cache(head_dim=60)) == 2
    assert attend(scale=0.0) == 1 and attend(scale=math.nan) == 1 and attend(scale=math.inf) == 1 and attend(window=-1) == 1
    assert attend(q=_heads(PTR + 2)) == 2 and attend(q=_heads(ts=513)) == 2 and attend(o=_heads(hs=4)) == 2
    assert attend(c=_cache(k_token_stride=100)) == 2 and attend(c=_cache(v_page_stride=4100)) == 2
    assert attend(c=_cache(k=PTR + 8)) == 2
    assert attend(q=_heads(0)) == 1 and attend(starts=None) == 1 and attend(tokens=-1) == 1
    assert attend(tokens=0) == 0 and attend(c=_cache(batch=0)) == 0
    assert attend(tokens=1 << 30, heads=32) == 1
    n = C.c_size_t()
    assert L.sb_paged_attention_workspace(C.byref(c), 8, 3, None) == 1
    assert L.sb_paged_attention_workspace(None, 8, 3, C.byref(n)) == 1


@pytest.mark.parametrize("tokens,heads", [((1 << 28) - 4, 32), ((1 << 27) + 1, 32), ((1 << 30), 8)])
def test_attention_refuses_rows_that_its_counters_cannot_hold(tokens, heads):
    c, h, n = _cache(), _heads(), C.c_size_t()
    assert L.sb_paged_attention(C.byref(c), C.byref(h), C.byref(h), heads, tokens, PTR, 0.125, 0, PTR, 1 << 40, None) == 1
    assert b"2^30" in L.sb_last_error()
    assert L.sb_paged_attention_workspace(C.byref(c), heads, tokens, C.byref(n)) == 1


def test_the_most_negative_stride_is_out_of_range():
    """Its magnitude does not fit 64 bits."""
    low, c, h = -(1 << 63), _cache(), _heads()
    for bad in (_heads(ts=low), _heads(hs=low)):
        assert _rotary(x=bad) == 1 and _rotary(y=bad) == 1
        assert L.sb_paged_append(C.byref(c), C.byref(bad), C.byref(h), None, None, 0, 3, PTR, None, None) == 1
        assert L.sb_paged_attention(C.byref(c), C.byref(bad), C.byref(h), 8, 3, PTR, 0.125, 0, PTR, 1 << 40, None) == 1
    for name in ("k_page_stride", "k_token_stride", "k_head_stride", "v_page_stride", "v_token_stride", "v_head_stride",
                 "page_table_stride"):
        bad = _cache(**{name: low})
        assert L.sb_paged_attention(C.byref(bad), C.byref(h), C.byref(h), 8, 3, PTR, 0.125, 0, PTR, 1 << 40, None) == 1, name
    for xs, ys in ((low, 48), (200, low)):
        assert L.sb_linear_w4(C.byref(_weights()), PTR, xs, None, PTR, ys, 2, None) == 1


@pytest.mark.parametrize("bad", [_heads(ts=0), _heads(hs=0), _heads(ts=56), _heads(hs=-56), _heads(ts=-8, hs=512)],
                         ids=["tokens on one", "heads on one", "tokens", "heads", "tokens backwards"])
def test_results_whose_rows_overlap_are_refused(bad):
    c, h, t = _cache(), _heads(), _table()
    assert _rotary(y=bad) == 1 and b"overlap" in L.sb_last_error()
    assert L.sb_paged_append(C.byref(c), C.byref(h), C.byref(h), C.byref(h), C.byref(bad), 8, 3, PTR, C.byref(t), None) == 1
    assert b"overlap" in L.sb_last_error()
    assert L.sb_paged_attention(C.byref(c), C.byref(h), C.byref(bad), 8, 3, PTR, 0.125, 0, PTR, 1 << 40, None) == 1
    assert b"overlap" in L.sb_last_error()


def _weights(**kw):
    d = dict(data=PTR, elem_type=16, group_size=64, out_features=48, in_features=200, has_zeros=0)
    d.update(kw)
    return _native.W4Weights(**d)


def test_w4_layout_bytes():
    """Tiles of 16 x 64 codes (512 bytes), then 16 scales per tile and group, then as many zero bytes,
    groups in whole eights."""
    n = C.c_size_t()
    assert L.sb_w4_layout_bytes(C.byref(_weights()), C.byref(n)) == 0
    assert n.value == 3 * 4 * 512 + 3 * 8 * 32
    assert L.sb_w4_layout_bytes(C.byref(_weights(has_zeros=1, out_features=49)), C.byref(n)) == 0
    assert n.value == 4 * 4 * 512 + 4 * 8 * 32 + 4 * 8 * 16


@pytest.mark.parametrize("kw,status", [
    (dict(elem_type=1), 2), (dict(group_size=0), 2), (dict(group_size=48), 2), (dict(group_size=-32), 2), (dict(out_features=0), 1),
    (dict(in_features=0), 1), (dict(out_features=1 << 31), 1)])
def test_w4_weights_are_checked(kw, status):
    w, n = _weights(**kw), C.c_size_t()
    assert L.sb_w4_layout_bytes(C.byref(w), C.byref(n)) == status
    assert L.sb_w4_layout(C.byref(w), PTR, 100, PTR, None, PTR, None) == status
    assert L.sb_linear_w4(C.byref(w), PTR, 200, None, PTR, 48, 1, None) == status


def test_w4_refuses():
    w = _weights()
    def layout(w=w, packed=PTR, row=100, scales=PTR, zeros=None, data=PTR):
        return L.sb_w4_layout(C.byref(w), packed, row, scales, zeros, data, None)
    assert layout(packed=None) == 1 and layout(scales=None) == 1 and layout(data=None) == 1 and layout(data=PTR + 16) == 1
    assert layout(row=99) == 1 and layout(scales=PTR + 1) == 1
    assert layout(zeros=PTR) == 1 and layout(w=_weights(has_zeros=1)) == 1
    def linear(w=w, x=PTR, xs=200, bias=None, y=PTR, ys=48, rows=2):
        return L.sb_linear_w4(C.byref(w), x, xs, bias, y, ys, rows, None)
    assert linear(x=None) == 1 and linear(y=None) == 1 and linear(x=PTR + 1) == 1 and linear(bias=PTR + 1) == 1
    assert linear(w=_weights(data=0)) == 1 and linear(w=_weights(data=PTR + 128)) == 1
    assert linear(rows=-1) == 1 and linear(ys=47) == 1 and linear(xs=1 << 41) == 1
    assert linear(rows=0) == 0


def test_tensors_off_the_gpu_are_refused():
    import torch
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pos = torch.zeros(2, dtype=torch.int64)
    t = decoder.RotaryTable(64, device="cpu")
    with pytest.raises(B200ArgumentError, match="CUDA"):
        decoder.rotary(x, pos, t)
    with pytest.raises(B200ArgumentError, match="CUDA"):
        decoder.PagedCache(x[None], x[None], torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(B200ArgumentError, match="CUDA"):
        decoder.W4Weights(torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.float16), in_features=64, group_size=64)


def test_what_autograd_would_have_to_record():
    import torch
    from torch.autograd import forward_ad
    x = torch.ones(3)
    assert not decoder._derived(x) and decoder._derived(x.clone().requires_grad_())
    with torch.no_grad():
        assert not decoder._derived(x.clone().requires_grad_())
    with forward_ad.dual_level():
        assert not decoder._derived(x) and decoder._derived(forward_ad.make_dual(x, x))
        with torch.no_grad():          # which leaves tangents alone
            assert decoder._derived(forward_ad.make_dual(x, x))
    seen = []
    torch.func.jvp(lambda z: (seen.append(decoder._derived(z)), z)[1], (x,), (x,))
    torch.func.grad(lambda z: (seen.append(decoder._derived(z)), z.sum())[1])(x)
    assert seen == [True, True]
