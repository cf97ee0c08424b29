"""Host side of the residual norms, mixture-of-experts layers and sampling (no GPU needed): what the C entry points
refuse before a device is touched, calls without rows, and workspace sizes."""
import ctypes as C
import math

import pytest

from shorokoo_b200 import B200ArgumentError, _native, decoder

L = _native.lib()
PTR = 1 << 20   # an address that the checks look at and nothing reads


def _norm(**kw):
    d = dict(x=PTR, residual=PTR, gate=None, sum=PTR, y=PTR + 4096, x_row_stride=64, residual_row_stride=64, gate_row_stride=0,
             sum_row_stride=64, y_row_stride=64, weight=PTR, bias=None, post_weight=None, post_bias=None, rows=3, width=64, elem_type=16,
             sum_type=16, weight_type=16, layer_norm=0, scale=1.0, eps=1e-6, weight_offset=0.0)
    d.update(kw)
    return L.sb_residual_norm(C.byref(_native.ResidualNorm(**d)), None)


@pytest.mark.parametrize("kw,status", [
    (dict(elem_type=11), 2), (dict(sum_type=10), 1), (dict(weight_type=10), 1), (dict(rows=-1), 1), (dict(rows=(1 << 30) + 1), 1),
    (dict(width=0), 1), (dict(width=32769), 2), (dict(scale=math.nan), 1), (dict(eps=-1e-9), 1), (dict(eps=math.inf), 1),
    (dict(weight_offset=math.inf), 1), (dict(y=None, sum=None, weight=None), 1), (dict(y=None), 1), (dict(weight=None), 1),
    (dict(y=None, weight=None, bias=PTR), 1), (dict(post_bias=PTR), 1), (dict(x=None), 1), (dict(y=PTR), 1), (dict(x=PTR + 1), 1),
    (dict(sum=PTR + 1), 1), (dict(sum_type=1, sum=PTR + 2), 1), (dict(weight_type=1, weight=PTR + 2), 1), (dict(gate=PTR + 1), 1),
    (dict(x_row_stride=1 << 41), 1), (dict(gate_row_stride=-(1 << 63)), 1), (dict(y_row_stride=63), 1), (dict(y_row_stride=0), 1),
    (dict(sum_row_stride=-63), 1)])
def test_residual_norm_refuses(kw, status):
    assert _norm(**kw) == status, L.sb_last_error()
    assert L.sb_last_error().decode().startswith("sb_residual_norm:")


def test_residual_norm_of_nothing_is_fine():
    assert _norm(rows=0) == 0 and _norm(rows=0, x=None) == 0
    assert L.sb_residual_norm(None, None) == 1


def _weights(**kw):
    d = dict(router=PTR, gate_up=PTR, down=PTR, selection_bias=None, router_row_stride=64, gate_up_expert_stride=4096, gate_up_row_stride=64,
             down_expert_stride=2048, down_row_stride=32, experts=8, width=64, inner=32, elem_type=16, router_type=16, top_k=2, scoring=0,
             normalize=1, activation=0, scale=1.0)
    d.update(kw)
    return _native.MoEWeights(**d)


@pytest.mark.parametrize("kw,status", [
    (dict(elem_type=1), 2), (dict(router_type=10), 1), (dict(experts=0), 1), (dict(experts=513), 2), (dict(width=0), 1), (dict(width=60), 2),
    (dict(inner=36), 2), (dict(inner=1 << 20), 2), (dict(top_k=0), 1), (dict(top_k=9), 1), (dict(top_k=33, experts=64), 2), (dict(scoring=2), 1),
    (dict(activation=-1), 1), (dict(scale=math.inf), 1), (dict(router=None), 1), (dict(gate_up=None), 1), (dict(down=None), 1),
    (dict(router=PTR + 2), 2), (dict(gate_up=PTR + 8), 2), (dict(selection_bias=PTR + 2), 1), (dict(gate_up_row_stride=65), 2),
    (dict(down_expert_stride=4), 2), (dict(down_row_stride=1 << 41), 1), (dict(router_row_stride=-(1 << 63)), 1)])
def test_moe_weights_are_checked_by_both(kw, status):
    w, n = _weights(**kw), C.c_size_t()
    assert L.sb_moe_workspace(C.byref(w), 3, C.byref(n)) == status, L.sb_last_error()
    assert L.sb_moe(C.byref(w), PTR, 64, PTR, 64, 3, PTR, 1 << 40, None) == status
    assert L.sb_last_error().decode().startswith("sb_moe:")


def test_moe_refuses():
    w, n = _weights(), C.c_size_t()
    def moe(x=PTR, xs=64, y=PTR, ys=64, tokens=3, ws=PTR, size=1 << 40):
        return L.sb_moe(C.byref(w), x, xs, y, ys, tokens, ws, size, None)
    assert moe(x=None) == 1 and moe(y=None) == 1 and moe(tokens=-1) == 1 and moe(tokens=(1 << 30) + 1) == 1
    assert moe(x=PTR + 8) == 2 and moe(xs=60) == 2 and moe(ys=68) == 2 and moe(xs=1 << 41) == 1
    assert moe(ys=56) == 1 and moe(ys=0) == 1 and moe(ys=-(1 << 63)) == 1
    assert L.sb_moe_workspace(C.byref(w), 3, C.byref(n)) == 0
    assert moe(tokens=0) == 0
    assert L.sb_moe_workspace(C.byref(w), 3, None) == 1 and L.sb_moe_workspace(None, 3, C.byref(n)) == 1
    assert L.sb_moe_workspace(C.byref(w), -1, C.byref(n)) == 1


def test_moe_workspace_does_not_grow_with_the_pieces_of_a_long_call():
    n, sizes = C.c_size_t(), []
    for tokens in (1, 256, 257, 10000, 1 << 30):
        assert L.sb_moe_workspace(C.byref(_weights()), tokens, C.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] <= sizes[1] <= sizes[2] and sizes[2] == sizes[3] == sizes[4]


def _sample(logits=PTR, stride=100, elem=1, rows=3, vocab=100, uniform=PTR, tokens=PTR, by=True, **kw):
    d = dict(temperature_of=None, top_p_of=None, min_p_of=None, top_k_of=None, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
    d.update(kw)
    s = _native.Sampling(**d)
    return L.sb_sample(logits, stride, elem, rows, vocab, uniform, C.byref(s) if by else None, tokens, None)


@pytest.mark.parametrize("kw,status", [
    (dict(elem=11), 2), (dict(rows=-1), 1), (dict(rows=(1 << 26) + 1), 1), (dict(vocab=0), 1), (dict(vocab=(1 << 24) + 1), 2), (dict(by=False), 1),
    (dict(temperature=math.nan), 1), (dict(top_p=math.nan), 1), (dict(min_p=math.nan), 1), (dict(logits=None), 1), (dict(uniform=None), 1),
    (dict(tokens=None), 1), (dict(logits=PTR + 2), 1), (dict(uniform=PTR + 2), 1), (dict(tokens=PTR + 4), 1), (dict(top_k_of=PTR + 2), 1),
    (dict(temperature_of=PTR + 1), 1), (dict(stride=1 << 41), 1)])
def test_sample_refuses(kw, status):
    assert _sample(**kw) == status, L.sb_last_error()
    assert L.sb_last_error().decode().startswith("sb_sample:")


def test_sample_of_nothing_is_fine():
    assert _sample(rows=0) == 0 and _sample(rows=0, logits=None) == 0


def test_tensors_off_the_gpu_are_refused():
    import torch
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(B200ArgumentError, match="CUDA"):
        decoder.residual_norm(x, x[0])
    with pytest.raises(B200ArgumentError, match="CUDA"):
        decoder.MoEWeights(x, x[None], x[None], top_k=1)
    with pytest.raises(B200ArgumentError, match="CUDA"):
        decoder.sample(x, torch.zeros(2))
    with pytest.raises(B200ArgumentError, match="MoEWeights"):
        decoder.moe(x, None)
