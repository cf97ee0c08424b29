"""Decoder-layer operators on device tensors: what a language model runs per step when it answers from a
paged cache (the sb_rotary*, sb_paged_*, sb_*w4*, sb_residual_norm, sb_moe* and sb_sample entry points of the
library's C ABI).

    weights = W4Weights(packed, scales, zeros, in_features=4096, group_size=128)     # once
    table = RotaryTable(128, 500000.0)                                               # once
    cache = PagedCache(k_pages, v_pages, page_table, context_lengths)                # once per step's batch
    qkv = linear_w4(x, weights)
    q = paged_append(cache, k, v, query_starts, q=q, table=table)
    o = paged_attention(cache, q, query_starts)
    y, h = residual_norm(linear_w4(o.flatten(1), projection), weight, residual=h)
    experts = MoEWeights(router, gate_up, down, top_k=8)                             # once
    y, h = residual_norm(moe(y, experts), weight, residual=h)
    tokens = sample(linear_w4(y, head), uniform, temperature=0.7, top_p=0.9)

Tensors are torch CUDA tensors. Every call enqueues its kernels on torch's current stream of the
tensors' device and returns; nothing waits, and results are new tensors of torch's allocator unless
``out`` is given, so calls can be captured into CUDA graphs and run on several streams. The operators
compute no autograd graph and no tangents, and refuse tensors that require either. Errors are the backend's
(``B200ArgumentError`` and so on).
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _native
from .backend import B200ArgumentError, B200NotSupportedError, _check

_ELEM = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "by_parts": 3}
_fn = {}


def _call(name: str, device: torch.device, *args) -> None:
    """Calls an entry point on the current stream of `device` (its last argument)."""
    f = _fn.get(name)
    if f is None:
        f = _fn[name] = getattr(_native.lib(), name)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        status = f(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = f(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _check(status)


def _bad(msg: str) -> None:
    raise B200ArgumentError(msg)


def _cuda(x, name: str) -> torch.device:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _bad(f"{name} must be a CUDA tensor")
    return x.device


def _derived(x) -> bool:
    """Whether autograd would have to record what is computed from x, backward or forward."""
    return (x.requires_grad and torch.is_grad_enabled()) or (forward_ad._current_level >= 0
                                                             and forward_ad.unpack_dual(x).tangent is not None)


def _on(x, name: str, device: torch.device, dtype: torch.dtype, dims: int) -> None:
    if not isinstance(x, torch.Tensor) or x.device != device:
        _bad(f"{name} must be a tensor on {device}")
    if x.dtype is not dtype:
        _bad(f"{name} must be {dtype}, got {x.dtype}")
    if x.dim() != dims:
        _bad(f"{name} must have {dims} dimensions, got shape {tuple(x.shape)}")
    if _derived(x):
        raise B200NotSupportedError(f"{name} requires a gradient or has a tangent, which these operators do not record")


_pack_heads = struct.Struct("Pqq").pack   # sb_heads


def _heads(x, name: str, device: torch.device, dtype: torch.dtype):
    """(tokens, heads, head_dim, sb_heads) of a [tokens, heads, head_dim] tensor."""
    try:
        tokens, heads, dim = x.shape
        token, head, last = x.stride()
        if x.dtype is dtype and x.get_device() == device.index and (last == 1 or dim == 1) and not _derived(x):
            return tokens, heads, dim, _pack_heads(x.data_ptr(), token, head)
    except (AttributeError, TypeError, ValueError):
        pass
    _on(x, name, device, dtype, 3)
    _bad(f"{name} must be contiguous along its last dimension")


def _starts(x, device: torch.device, batch: int) -> int:
    try:
        if (x.dtype is torch.int32 and x.get_device() == device.index and x.shape == (batch + 1,)
                and (x.stride() == (1,) or batch == 0)):
            return x.data_ptr()
    except AttributeError:
        pass
    _on(x, "query_starts", device, torch.int32, 1)
    _bad(f"query_starts must be {batch + 1} contiguous values, got {tuple(x.shape)}")


class RotaryTable:
    """Rotary frequencies of the first ``rotary_dim`` elements of a head, on ``device``.

    ``interleaved`` pairs elements (2i, 2i + 1), otherwise (i, i + rotary_dim / 2). ``scaling`` for
    contexts ``factor`` times the trained one: "linear" divides every frequency by factor, "ntk"
    multiplies base by factor^(r / (r - 2)), "by_parts" keeps pairs that turn more than beta_fast times
    in original_context positions, divides those below beta_slow turns by factor, mixes those between
    linearly in their turns and multiplies rotated values by 0.1 ln(factor) + 1. Checkpoints whose scaling
    mixes linearly in the pair's index need ``from_frequencies``, which takes any frequencies (radians per
    position)."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, *, interleaved: bool = False, scaling: str = "none",
                 factor: float = 1.0, original_context: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device="cuda"):
        if scaling not in _SCALINGS:
            _bad(f"scaling must be one of {sorted(_SCALINGS)}, got {scaling!r}")
        freqs = (C.c_double * max(1, int(rotary_dim) // 2))()
        magnitude = C.c_double()
        _check(_native.lib().sb_rotary_frequencies(int(rotary_dim), float(base), _SCALINGS[scaling], float(factor),
                                                   float(original_context), float(beta_fast), float(beta_slow), freqs,
                                                   C.byref(magnitude)))
        self._set(list(freqs), interleaved, magnitude.value, device)

    @classmethod
    def from_frequencies(cls, frequencies: Sequence[float], *, interleaved: bool = False, magnitude: float = 1.0,
                         device="cuda") -> "RotaryTable":
        self = cls.__new__(cls)
        self._set([float(f) for f in frequencies], interleaved, float(magnitude), device)
        return self

    def _set(self, freqs, interleaved, magnitude, device) -> None:
        self.frequencies, self.magnitude, self.interleaved = freqs, magnitude, bool(interleaved)
        n = len(freqs)
        phases = (C.c_uint64 * max(1, n))()
        _check(_native.lib().sb_rotary_phases((C.c_double * max(1, n))(*freqs), n, phases))
        signed = [p - (1 << 64) if p >> 63 else p for p in phases]
        self._phases = torch.tensor(signed, dtype=torch.int64).to(device)
        self.device = self._phases.device
        self._c = _native.RotaryTable(self._phases.data_ptr(), n, int(self.interleaved), magnitude)
        self._ref = C.byref(self._c)


def _table(table, device: torch.device):
    if not isinstance(table, RotaryTable):
        _bad("table must be a RotaryTable")
    if table.device != device:
        _bad(f"table is on {table.device}, the tensors on {device}")
    return table._ref


def rotary(x: torch.Tensor, positions: torch.Tensor, table: RotaryTable, inverse: bool = False,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [tokens, heads, head_dim] (float32, float16, bfloat16) with each token turned by its position
    (int32 or int64 [tokens], any sign). ``inverse`` turns back and multiplies by the table's magnitude all
    the same, which is the adjoint: the gradient of x for the gradient of the result. ``out`` may be x
    itself, but not overlap it otherwise."""
    device = _cuda(x, "x")
    dtype = x.dtype
    elem = _ELEM.get(dtype)
    if elem is None:
        raise B200NotSupportedError(f"element type {dtype} is not supported")
    tokens, heads, dim, xh = _heads(x, "x", device, dtype)
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        _bad("positions must be an int32 or int64 tensor")
    if positions.get_device() != device.index or positions.shape != (tokens,) or not positions.is_contiguous():
        _bad(f"positions must be {tokens} contiguous values on {device}, got {tuple(positions.shape)} on {positions.device}")
    if out is None:
        out = torch.empty_like(x)
    t, h, d, yh = _heads(out, "out", device, dtype)
    if t != tokens or h != heads or d != dim:
        _bad(f"out must have shape {tuple(x.shape)}, got {tuple(out.shape)}")
    _call("sb_rotary", device, xh, yh, elem, tokens, heads, dim, positions.data_ptr(), positions.dtype is torch.int64,
          _table(table, device), bool(inverse))
    return out


class PagedCache:
    """A paged cache of keys and values and the step's view of it.

    ``k_pages``, ``v_pages``: [pages, page_size, kv_heads, head_dim] float16 or bfloat16, of any strides
    along the first three dimensions. Position j of sequence b is row j % page_size of page
    ``page_table[b, j // page_size]`` (int32 [batch, max_pages]); ``context_lengths`` (int32 [batch])
    counts each sequence's positions, those of the current step's tokens among them. Positions past
    the table, and those whose table entry is no page, hold nothing: they are not written, and attention
    leaves them out. The object keeps the tensors; their contents may change between calls."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 context_lengths: torch.Tensor):
        device = _cuda(k_pages, "k_pages")
        if k_pages.dtype not in (torch.float16, torch.bfloat16):
            raise B200NotSupportedError(f"cache element type {k_pages.dtype} is not supported")
        _on(k_pages, "k_pages", device, k_pages.dtype, 4)
        _on(v_pages, "v_pages", device, k_pages.dtype, 4)
        _on(page_table, "page_table", device, torch.int32, 2)
        _on(context_lengths, "context_lengths", device, torch.int32, 1)
        if v_pages.shape != k_pages.shape:
            _bad(f"v_pages must have shape {tuple(k_pages.shape)}, got {tuple(v_pages.shape)}")
        batch, width = page_table.shape
        if context_lengths.shape[0] != batch or not context_lengths.is_contiguous():
            _bad(f"context_lengths must be {batch} contiguous values, got {tuple(context_lengths.shape)}")
        for name, p in (("k_pages", k_pages), ("v_pages", v_pages)):
            if p.stride(3) != 1 and p.shape[3] != 1:
                _bad(f"{name} must be contiguous along its last dimension")
        if page_table.stride(1) != 1 and width > 1:
            _bad("page_table must be contiguous along its last dimension")
        self.k_pages, self.v_pages, self.page_table, self.context_lengths = k_pages, v_pages, page_table, context_lengths
        self.device, self.dtype, self.batch = device, k_pages.dtype, batch
        pages, size, self.kv_heads, self.head_dim = k_pages.shape
        ks, vs = k_pages.stride(), v_pages.stride()
        self._c = _native.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                                     page_table.data_ptr(), context_lengths.data_ptr(), page_table.stride(0), pages,
                                     _ELEM[self.dtype], size, width, batch, self.kv_heads, self.head_dim)
        self._ref = C.byref(self._c)
        self._space = {}

    def _workspace(self, heads: int, tokens: int) -> int:
        n = self._space.get((heads, tokens))
        if n is None:
            size = C.c_size_t()
            with torch.cuda.device(self.device):
                _check(_native.lib().sb_paged_attention_workspace(self._ref, heads, tokens, C.byref(size)))
            if len(self._space) > 64:
                self._space.clear()
            n = self._space[(heads, tokens)] = size.value
        return n

    def _rows(self, x, name: str, heads: Optional[int], tokens: Optional[int]):
        """(tokens, heads, sb_heads) of a tensor of the step's rows; None: any number."""
        t, h, d, packed = _heads(x, name, self.device, self.dtype)
        if (tokens is not None and t != tokens) or (heads is not None and h != heads) or d != self.head_dim:
            _bad(f"{name} must have shape [{'tokens' if tokens is None else tokens}, {'heads' if heads is None else heads}, "
                 f"{self.head_dim}], got {tuple(x.shape)}")
        return t, h, packed


def _device(cache) -> torch.device:
    if not isinstance(cache, PagedCache):
        _bad("cache must be a PagedCache")
    if _derived(cache.k_pages) or _derived(cache.v_pages):   # since it was made, or made without recording
        raise B200NotSupportedError("the cache's pages require a gradient or have a tangent, which these operators do not record")
    return cache.device


def paged_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, query_starts: torch.Tensor, *,
                 q: Optional[torch.Tensor] = None, table: Optional[RotaryTable] = None,
                 out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the step's keys and values (k, v [tokens, kv_heads, head_dim]) into the cache. Sequence b
    has rows query_starts[b] .. query_starts[b + 1] - 1 (int32 [batch + 1]), its last positions in order.
    With a table, k is turned by its position first, and so is q [tokens, heads, head_dim], which is
    returned (in ``out``, which may be q itself). Rows of no sequence are not written, and what they hold
    has no effect."""
    device = _device(cache)
    tokens, _, kh = cache._rows(k, "k", cache.kv_heads, None)
    _, _, vh = cache._rows(v, "v", cache.kv_heads, tokens)
    starts = _starts(query_starts, device, cache.batch)
    ref = None if table is None else _table(table, device)
    if q is None:
        if out is not None:
            _bad("out needs q")
        _call("sb_paged_append", device, cache._ref, kh, vh, None, None, 0, tokens, starts, ref)
        return None
    if table is None:
        _bad("q needs a table")
    _, heads, qh = cache._rows(q, "q", None, tokens)
    if out is None:
        out = torch.empty_like(q)
    _, _, oh = cache._rows(out, "out", heads, tokens)
    _call("sb_paged_append", device, cache._ref, kh, vh, qh, oh, heads, tokens, starts, ref)
    return out


def paged_attention(cache: PagedCache, q: torch.Tensor, query_starts: torch.Tensor, *, scale: Optional[float] = None,
                    window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of the step's queries q [tokens, heads, head_dim] over the cache, each token
    over the positions of its sequence up to its own (``window`` > 0: the last ``window`` of them). Rows
    are as in ``paged_append``; query head h reads key head h // (heads // kv_heads); scale defaults to
    1 / sqrt(head_dim). A token that sees nothing gets zeros; rows of no sequence are not written."""
    device = _device(cache)
    tokens, heads, qh = cache._rows(q, "q", None, None)
    starts = _starts(query_starts, device, cache.batch)
    if out is None:
        out = torch.empty_like(q)
    _, _, oh = cache._rows(out, "out", heads, tokens)
    n = cache._workspace(heads, tokens)
    space = torch.empty(n, dtype=torch.uint8, device=device)
    _call("sb_paged_attention", device, cache._ref, qh, oh, heads, tokens, starts,
          cache.head_dim ** -0.5 if scale is None else scale, min(window, 1 << 30), space.data_ptr(), n)
    return out


def check(device="cuda") -> None:
    """Waits for the current stream of ``device`` and raises if a pipeline wait inside an attention call
    has run out there since the last check (its rows hold NaN or were not written)."""
    with torch.cuda.device(device):
        index = torch.cuda.current_device()
        _check(_native.lib().sb_decoder_status(torch._C._cuda_getCurrentRawStream(index)))


class W4Weights:
    """Weights (code - zero) * scale of a linear layer, codes in 4 bits, in the order the kernel reads.

    ``packed``: uint8 [out_features, ceil(in_features / 2)], element k of a row in the low half of byte
    k // 2 for even k, in the high half for odd k. ``scales``: [out_features, ceil(in_features /
    group_size)] float16 or bfloat16, the type of the layer's inputs. ``zeros``: uint8 of the same shape
    (0 to 15), or None for 8. ``group_size``: a multiple of 32. The laid out copy is made here, once, on
    the current stream (another stream waits for it before it uses the object); the arguments are not
    kept."""

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
                 in_features: int, group_size: int):
        device = _cuda(packed, "packed")
        _on(packed, "packed", device, torch.uint8, 2)
        if not isinstance(scales, torch.Tensor) or scales.dtype not in (torch.float16, torch.bfloat16):
            raise B200NotSupportedError("scales must be float16 or bfloat16")
        _on(scales, "scales", device, scales.dtype, 2)
        n, k, g = packed.shape[0], int(in_features), int(group_size)
        if g <= 0 or k <= 0:
            _bad("in_features and group_size must be positive")
        if packed.shape[1] != (k + 1) // 2 or (packed.stride(1) != 1 and packed.shape[1] > 1):
            _bad(f"packed must be [{n}, {(k + 1) // 2}] and contiguous along its rows, got {tuple(packed.shape)}")
        shape = (n, -(-k // g))
        if tuple(scales.shape) != shape or not scales.is_contiguous():
            _bad(f"scales must be {shape} and contiguous, got {tuple(scales.shape)}")
        if zeros is not None:
            _on(zeros, "zeros", device, torch.uint8, 2)
            if tuple(zeros.shape) != shape or not zeros.is_contiguous():
                _bad(f"zeros must be {shape} and contiguous, got {tuple(zeros.shape)}")
        self.out_features, self.in_features, self.group_size = n, k, g
        self.dtype, self.device = scales.dtype, device
        self._c = _native.W4Weights(None, _ELEM[scales.dtype], g, n, k, int(zeros is not None))
        size = C.c_size_t()
        _check(_native.lib().sb_w4_layout_bytes(C.byref(self._c), C.byref(size)))
        self._data = torch.empty(size.value, dtype=torch.uint8, device=device)
        self._c.data = self._data.data_ptr()
        self._ref = C.byref(self._c)
        _call("sb_w4_layout", device, self._ref, packed.data_ptr(), max(packed.stride(0), packed.shape[1]) if n == 1 else packed.stride(0),
              scales.data_ptr(), None if zeros is None else zeros.data_ptr(), self._data.data_ptr())


def linear_w4(x: torch.Tensor, weights: W4Weights, bias: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [rows, in_features] times the weights' transpose, plus bias [out_features], as [rows,
    out_features]; x, bias and the result have the weights' type. Meant for few rows: the weights are
    read once for every 32 of them."""
    if not isinstance(weights, W4Weights):
        _bad("weights must be W4Weights")
    device, dtype, n, k = weights.device, weights.dtype, weights.out_features, weights.in_features
    rows, xs = _matrix(x, "x", device, dtype, None, k)
    out = x.new_empty((rows, n)) if out is None else out
    ys = _matrix(out, "out", device, dtype, rows, n)[1]
    at = None
    if bias is not None:
        try:
            if (bias.dtype is dtype and bias.get_device() == device.index and bias.shape == (n,) and bias.is_contiguous()
                    and not _derived(bias)):
                at = bias.data_ptr()
        except AttributeError:
            pass
        if at is None:
            _on(bias, "bias", device, dtype, 1)
            _bad(f"bias must be {n} contiguous values, got {tuple(bias.shape)}")
    _call("sb_linear_w4", device, weights._ref, x.data_ptr(), xs, at, out.data_ptr(), ys, rows)
    return out


def _matrix(x, name: str, device: torch.device, dtype: torch.dtype, rows: Optional[int], columns: Optional[int]):
    """(rows, row stride) of a matrix whose rows are contiguous; rows or columns None: any number."""
    try:
        m, n = x.shape
        stride, last = x.stride()
        if (x.dtype is dtype and x.get_device() == device.index and (columns is None or n == columns) and (rows is None or m == rows)
                and (last == 1 or n == 1) and not _derived(x)):
            return m, stride
    except (AttributeError, TypeError, ValueError):
        pass
    _on(x, name, device, dtype, 2)
    _bad(f"{name} must be [{'rows' if rows is None else rows}, {'width' if columns is None else columns}] and contiguous along its rows, got {tuple(x.shape)}")


def _vector(x, name: str, device: torch.device, dtypes, n: int) -> int:
    """The address of n contiguous values of one of the types; 0 of None."""
    if x is None:
        return 0
    try:
        if x.dtype in dtypes and x.get_device() == device.index and x.shape == (n,) and (n == 1 or x.stride() == (1,)) and not _derived(x):
            return x.data_ptr()
    except AttributeError:
        pass
    _on(x, name, device, getattr(x, "dtype", None) if getattr(x, "dtype", None) in dtypes else dtypes[0], 1)
    _bad(f"{name} must be {n} contiguous values, got {tuple(x.shape)}")


_pack_norm = struct.Struct("PPPPPqqqqqPPPPqqiiiifff4x").pack   # sb_residual_norm_args
_pack_sampling = struct.Struct("PPPPfffi").pack              # sb_sampling


def residual_norm(x: torch.Tensor, weight: Optional[torch.Tensor], *, bias: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, scale: float = 1.0, kind: str = "rms",
                  eps: float = 1e-6, weight_offset: float = 0.0, out: Optional[torch.Tensor] = None,
                  residual_out: Optional[torch.Tensor] = None):
    """The norms around a block's residual, for each row of x [rows, width] (float32, float16, bfloat16):

        t = norm(x) post_weight + post_bias     (x without a post_weight)
        h = residual + scale gate t
        y = norm(h) weight + bias

    as (y, h). norm(z) is z / sqrt(mean(z^2) + eps) or, with kind "layer", the same of z less its mean.
    ``residual`` [rows, width] has x's type or float32, and so has h; ``gate`` is [width] or [rows, width] of x's
    type; weights and biases [width] have x's type or float32, all of them the same one; ``weight_offset`` is added
    to both weights. Without residual, gate, post_weight and scale h is x itself, or a copy where ``out`` is x; without a
    weight y is None. y is taken of h before h is rounded. ``out`` may be x, and ``residual_out`` x or residual; they may
    not overlap an input otherwise. Rows that begin alike within 16 bytes, and weights that are 16-byte aligned (whole tensors
    are), go in wide accesses; others element by element, up to three times as slow."""
    device = _cuda(x, "x")
    dtype = x.dtype
    elem = _ELEM.get(dtype)
    if elem is None:
        raise B200NotSupportedError(f"element type {dtype} is not supported")
    if kind != "rms" and kind != "layer":
        _bad(f"kind must be 'rms' or 'layer', got {kind!r}")
    rows, xs = _matrix(x, "x", device, dtype, None, None)
    n = x.shape[1]
    sum_type, rs, rp = dtype, 0, 0
    if residual is not None:
        if getattr(residual, "dtype", None) is torch.float32:
            sum_type = torch.float32
        rs = _matrix(residual, "residual", device, sum_type, rows, n)[1]
        rp = residual.data_ptr()
    elif residual_out is not None and getattr(residual_out, "dtype", None) is torch.float32:
        sum_type = torch.float32
    gp, gs = 0, 0
    if gate is not None:
        if isinstance(gate, torch.Tensor) and gate.dim() == 1:
            gp = _vector(gate, "gate", device, (dtype,), n)
        else:
            gs = _matrix(gate, "gate", device, dtype, rows, n)[1]
            gp = gate.data_ptr()
    first = weight if weight is not None else post_weight
    kinds = (dtype,)
    if first is not None:
        if getattr(first, "dtype", None) is torch.float32:
            kinds = (torch.float32,)
        wp = _vector(weight, "weight", device, kinds, n)
        bp = _vector(bias, "bias", device, kinds, n) if bias is not None else 0
        pp = _vector(post_weight, "post_weight", device, kinds, n) if post_weight is not None else 0
        cp = _vector(post_bias, "post_bias", device, kinds, n) if post_bias is not None else 0
    else:
        wp = pp = bp = cp = 0
    if weight is None and (bias is not None or out is not None):
        _bad("bias and out need a weight")
    if post_weight is None and post_bias is not None:
        _bad("post_bias needs a post_weight")
    h, hp, ss = x, 0, 0
    over = weight is not None and out is not None and isinstance(out, torch.Tensor) and out.data_ptr() == x.data_ptr()
    if residual is not None or gate is not None or post_weight is not None or scale != 1.0 or residual_out is not None or over:
        if residual_out is None:
            h, ss = x.new_empty((rows, n), dtype=sum_type), n
        else:
            h, ss = residual_out, _matrix(residual_out, "residual_out", device, sum_type, rows, n)[1]
        hp = h.data_ptr()
    elif weight is None:
        _bad("there is nothing to compute")
    y, yp, ys = None, 0, 0
    if weight is not None:
        if out is None:
            y, ys = x.new_empty((rows, n)), n
        else:
            y, ys = out, _matrix(out, "out", device, dtype, rows, n)[1]
        yp = y.data_ptr()
    try:
        a = _pack_norm(x.data_ptr(), rp, gp, hp, yp, xs, rs, gs, ss, ys, wp, bp, pp, cp, rows, n, elem, _ELEM[sum_type], _ELEM[kinds[0]],
                       kind == "layer", scale, eps, weight_offset)
    except (struct.error, OverflowError) as e:
        raise B200ArgumentError(f"scale, eps and weight_offset must be numbers of 32 bits: {e}") from None
    _call("sb_residual_norm", device, a)
    return y, h


class MoEWeights:
    """Weights of a mixture-of-experts layer, and how a token chooses: ``router`` [experts, width] (the weights' type or
    float32), ``gate_up`` [experts, 2 * inner, width] (the gates' rows first), ``down`` [experts, width, inner],
    float16 or bfloat16, of any strides (multiples of 8) along all but the last dimension. A token's scores are the
    softmax (``scoring`` "softmax") or the sigmoids ("sigmoid") of router x; its experts the ``top_k`` largest of
    score + ``selection_bias`` (float32 [experts]; equal ones: the lower first), their shares the scores, divided by
    their sum with ``normalize``, times ``scale``. ``activation`` of the gates: "silu" or "gelu". The object keeps the
    tensors; their contents may change between calls."""

    def __init__(self, router: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, *, top_k: int, scoring: str = "softmax",
                 normalize: bool = True, scale: float = 1.0, selection_bias: Optional[torch.Tensor] = None, activation: str = "silu"):
        device = _cuda(gate_up, "gate_up")
        dtype = gate_up.dtype
        if dtype not in (torch.float16, torch.bfloat16):
            raise B200NotSupportedError(f"element type {dtype} is not supported")
        _on(gate_up, "gate_up", device, dtype, 3)
        _on(down, "down", device, dtype, 3)
        _on(router, "router", device, torch.float32 if getattr(router, "dtype", None) is torch.float32 else dtype, 2)
        experts, wide, width = gate_up.shape
        inner = wide // 2
        if wide != 2 * inner or tuple(down.shape) != (experts, width, inner) or tuple(router.shape) != (experts, width):
            _bad(f"router, gate_up and down must be [experts, width], [experts, 2 * inner, width] and [experts, width, inner], got "
                 f"{tuple(router.shape)}, {tuple(gate_up.shape)} and {tuple(down.shape)}")
        for name, p in (("router", router), ("gate_up", gate_up), ("down", down)):
            if p.stride(-1) != 1 and p.shape[-1] > 1:
                _bad(f"{name} must be contiguous along its last dimension")
        if scoring not in ("softmax", "sigmoid"):
            _bad(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
        if activation not in ("silu", "gelu"):
            _bad(f"activation must be 'silu' or 'gelu', got {activation!r}")
        try:
            top_k, scale = int(top_k), float(scale)
        except (TypeError, ValueError, OverflowError) as e:
            raise B200ArgumentError(f"top_k and scale must be numbers: {e}") from None
        if not 0 < top_k <= experts:   # (the C structure would keep 32 bits of it)
            _bad(f"top_k {top_k} of {experts} experts")
        bias = _vector(selection_bias, "selection_bias", device, (torch.float32,), experts)
        self.router, self.gate_up, self.down, self.selection_bias = router, gate_up, down, selection_bias
        self.device, self.dtype, self.experts, self.width, self.inner, self.top_k = device, dtype, experts, width, inner, top_k
        self._c = _native.MoEWeights(router.data_ptr(), gate_up.data_ptr(), down.data_ptr(), bias, router.stride(0), gate_up.stride(0),
                                     gate_up.stride(1), down.stride(0), down.stride(1), experts, width, inner, _ELEM[dtype],
                                     _ELEM[router.dtype], self.top_k, int(scoring == "sigmoid"), int(bool(normalize)),
                                     int(activation == "gelu"), scale)
        self._ref = C.byref(self._c)
        self._space = {}
        self._workspace(1)   # refuses what the layer does not support

    def _workspace(self, tokens: int) -> int:
        n = self._space.get(tokens)
        if n is None:
            size = C.c_size_t()
            _check(_native.lib().sb_moe_workspace(self._ref, tokens, C.byref(size)))
            if len(self._space) > 64:
                self._space.clear()
            n = self._space[tokens] = size.value
        return n


def moe(x: torch.Tensor, weights: MoEWeights, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The mixture-of-experts layer of x [tokens, width], of the weights' type: for each token the sum over its
    experts of share * down (act(gate x) * (up x)). Meant for few tokens: an expert's weights are read from memory anew for
    every 256 tokens (2048 / top_k where that is less). Hidden values are held as two numbers of the weights' type (16 bits in bfloat16, 22 in
    float16, where they overflow beyond 65504). ``out`` may be x itself."""
    if not isinstance(weights, MoEWeights):
        _bad("weights must be MoEWeights")
    for name in ("router", "gate_up", "down", "selection_bias"):   # since the object was made, or made without recording
        t = getattr(weights, name)
        if t is not None and _derived(t):
            raise B200NotSupportedError(f"{name} requires a gradient or has a tangent, which these operators do not record")
    device, dtype = weights.device, weights.dtype
    tokens, xs = _matrix(x, "x", device, dtype, None, weights.width)
    if out is None:
        out, ys = x.new_empty((tokens, weights.width)), weights.width
    else:
        ys = _matrix(out, "out", device, dtype, tokens, weights.width)[1]
    n = weights._workspace(tokens)
    space = torch.empty(n, dtype=torch.uint8, device=device)
    _call("sb_moe", device, weights._ref, x.data_ptr(), xs, out.data_ptr(), ys, tokens, space.data_ptr(), n)
    return out


def sample(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The next token of each row of logits [rows, vocab] (float32, float16, bfloat16; NaN counts as -inf), int64
    [rows], from the row's number in ``uniform`` (float32 [rows], in [0, 1)). With w = exp((l - max) / temperature),
    kept are w >= min_p, of these the top_k largest, of these the fewest largest whose sum is at least top_p of theirs
    (equal logits: the lower index first); the token is the first index at which the running sum of the kept w, in order
    of the index, exceeds uniform times their sum. Each setting is a number or a tensor of one per row (float32, top_k
    int32). Temperature 0 (or less): the first of the largest; top_k 0 (or less), top_p 1 (or more) and min_p 0 (or
    less) filter nothing, and at any min_p the largest is kept. A row without a logit above -inf gives -1. Weights below
    2^-43 count as 0."""
    device = _cuda(logits, "logits")
    dtype = logits.dtype
    elem = _ELEM.get(dtype)
    if elem is None:
        raise B200NotSupportedError(f"element type {dtype} is not supported")
    rows, stride = _matrix(logits, "logits", device, dtype, None, None)
    at = _vector(uniform, "uniform", device, _FLOAT, rows)
    tp = pp = mp = kp = 0
    if isinstance(temperature, torch.Tensor):
        tp, temperature = _vector(temperature, "temperature", device, _FLOAT, rows), 1.0
    if isinstance(top_k, torch.Tensor):
        kp, top_k = _vector(top_k, "top_k", device, (torch.int32,), rows), 0
    if isinstance(top_p, torch.Tensor):
        pp, top_p = _vector(top_p, "top_p", device, _FLOAT, rows), 1.0
    if isinstance(min_p, torch.Tensor):
        mp, min_p = _vector(min_p, "min_p", device, _FLOAT, rows), 0.0
    if out is None:
        out = logits.new_empty((rows,), dtype=torch.int64)
        to = out.data_ptr()
    else:
        to = _vector(out, "out", device, (torch.int64,), rows)
    try:
        by = _pack_sampling(tp, pp, mp, kp, temperature, top_p, min_p, min(max(int(top_k), 0), 0x7fffffff))
    except (struct.error, TypeError, ValueError, OverflowError) as e:
        raise B200ArgumentError(f"temperature, top_k, top_p and min_p must be numbers of 32 bits or tensors: {e}") from None
    _call("sb_sample", device, logits.data_ptr(), stride, elem, rows, logits.shape[1], at, by, to)
    return out


_FLOAT = (torch.float32,)
