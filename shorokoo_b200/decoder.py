"""Decoder-layer operators on device tensors: what one layer of a language model runs per step when it
answers from a paged cache (the sb_rotary*, sb_paged_* and sb_*w4* entry points of the library's C ABI).

    weights = W4Weights(packed, scales, zeros, in_features=4096, group_size=128)     # once
    table = RotaryTable(128, 500000.0)                                               # once
    cache = PagedCache(k_pages, v_pages, page_table, context_lengths)                # once per step's batch
    qkv = linear_w4(x, weights)
    q = paged_append(cache, k, v, query_starts, q=q, table=table)
    o = paged_attention(cache, q, query_starts)

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


def _matrix(x, name: str, device: torch.device, dtype: torch.dtype, rows: Optional[int], columns: int):
    """(rows, row stride) of a matrix whose rows are contiguous; rows None: any number."""
    try:
        m, n = x.shape
        stride, last = x.stride()
        if (x.dtype is dtype and x.get_device() == device.index and n == columns and (rows is None or m == rows)
                and (last == 1 or n == 1) and not _derived(x)):
            return m, stride
    except (AttributeError, TypeError, ValueError):
        pass
    _on(x, name, device, dtype, 2)
    _bad(f"{name} must be [{'rows' if rows is None else rows}, {columns}] and contiguous along its rows, got {tuple(x.shape)}")
