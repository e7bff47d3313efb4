"""Attention over torch CUDA tensors: norms of queries and keys with their rotation, a paged cache of keys and values,
and attention of one new token over it.

Part of the device-resident layer (see ``device``): every operation is one call into ``liblapis_b200.so`` on torch's
current stream, operands are tensors of the current device, results are new tensors.  Nothing is recorded for autograd.  A serving
step is

    q = cache.append_norm_rope(q, k, v, q_weight, k_weight, cos, sin, pos, crd, row, place)
    out = paged_attention(q, cache, pos, crd, length)

Which pages hold a request's tokens is a CSR pattern: place ``p`` of request ``r`` lies in page ``crd[pos[r] + p //
page_size]``, slot ``p % page_size``.  ``pos``, ``crd``, ``row``, ``place`` and ``length`` are all int32 or all int64.
What the lists say is checked on the device: places, requests and pages that do not exist are never accessed.  Rows of
heads ([tokens, heads, dim], dim at most 256) may be views with any strides whose last one is 1.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import KvCache, check
from .device import _calls

_CACHE_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_ROW_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _tensors(**named):
    """Operands that are looked at first: tensors, of three extents where the name says so."""
    for name, t in named.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if name in ("q", "k", "v", "dq", "dk") and t.dim() != 3:
            raise ValueError(f"{name} must be [tokens, heads, dim]")


def _check_rows(name, t, dtype, tokens, dim, heads=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _ROW_TYPES or t.dtype != dtype:
        raise TypeError(f"{name} must be a CUDA tensor of float32, float16 or bfloat16, the same for all rows")
    if t.device.index != torch.cuda.current_device():
        raise TypeError(f"{name} must be on the current device")
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, heads, dim]")
    if t.stride(2) != 1 and dim > 1:
        raise TypeError(f"{name}: the values of a head must lie next to one another")


def _check_indices(dtype, **tensors):
    for name, (t, count) in tensors.items():
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != dtype or dtype not in (torch.int32, torch.int64) or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous CUDA tensor, all indices int32 or all int64")
        if t.device.index != torch.cuda.current_device():
            raise TypeError(f"{name} must be on the current device")
        if t.dim() != 1 or (count is not None and t.numel() != count):
            raise ValueError(f"{name} has the wrong length")


def _check_lists(pos, crd):
    _check_indices(getattr(pos, "dtype", None), pos=(pos, None), crd=(crd, None))
    if pos.numel() < 1:
        raise ValueError("pos must have requests + 1 entries")


def _check_how(dtype, dim, q_weight, k_weight, cos, sin):
    _tensors(q_weight=q_weight, cos=cos)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if not isinstance(w, torch.Tensor) or not w.is_cuda or not w.is_contiguous() or w.dtype not in (torch.float32, dtype) or w.dtype != q_weight.dtype:
            raise TypeError(f"{name} must be a contiguous CUDA tensor of float32 or of the rows' type, the same for both")
        if w.device.index != torch.cuda.current_device():
            raise TypeError(f"{name} must be on the current device")
        if tuple(w.shape) != (dim,):
            raise ValueError(f"{name} must be [dim]")
    for name, t in (("cos", cos), ("sin", sin)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous() or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a contiguous float32 CUDA tensor")
        if t.device.index != torch.cuda.current_device():
            raise TypeError(f"{name} must be on the current device")
        if t.dim() != 2 or t.shape != cos.shape or 2 * t.shape[1] > dim:
            raise ValueError(f"{name} must be [places, rot / 2] with rot <= dim")


def _raise(what):
    raise TypeError(f"{what}: operands of the wrong kind")


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, place, eps: float = 1e-6, interleaved: bool = False):
    """(q, k) normalised head by head, x / sqrt(mean x^2 + eps) * weight, and rotated by the angle of their token's place.

    ``cos``/``sin`` [places, rot / 2]: the first ``rot`` values of a head are turned in pairs (i, i + rot/2), or (2i, 2i+1)
    with ``interleaved``.  Computed in 32 bits.  A token whose place is outside the tables is padding and gives zeros."""
    got = _calls.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps, interleaved, place)
    if type(got) is int:
        if got < 0:
            _tensors(q=q, k=k)
            _check_rows("q", q, q.dtype, q.shape[0], q.shape[2])
            _check_rows("k", k, q.dtype, q.shape[0], q.shape[2])
            _check_how(q.dtype, q.shape[2], q_weight, k_weight, cos, sin)
            _check_indices(getattr(place, "dtype", None), place=(place, q.shape[0]))
            _raise("qk_norm_rope")
        check(got)
    return got


def qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, place, eps: float = 1e-6, interleaved: bool = False):
    """Gradients of :func:`qk_norm_rope` for those of its outputs, ``dq`` and ``dk``, and its inputs: (of q, of k, of
    q_weight, of k_weight).  Those of the weights are float32, sums over all tokens and heads in a fixed order."""
    got = _calls.qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, eps, interleaved, place)
    if type(got) is int:
        if got < 0:
            _tensors(dq=dq, dk=dk, q=q, k=k)
            _check_rows("q", q, q.dtype, q.shape[0], q.shape[2])
            _check_rows("k", k, q.dtype, q.shape[0], q.shape[2])
            _check_rows("dq", dq, q.dtype, q.shape[0], q.shape[2], q.shape[1])
            _check_rows("dk", dk, q.dtype, q.shape[0], q.shape[2], k.shape[1])
            _check_how(q.dtype, q.shape[2], q_weight, k_weight, cos, sin)
            _check_indices(getattr(place, "dtype", None), place=(place, q.shape[0]))
            _raise("qk_norm_rope_backward")
        check(got)
    q_grad, k_grad, weights = got
    return q_grad, k_grad, *weights.unbind()


class PagedCache:
    """Keys and values of many requests in pages of ``page_size`` tokens (``lapis_b200_kv_cache``).

    ``k``/``v`` [pages, heads, page_size, dim]: float32, float16, bfloat16, int8 or float8_e4m3fn CUDA tensors; a quantised
    cache has float32 scales [pages, heads, page_size], one for each head of each token.  The tensors are borrowed (kept
    referenced here)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous() or t.dtype not in _CACHE_TYPES or t.dtype != k.dtype:
                raise TypeError(f"{name} must be a contiguous CUDA tensor of float32, float16, bfloat16, int8 or float8_e4m3fn")
            if t.dim() != 4 or t.shape != k.shape or min(t.shape[1:]) < 1:
                raise ValueError(f"{name} must be [pages, heads, page_size, dim]")
        if k.shape[3] > 256:
            raise ValueError("heads of more than 256 values")
        quantised = k.dtype in (torch.int8, torch.float8_e4m3fn)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if (t is not None) != quantised:
                raise ValueError(f"{name}: scales belong to a quantised cache")
            if quantised and not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
                raise TypeError(f"{name} must be a contiguous float32 CUDA tensor")
            if quantised and t.shape != k.shape[:3]:
                raise ValueError(f"{name} must be [pages, heads, page_size]")
        for t in (v, k_scale, v_scale):
            if t is not None and t.device != k.device:
                raise ValueError("the arrays of a cache must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page_size, self.dim = (int(n) for n in k.shape)

        def address(t):
            return None if t is None or t.numel() == 0 else t.data_ptr()
        self._c = KvCache(_CACHE_TYPES[k.dtype], self.pages, self.heads, self.page_size, self.dim, address(k), address(v), address(k_scale),
                          address(v_scale))
        self._addr = ctypes.addressof(self._c)
        self._device = k.device.index

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedCache":
        """A cache whose slots hold nothing yet (uninitialised: a slot is read only after it has been written)."""
        shape = (pages, heads, page_size, dim)
        scales = [torch.empty(shape[:3], dtype=torch.float32, device=device) if dtype in (torch.int8, torch.float8_e4m3fn) else None for _ in range(2)]
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device), *scales)

    def _here(self, what):
        if self._device != torch.cuda.current_device():
            raise TypeError(f"{what}: the cache must be on the current device")

    def _check_new(self, k, v, pos, crd, row, place):
        _tensors(k=k, v=v)
        _check_rows("k", k, k.dtype, k.shape[0], self.dim, self.heads)
        _check_rows("v", v, k.dtype, k.shape[0], self.dim, self.heads)
        _check_lists(pos, crd)
        _check_indices(pos.dtype, crd=(crd, None), row=(row, k.shape[0]), place=(place, k.shape[0]))

    def append(self, k, v, pos, crd, row, place) -> None:
        """Writes token t of ``k``, ``v`` [tokens, heads, dim] at place ``place[t]`` of request ``row[t]``, quantised where the
        cache is."""
        self._here("append")
        status = _calls.kv_append(self._addr, k, v, pos, crd, row, place)
        if status:
            if status < 0:
                self._check_new(k, v, pos, crd, row, place)
                _raise("append")
            check(status)

    def append_norm_rope(self, q, k, v, q_weight, k_weight, cos, sin, pos, crd, row, place, eps: float = 1e-6, interleaved: bool = False):
        """:func:`qk_norm_rope` and :meth:`append` in one launch: returns the queries; the keys are quantised, where the cache
        is, from 32 bits, without a rounding to their own type in between.  Padding (see there) is not written."""
        self._here("append_norm_rope")
        got = _calls.kv_append_norm_rope(self._addr, q, k, v, q_weight, k_weight, cos, sin, eps, interleaved, pos, crd, row, place)
        if type(got) is int:
            if got < 0:
                self._check_new(k, v, pos, crd, row, place)
                _tensors(q=q)
                _check_rows("q", q, k.dtype, k.shape[0], self.dim)
                _check_how(k.dtype, self.dim, q_weight, k_weight, cos, sin)
                _raise("append_norm_rope")
            check(got)
        return got

    def read(self, pos, crd, row, place, dtype: torch.dtype = torch.bfloat16):
        """(k, v) [tokens, heads, dim] of the tokens at ``place[t]`` of requests ``row[t]``, in ``dtype``; zeros where the lists
        name no page."""
        self._here("read")
        if dtype not in _ROW_TYPES:
            raise TypeError("read: dtype must be float32, float16 or bfloat16")
        got = _calls.kv_read(self._addr, pos, crd, row, place, _CACHE_TYPES[dtype])
        if type(got) is int:
            if got < 0:
                _check_lists(pos, crd)
                _tensors(row=row)
                _check_indices(pos.dtype, crd=(crd, None), row=(row, row.numel()), place=(place, row.numel()))
                _raise("read")
            check(got)
        return got


def paged_attention(q, cache: PagedCache, pos, crd, length, scale: float | None = None, window: int = 0, return_lse: bool = False):
    """softmax(scale * q.k) v of one new token of each request, ``q`` [requests, heads, dim], over the first ``length[r]``
    places of its list (the new token's own key and value among them), or the last ``window`` of these.

    Query heads share the cache's heads in consecutive groups.  ``scale`` defaults to dim ** -0.5.  With ``return_lse`` also
    the natural logarithm of each head's sum of exponentials, float32 [requests, heads], with which results over parts of a
    context are joined.  A request of length 0 gets zeros and -inf."""
    cache._here("paged_attention")
    got = _calls.paged_attention(cache._addr, q, pos, crd, length, cache.dim ** -0.5 if scale is None else scale, window or 0, return_lse)
    if type(got) is int:
        if got < 0:
            _tensors(q=q)
            _check_rows("q", q, q.dtype, q.shape[0], cache.dim)
            _check_lists(pos, crd)
            _check_indices(pos.dtype, crd=(crd, None), length=(length, q.shape[0]))
            _raise("paged_attention")
        check(got)
    return got
