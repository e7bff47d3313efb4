"""A layer of experts over torch CUDA tensors: the router, each expert's tokens as CSR rows, rows there and back, and products of
few rows with weights of 4 bits.

Part of the device-resident layer (see ``device``): every operation is one call into ``liblapis_b200.so`` on torch's
current stream, operands are tensors of the current device, results are new tensors.  Nothing is recorded for autograd:
gradients are calls of their own.  A serving step is

    weights, expert = route(logits, k)
    lists = ExpertLists(expert, experts)
    rows = down.matmul(up.matmul(x, lists, fetch=True), lists)      # Int4Matrix, `up` gated
    out = lists.combine(rows, weights)

and training has ``lists.gather(x)`` in front of the products of its experts, rows ``lists.pos[e]`` to ``lists.pos[e + 1]`` being
expert e's.  Rows ([tokens, dim]) are float32, float16 or bfloat16 and may be views with any strides whose last one is 1.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import Int4, check, load
from .device import _calls, _ptr, _stream

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _check_rows(name, t, rows=None, dim=None, dtype=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _TYPES or (dtype is not None and t.dtype != dtype):
        raise TypeError(f"{name} must be a CUDA tensor of float32, float16 or bfloat16, the same for all rows")
    if t.device.index != torch.cuda.current_device():
        raise TypeError(f"{name} must be on the current device")
    if t.dim() != 2 or (rows is not None and t.shape[0] != rows) or (dim is not None and t.shape[1] != dim):
        raise ValueError(f"{name} must be [{'rows' if rows is None else rows}, {'dim' if dim is None else dim}]")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise TypeError(f"{name}: the values of a row must lie next to one another")


def _check_slots(name, t, dtypes, shape=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous CUDA tensor of {' or '.join(str(d)[6:] for d in dtypes)}")
    if t.device.index != torch.cuda.current_device():
        raise TypeError(f"{name} must be on the current device")
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{name} must be [tokens, k]")


def _raise(what):
    raise TypeError(f"{what}: operands of the wrong kind")


def route(logits, k: int, normalise: bool = True):
    """(weights, expert) [tokens, k] of the ``k`` largest of each token's ``logits`` [tokens, experts], the largest first, of equal
    ones the lowest expert first: float32 shares of the softmax of the chosen ones, or of all without ``normalise``, and int32
    numbers.

    A logit of -inf is never chosen: where too few are left (a token of padding has none) the expert is -1 and the weight 0.  A
    NaN counts as the largest logit; with it, or with +inf, the token's weights are NaN.  At most 1024 experts, k at most 32."""
    got = _calls.route(logits, k, normalise)
    if type(got) is int:
        if got < 0:
            _check_rows("logits", logits)
            if not 0 <= k <= logits.shape[1]:
                raise ValueError("route: k must be between 0 and the number of experts")
            _raise("route")
        check(got)
    return got


def route_backward(dweights, logits, expert, normalise: bool = True):
    """Gradient of :func:`route` for its ``logits``, of their type: ``dweights`` [tokens, k] of its weights, ``expert`` as it
    returned them (numbers outside [0, experts) count as no choice)."""
    got = _calls.route_backward(dweights, logits, expert, normalise)
    if type(got) is int:
        if got < 0:
            _check_rows("logits", logits)
            _check_slots("expert", expert, (torch.int32,))
            if expert.shape[0] != logits.shape[0] or expert.shape[1] > logits.shape[1]:
                raise ValueError("expert must be [tokens, k] with k at most the number of experts")
            _check_slots("dweights", dweights, (torch.float32,), tuple(expert.shape))
            _raise("route_backward")
        check(got)
    return got


class ExpertLists:
    """The slots of each expert as the rows of a CSR pattern: slot ``token * k + j`` is the token's j-th of ``expert`` [tokens, k]
    (int32 or int64).

    ``crd`` holds the slots sorted by expert, ascending within each; those of expert e are ``crd[pos[e]:pos[e + 1]]``.  Slots whose
    expert is outside [0, experts), padding or experts that another process holds, follow behind ``pos[experts]``.
    ``place`` [tokens, k] is where a slot stands in ``crd``.  All int32.  At most 1024 experts."""

    def __init__(self, expert: torch.Tensor, experts: int):
        got = _calls.expert_lists(expert, experts)
        if type(got) is int:
            if got < 0:
                _check_slots("expert", expert, (torch.int32, torch.int64))
                if not 0 <= experts <= 1024:
                    raise ValueError("ExpertLists: experts must be between 0 and 1024")
                _raise("ExpertLists")
            check(got)
        self.pos, self.crd, self.place = got

    @property
    def experts(self) -> int:
        return self.pos.numel() - 1

    def _raise(self, what):
        for name in ("pos", "crd", "place"):
            t = getattr(self, name)
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or not t.is_contiguous():
                raise TypeError(f"{what}: {name} must be a contiguous int32 CUDA tensor")
            if t.device.index != torch.cuda.current_device():
                raise TypeError(f"{what}: the lists must be on the current device")
        _raise(what)

    def gather(self, x):
        """Rows [tokens * k, dim] in the order of the lists: the token's row ``x`` [tokens, dim] at the place of each of its slots,
        zeros for slots of no expert."""
        got = _calls.expert_gather(x, self.pos, self.crd, self.place)
        if type(got) is int:
            if got < 0:
                _check_rows("x", x, self.place.shape[0])
                self._raise("gather")
            check(got)
        return got

    def gather_backward(self, drows):
        """Gradient of :meth:`gather` for x: the sums of its slots' rows of ``drows`` [tokens * k, dim], for slots of no expert
        nothing, in 32 bits and in the order of the slots."""
        return self._combine("gather_backward", "drows", drows, None)

    def combine(self, rows, weights):
        """[tokens, dim]: the sums of the slots' ``rows`` [tokens * k, dim] times their ``weights`` (float32 [tokens, k]), in 32 bits and
        in the order of the slots.  Rows of no expert are not looked at."""
        if weights is None:
            raise TypeError("weights must be a contiguous CUDA tensor of float32")
        return self._combine("combine", "rows", rows, weights)

    def _combine(self, what, name, rows, weights):
        got = _calls.expert_combine(rows, weights, self.pos, self.crd, self.place)
        if type(got) is int:
            if got < 0:
                _check_rows(name, rows, self.crd.numel())
                if weights is not None:
                    _check_slots("weights", weights, (torch.float32,), tuple(self.place.shape))
                self._raise(what)
            check(got)
        return got

    def combine_backward(self, dout, rows, weights):
        """Gradients of :meth:`combine` for its ``rows`` and ``weights``, ``dout`` [tokens, dim] of its result: (of rows, zeros for those
        of no expert; of weights, float32)."""
        got = _calls.expert_combine_backward(dout, rows, weights, self.pos, self.crd, self.place)
        if type(got) is int:
            if got < 0:
                _check_rows("rows", rows, self.crd.numel())
                _check_rows("dout", dout, self.place.shape[0], rows.shape[1], rows.dtype)
                _check_slots("weights", weights, (torch.float32,), tuple(self.place.shape))
                self._raise("combine_backward")
            check(got)
        return got


class Int4Matrix:
    """Weights of 4 bits, w = (code - zero) * scale, for one product or for that of each expert (``lapis_b200_int4``).

    ``codes`` uint8 [outputs, ceil(columns / 2)] or [experts, outputs, ceil(columns / 2)], the even column in the low half of a byte;
    ``scale`` float32, float16 or bfloat16 [.., outputs, ceil(columns / group)]; ``zero`` uint8 of the same shape (0 to 15), or None:
    8 throughout.  ``group`` is 32, 64 or 128 columns.  ``gated``: the first half of the outputs are gates, and a product is
    silu(gate) * the other half.  The weights are laid out anew here, once; the call returns when that is done, and the tensors
    are not needed any more.  Products may run on any stream: the memory of weights that are dropped is kept until they have ended.  (Graphs
    that were captured need their weights kept by the caller.)"""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, zero: torch.Tensor | None = None, *, columns: int, group: int = 128, gated: bool = False):
        for name, t, dtypes in (("codes", codes, (torch.uint8,)), ("scale", scale, tuple(_TYPES)), ("zero", zero, (torch.uint8,))):
            if name == "zero" and t is None:
                continue
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes or not t.is_contiguous():
                raise TypeError(f"{name} must be a contiguous CUDA tensor of {' or '.join(str(d)[6:] for d in dtypes)}")
            if t.device.index != torch.cuda.current_device():
                raise TypeError(f"{name} must be on the current device")
        if group not in (32, 64, 128):
            raise ValueError("groups of 32, 64 or 128 columns")
        if codes.dim() not in (2, 3) or columns < 0 or codes.shape[-1] != (columns + 1) // 2:
            raise ValueError("codes must be [outputs, ceil(columns / 2)] or [experts, outputs, ceil(columns / 2)]")
        for name, t in (("scale", scale), ("zero", zero)):
            if t is not None and tuple(t.shape) != (*codes.shape[:-1], -(-columns // group)):
                raise ValueError(f"{name} must be [.., outputs, ceil(columns / group)]")
        if gated and codes.shape[-2] % 2:
            raise ValueError("gated weights have an even number of outputs")
        self.experts, self.outputs, self.columns, self.group, self.gated = codes.shape[0] if codes.dim() == 3 else 1, codes.shape[-2], columns, group, bool(gated)
        lib = load()
        self._c = Int4(self.experts, self.outputs, columns, group, _TYPES[scale.dtype], zero is not None, self.gated, None)
        size = lib.lapis_b200_int4_bytes(ctypes.byref(self._c))
        if size < 0:
            check(lib.lapis_last_error())
        self._packed = torch.empty(size, dtype=torch.uint8, device=codes.device)
        self._c.d_packed = self._packed.data_ptr() if size else None
        check(lib.lapis_b200_int4_pack(ctypes.byref(self._c), _ptr(codes), _ptr(scale), _ptr(zero), _ptr(self._packed), _stream()))
        self._addr = ctypes.addressof(self._c)
        self._device = codes.device.index
        self._streams = {_stream()}

    @classmethod
    def quantise(cls, w: torch.Tensor, group: int = 128, zeros: bool = False, scale_dtype: torch.dtype | None = None, gated: bool = False) -> "Int4Matrix":
        """Dense weights [outputs, columns] or [experts, outputs, columns] rounded to 4 bits, see :func:`quantise_int4`."""
        codes, scale, zero = quantise_int4(w, group, zeros, scale_dtype)
        return cls(codes, scale, zero, columns=w.shape[-1], group=group, gated=gated)

    def matmul(self, x, lists: ExpertLists | None = None, fetch: bool = False):
        """x w^T of rows ``x`` [rows, columns], of their type.  Every product of a code and a value is exact, but for what float32 values
        below 2^-110 have below 2^-133; sums are in 32 bits, cut instead of rounded within a group, and rounded to the type once.

        With ``lists`` row i of the result is that of slot ``lists.crd[i]``, times its expert's weights, zeros for slots of no
        expert; ``x`` holds the slots' rows in the same order, or with ``fetch`` those of the tokens [tokens, columns].

        Made for few rows: a pass over the weights serves 8, 32, 64 or, with groups of 128, 128 of them (a third of that where they
        are float32), as many as there are, or with ``lists`` as twice the slots / experts.  An expert with more rows takes
        further passes, one after the other.  With more than 8 the kernel's waits are bounded: where one gave up, the result is not
        valid and ``device.bgemm_status()`` raises."""
        if self._device != torch.cuda.current_device():
            raise TypeError("matmul: the weights must be on the current device")
        if (stream := torch._C._cuda_getCurrentRawStream(self._device)) not in self._streams:  # nobody else has the weights' memory to say so
            self._packed.record_stream(torch.cuda.current_stream())
            self._streams.add(stream)
        if lists is None:
            if fetch:
                raise ValueError("matmul: rows are fetched by lists")
            got = _calls.int4_matmul(self._addr, x)
        else:
            got = _calls.int4_matmul_lists(self._addr, x, fetch, lists.pos, lists.crd, lists.place)
        if type(got) is int:
            if got < 0:
                _check_rows("x", x, dim=self.columns)
                if lists is not None:
                    lists._raise("matmul")
                _raise("matmul")
            check(got)
        return got


def quantise_int4(w: torch.Tensor, group: int = 128, zeros: bool = False, scale_dtype: torch.dtype | None = None):
    """(codes, scale, zero or None) of dense weights [.., columns], to the nearest code, for :class:`Int4Matrix`.

    Without ``zeros`` a group's scale is its largest magnitude / 7 and the codes are 1 to 15; with them the scale is the range of the
    group and 0, / 15.  ``scale_dtype`` defaults to the type of ``w``; codes are those of the rounded scale.  A group that is not
    finite gets a scale of NaN."""
    if not isinstance(w, torch.Tensor) or not w.is_cuda or w.dtype not in _TYPES or not w.is_contiguous():
        raise TypeError("w must be a contiguous CUDA tensor of float32, float16 or bfloat16")
    if w.device.index != torch.cuda.current_device():
        raise TypeError("w must be on the current device")
    if w.dim() < 2:
        raise ValueError("w must be [.., outputs, columns]")
    if group not in (32, 64, 128):
        raise ValueError("groups of 32, 64 or 128 columns")
    scale_dtype = w.dtype if scale_dtype is None else scale_dtype
    if scale_dtype not in _TYPES:
        raise TypeError("scale_dtype must be float32, float16 or bfloat16")
    lead, columns = w.shape[:-1], w.shape[-1]
    codes = torch.empty(*lead, (columns + 1) // 2, dtype=torch.uint8, device=w.device)
    scale = torch.empty(*lead, -(-columns // group), dtype=scale_dtype, device=w.device)
    zero = torch.empty(scale.shape, dtype=torch.uint8, device=w.device) if zeros else None
    check(load().lapis_b200_int4_quantise(_TYPES[w.dtype], lead.numel(), columns, _ptr(w), columns, group, _TYPES[scale_dtype], _ptr(codes), _ptr(scale),
                                          _ptr(zero), _stream()))
    return codes, scale, zero
