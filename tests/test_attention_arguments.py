"""Operands that the calls around attention cannot use: exceptions and statuses, without a GPU."""
import ctypes

import pytest
import torch

from lapis_b200 import _lib


def _unbacked(shape, dtype=torch.bfloat16):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True):
        return torch.empty(shape, dtype=dtype, device="cuda")  # a CUDA tensor without storage


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


class Heads(ctypes.Structure):
    _fields_ = [("d", ctypes.c_void_p), ("heads", ctypes.c_int64), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class How(ctypes.Structure):
    _fields_ = [("d_q_weight", ctypes.c_void_p), ("d_k_weight", ctypes.c_void_p), ("weight_type", ctypes.c_int), ("d_cos", ctypes.c_void_p),
                ("d_sin", ctypes.c_void_p), ("places", ctypes.c_int64), ("rot", ctypes.c_int64), ("interleaved", ctypes.c_int), ("eps", ctypes.c_double)]


class Lists(ctypes.Structure):
    _fields_ = [("idx_bytes", ctypes.c_int), ("rows", ctypes.c_int64), ("entries", ctypes.c_int64), ("d_pos", ctypes.c_void_p), ("d_crd", ctypes.c_void_p)]


OK, BADSHAPE, BADARG, TOOBIG = 0, 1, 4, 6
F32, F16, BF16, I8, E4M3 = range(5)


def changed(struct, **fields):
    new = type(struct).from_buffer_copy(struct)
    for name, value in fields.items():
        setattr(new, name, value)
    return new


HEADS, HOW, LISTS = Heads(64, 4, 512, 128), How(64, 64, F32, 64, 64, 100, 128, 0, 1e-6), Lists(4, 3, 10, 64, 64)
CACHE = _lib.KvCache(BF16, 10, 4, 16, 128, 64, 64, 64, 64)


def ref(x):
    return None if x is None else ctypes.addressof(x)


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": I8}), (BADARG, {"q": None}), (BADARG, {"how": None}), (BADSHAPE, {"tokens": -1}), (BADSHAPE, {"dim": 0}),
    (TOOBIG, {"dim": 257}), (TOOBIG, {"tokens": 2 ** 31}), (BADARG, {"q": changed(HEADS, d=None)}), (BADSHAPE, {"q": changed(HEADS, heads=-1)}),
    (BADSHAPE, {"how": changed(HOW, rot=130)}), (BADSHAPE, {"how": changed(HOW, rot=3)}), (BADSHAPE, {"how": changed(HOW, places=-1)}),
    (BADARG, {"how": changed(HOW, weight_type=F16)}), (BADARG, {"how": changed(HOW, d_k_weight=None)}), (BADARG, {"how": changed(HOW, d_sin=None)}),
    (BADARG, {"how": changed(HOW, eps=-1.0)}), (BADARG, {"how": changed(HOW, eps=float("nan"))}), (BADARG, {"idx": 2}), (BADARG, {"place": None}),
    (BADARG, {"out": None}), (OK, {"tokens": 0}), (OK, {"tokens": 0, "place": None, "out": None, "q": changed(HEADS, d=None)}),
])
def test_rotate_refuses(lib, want, kw):
    a = {"type": BF16, "tokens": 7, "dim": 128, "q": HEADS, "k": HEADS, "how": HOW, "idx": 4, "place": 64, "out": 64} | kw
    got = lib.lapis_b200_qk_norm_rope(a["type"], a["tokens"], a["dim"], ref(a["q"]), ref(a["k"]), ref(a["how"]), a["idx"], a["place"], a["out"], a["out"], None)
    assert got == want == lib.lapis_last_error()
    if want == OK:
        return
    got = lib.lapis_b200_qk_norm_rope_backward(a["type"], a["tokens"], a["dim"], ref(a["q"]), ref(a["k"]), ref(a["q"]), ref(a["k"]), ref(a["how"]), a["idx"],
                                               a["place"], a["out"], a["out"], 64, 64, None)
    assert got == want and b"backward" in lib.lapis_last_error_message()


def test_backward_refuses(lib):
    def call(dq=HEADS, dw=64):
        return lib.lapis_b200_qk_norm_rope_backward(BF16, 7, 128, ref(dq), ref(HEADS), ref(HEADS), ref(HEADS), ref(HOW), 4, 64, 64, 64, dw, 64, None)
    assert call(changed(HEADS, heads=3)) == BADSHAPE
    assert call(dw=None) == BADARG


BAD_CACHES = [
    (BADARG, None), (BADARG, changed(CACHE, type=7)), (BADSHAPE, changed(CACHE, pages=-1)), (BADSHAPE, changed(CACHE, heads=0)),
    (BADSHAPE, changed(CACHE, page_size=0)), (BADSHAPE, changed(CACHE, dim=0)), (TOOBIG, changed(CACHE, dim=264)), (TOOBIG, changed(CACHE, pages=2 ** 26)),
    (TOOBIG, changed(CACHE, pages=2 ** 62)), (BADARG, changed(CACHE, d_k=None)), (BADARG, changed(CACHE, type=I8, d_v_scale=None)),
    (BADARG, changed(CACHE, type=E4M3, d_k_scale=None)),
]
BAD_LISTS = [(BADARG, None), (BADARG, changed(LISTS, idx_bytes=3)), (BADSHAPE, changed(LISTS, rows=-1)), (BADSHAPE, changed(LISTS, entries=-1)),
             (BADARG, changed(LISTS, d_pos=None)), (BADARG, changed(LISTS, d_crd=None))]


@pytest.mark.parametrize("want,cache,lists", [(w, c, LISTS) for w, c in BAD_CACHES] + [(w, CACHE, x) for w, x in BAD_LISTS])
def test_bad_caches_and_lists_are_refused(lib, want, cache, lists):
    for how in (None, ref(HOW)):
        assert lib.lapis_b200_kv_append(BF16, 7, ref(HEADS), ref(HEADS), ref(HEADS), how, ref(cache), ref(lists), 64, 64, 64, None) == want
    assert lib.lapis_b200_kv_read(ref(cache), ref(lists), 7, 64, 64, BF16, 64, 64, None) == want
    assert lib.lapis_b200_paged_attention(BF16, 3, ref(HEADS), ref(cache), ref(lists), 64, 1.0, 0, 64, None, None) == want


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": E4M3}), (BADARG, {"type": F16}), (BADARG, {"k": None}), (BADARG, {"v": changed(HEADS, d=None)}), (BADSHAPE, {"k": changed(HEADS, heads=2)}),
    (BADSHAPE, {"tokens": -1}), (BADARG, {"row": None}), (BADARG, {"place": None}), (BADARG, {"how": HOW, "q": None}), (BADARG, {"how": HOW, "out": None}),
    (BADSHAPE, {"how": changed(HOW, rot=-2)}), (TOOBIG, {"tokens": 2 ** 31}), (OK, {"tokens": 0}), (OK, {"tokens": 0, "row": None, "place": None}),
])
def test_append_refuses(lib, want, kw):
    a = {"type": BF16, "tokens": 7, "q": HEADS, "k": HEADS, "v": HEADS, "how": None, "row": 64, "place": 64, "out": 64} | kw
    assert lib.lapis_b200_kv_append(a["type"], a["tokens"], ref(a["q"]), ref(a["k"]), ref(a["v"]), ref(a["how"]), ref(CACHE), ref(LISTS), a["row"], a["place"],
                                    a["out"], None) == want


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": I8}), (BADSHAPE, {"tokens": -1}), (BADARG, {"row": None}), (BADARG, {"k": None}), (TOOBIG, {"tokens": 2 ** 31}), (OK, {"tokens": 0, "k": None}),
])
def test_read_refuses(lib, want, kw):
    a = {"type": F32, "tokens": 7, "row": 64, "k": 64} | kw
    assert lib.lapis_b200_kv_read(ref(CACHE), ref(LISTS), a["tokens"], a["row"], 64, a["type"], a["k"], 64, None) == want


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": I8}), (BADARG, {"type": F16}), (BADARG, {"q": None}), (BADARG, {"q": changed(HEADS, d=None)}), (BADSHAPE, {"q": changed(HEADS, heads=6)}),
    (BADSHAPE, {"q": changed(HEADS, heads=0)}), (BADSHAPE, {"requests": -1}), (BADSHAPE, {"requests": 4}), (TOOBIG, {"requests": 65536}),
    (TOOBIG, {"q": changed(HEADS, heads=2 ** 17)}), (BADARG, {"window": -1}), (BADARG, {"scale": float("inf")}), (BADARG, {"scale": float("nan")}),
    (BADARG, {"length": None}), (BADARG, {"out": None}), (OK, {"requests": 0, "lists": changed(LISTS, rows=0), "out": None, "length": None}),
])
def test_attention_refuses(lib, want, kw):
    a = {"type": BF16, "requests": 3, "q": HEADS, "lists": LISTS, "length": 64, "scale": 0.1, "window": 0, "out": 64} | kw
    assert lib.lapis_b200_paged_attention(a["type"], a["requests"], ref(a["q"]), ref(CACHE), ref(a["lists"]), a["length"], a["scale"], a["window"], a["out"],
                                          None, None) == want


def test_structures_are_those_of_the_header():
    """Sizes and offsets by the host compiler's rules: C structures of natural alignment."""
    assert ctypes.sizeof(_lib.KvCache) == 72 and _lib.KvCache.d_k.offset == 40
    assert ctypes.sizeof(How) == 72 and How.d_cos.offset == 24 and How.eps.offset == 64
    assert ctypes.sizeof(Lists) == 40 and ctypes.sizeof(Heads) == 32


@pytest.mark.parametrize("make,error", [
    (lambda t: (t((2, 3, 4, 8), torch.float64), t((2, 3, 4, 8), torch.float64)), TypeError),
    (lambda t: (t((2, 3, 4, 8)), t((2, 3, 4, 8), torch.float16)), TypeError),
    (lambda t: (t((2, 3, 4, 8)), t((2, 3, 5, 8))), ValueError),
    (lambda t: (t((2, 3, 8)), t((2, 3, 8))), ValueError),
    (lambda t: (t((2, 3, 0, 8)), t((2, 3, 0, 8))), ValueError),
    (lambda t: (t((2, 3, 4, 264)), t((2, 3, 4, 264))), ValueError),
    (lambda t: (t((2, 3, 4, 8)).transpose(1, 2), t((2, 3, 4, 8)).transpose(1, 2)), TypeError),
    (lambda t: (t((2, 3, 4, 8), torch.int8), t((2, 3, 4, 8), torch.int8)), ValueError),
    (lambda t: (t((2, 3, 4, 8)), t((2, 3, 4, 8)), t((2, 3, 4), torch.float32), t((2, 3, 4), torch.float32)), ValueError),
    (lambda t: (t((2, 3, 4, 8), torch.int8), t((2, 3, 4, 8), torch.int8), t((2, 3, 4), torch.float16), t((2, 3, 4), torch.float32)), TypeError),
    (lambda t: (t((2, 3, 4, 8), torch.int8), t((2, 3, 4, 8), torch.int8), t((2, 3, 5), torch.float32), t((2, 3, 4), torch.float32)), ValueError),
    (lambda t: (torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 4, 8)), TypeError),
])
def test_caches_of_other_tensors_raise(make, error):
    from lapis_b200 import attention
    with pytest.raises(error):
        attention.PagedCache(*make(_unbacked))
