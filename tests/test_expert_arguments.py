"""Operands that the calls of a layer of experts cannot use: exceptions and statuses, without a GPU."""
import ctypes

import pytest
import torch

from lapis_b200 import _lib

OK, BADSHAPE, BADARG, TOOBIG = 0, 1, 4, 6
F32, F16, BF16, I8, E4M3 = range(5)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def ref(x):
    return None if x is None else ctypes.addressof(x)


def changed(struct, **fields):
    new = type(struct).from_buffer_copy(struct)
    for name, value in fields.items():
        setattr(new, name, value)
    return new


LISTS = _lib.ExpertLists(8, 2, 4, 64, 64, 64)
WEIGHTS = _lib.Int4(4, 32, 64, 32, BF16, 0, 0, 64)


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": I8}), (BADSHAPE, {"tokens": -1}), (BADSHAPE, {"experts": -1}), (BADSHAPE, {"k": -1}), (BADSHAPE, {"k": 9}), (TOOBIG, {"experts": 1025}),
    (TOOBIG, {"experts": 64, "k": 33}), (TOOBIG, {"tokens": 2 ** 31}), (BADARG, {"logits": None}), (BADARG, {"weights": None}), (BADARG, {"expert": None}),
    (OK, {"tokens": 0}), (OK, {"tokens": 0, "logits": None, "weights": None, "expert": None}), (OK, {"k": 0, "weights": None, "expert": None}),
])
def test_route(lib, want, kw):
    a = dict(type=BF16, tokens=4, experts=8, logits=64, stride=8, k=2, weights=64, expert=64) | kw
    assert lib.lapis_b200_route(a["type"], a["tokens"], a["experts"], a["logits"], a["stride"], a["k"], 1, a["weights"], a["expert"], None) == want


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": E4M3}), (BADSHAPE, {"tokens": -1}), (BADSHAPE, {"k": 9}), (TOOBIG, {"experts": 2000}), (BADARG, {"logits": None}), (BADARG, {"expert": None}),
    (BADARG, {"dweights": None}), (BADARG, {"dlogits": None}), (OK, {"tokens": 0, "logits": None, "dlogits": None}), (OK, {"experts": 0, "k": 0, "logits": None}),
])
def test_route_backward(lib, want, kw):
    a = dict(type=BF16, tokens=4, experts=8, logits=64, stride=8, k=2, expert=64, dweights=64, dlogits=64) | kw
    assert lib.lapis_b200_route_backward(a["type"], a["tokens"], a["experts"], a["logits"], a["stride"], a["k"], 1, a["expert"], a["dweights"], a["dlogits"],
                                         None) == want


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"idx": 2}), (BADSHAPE, {"tokens": -1}), (BADSHAPE, {"k": -1}), (BADSHAPE, {"experts": -1}), (TOOBIG, {"experts": 1025}), (TOOBIG, {"tokens": 2 ** 30}),
    (BADARG, {"expert": None}), (BADARG, {"pos": None}), (BADARG, {"crd": None}), (BADARG, {"place": None}),
])
def test_lists(lib, want, kw):
    a = dict(idx=4, tokens=4, k=2, experts=8, expert=64, pos=64, crd=64, place=64) | kw
    assert lib.lapis_b200_expert_lists_make(a["idx"], a["tokens"], a["k"], a["experts"], a["expert"], a["pos"], a["crd"], a["place"], None) == want


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": I8}), (BADSHAPE, {"dim": -1}), (TOOBIG, {"dim": 2 ** 31}), (BADARG, {"lists": None}), (BADSHAPE, {"lists": changed(LISTS, k=-1)}),
    (TOOBIG, {"lists": changed(LISTS, experts=1025)}), (BADARG, {"lists": changed(LISTS, d_pos=None)}), (BADARG, {"lists": changed(LISTS, d_place=None)}),
    (BADARG, {"x": None}), (BADARG, {"out": None}), (OK, {"dim": 0, "x": None, "out": None}),
    (OK, {"lists": changed(LISTS, tokens=0, d_crd=None, d_place=None), "x": None, "out": None}),
])
def test_rows(lib, want, kw):
    a = dict(type=BF16, dim=16, x=64, lists=LISTS, out=64) | kw
    assert lib.lapis_b200_expert_gather(a["type"], a["dim"], a["x"], 16, ref(a["lists"]), a["out"], None) == want
    assert lib.lapis_b200_expert_combine(a["type"], a["dim"], a["x"], 16, ref(a["lists"]), 64, a["out"], None) == want
    if a["dim"] != 0:
        assert lib.lapis_b200_expert_combine_backward(a["type"], a["dim"], a["x"], 16, a["x"], 16, ref(a["lists"]), 64, a["out"], 64, None) == want


def test_rows_backward_needs_weights(lib):
    assert lib.lapis_b200_expert_combine_backward(BF16, 16, 64, 16, 64, 16, ref(LISTS), None, 64, 64, None) == BADARG
    assert lib.lapis_b200_expert_combine_backward(BF16, 16, 64, 16, 64, 16, ref(LISTS), 64, 64, None, None) == BADARG


BAD_WEIGHTS = [(BADSHAPE, {"experts": -1}), (BADSHAPE, {"outputs": -1}), (BADSHAPE, {"columns": -1}), (BADSHAPE, {"group": 48}), (BADARG, {"scale_type": I8}),
               (BADSHAPE, {"gated": 1, "outputs": 33}), (TOOBIG, {"experts": 1025}), (TOOBIG, {"columns": 2 ** 25}), (TOOBIG, {"outputs": 2 ** 25})]


@pytest.mark.parametrize("want,fields", BAD_WEIGHTS)
def test_weights(lib, want, fields):
    w = changed(WEIGHTS, **fields)
    assert lib.lapis_b200_int4_bytes(ref(w)) == -1 and lib.lapis_last_error() == want
    assert lib.lapis_b200_int4_pack(ref(w), 64, 64, 64, 64, None) == want
    assert lib.lapis_b200_int4_matmul(BF16, ref(w), 16, 64, 64, ref(LISTS), 0, 64, None) == want


def test_weights_sizes(lib):
    """Codes in strips of 16 outputs and blocks of 64 columns, scales and zeros in records of 256 columns."""
    assert lib.lapis_b200_int4_bytes(ref(WEIGHTS)) == 4 * 2 * (512 + 16 * 8 * 2)
    assert lib.lapis_b200_int4_bytes(ref(changed(WEIGHTS, scale_type=F32, zeros=1))) == 4 * 2 * (512 + 16 * 8 * 4 + 16 * 8 // 2)
    assert lib.lapis_b200_int4_bytes(ref(changed(WEIGHTS, outputs=34, columns=65, group=128))) == 4 * 3 * (1024 + 16 * 2 * 2)
    assert lib.lapis_b200_int4_bytes(ref(changed(WEIGHTS, outputs=34, gated=1, group=64))) == 4 * 3 * (512 + 16 * 4 * 2)
    assert lib.lapis_b200_int4_bytes(ref(changed(WEIGHTS, columns=0))) == 0 and lib.lapis_b200_int4_bytes(None) == -1
    # beyond 32 bits
    assert lib.lapis_b200_int4_bytes(ref(changed(WEIGHTS, experts=1024, outputs=2 ** 20, columns=2 ** 20, group=128))) == 2 ** 50 // 2 + 2 ** 50 // 64


@pytest.mark.parametrize("want,kw", [
    (BADARG, {"type": I8}), (BADARG, {"w": None}), (BADSHAPE, {"rows": -1}), (TOOBIG, {"rows": 2 ** 31, "lists": None, "w": changed(WEIGHTS, experts=1)}),
    (BADSHAPE, {"lists": None}), (BADSHAPE, {"lists": changed(LISTS, experts=5)}), (BADSHAPE, {"rows": 8}), (BADSHAPE, {"fetch": 1}), (BADARG, {"x": None}),
    (BADARG, {"y": None}), (BADARG, {"w": changed(WEIGHTS, d_packed=None)}), (BADARG, {"lists": changed(LISTS, d_crd=None)}),
    (OK, {"rows": 0, "lists": changed(LISTS, tokens=0), "x": None, "y": None}), (OK, {"w": changed(WEIGHTS, outputs=0, d_packed=None), "x": None, "y": None}),
])
def test_matmul(lib, want, kw):
    a = dict(type=BF16, w=WEIGHTS, rows=16, x=64, lists=LISTS, fetch=0, y=64) | kw
    assert lib.lapis_b200_int4_matmul(a["type"], ref(a["w"]), a["rows"], a["x"], 64, ref(a["lists"]), a["fetch"], a["y"], None) == want


@pytest.mark.parametrize("want,kw", [(BADARG, {"type": E4M3}), (BADSHAPE, {"rows": -1}), (BADSHAPE, {"group": 16}), (BADARG, {"scale_type": I8}),
                                     (BADARG, {"w": None}), (BADARG, {"codes": None}), (BADARG, {"scale": None}), (OK, {"rows": 0, "w": None})])
def test_quantise(lib, want, kw):
    a = dict(type=F32, rows=4, columns=64, w=64, group=32, scale_type=F32, codes=64, scale=64) | kw
    assert lib.lapis_b200_int4_quantise(a["type"], a["rows"], a["columns"], a["w"], 64, a["group"], a["scale_type"], a["codes"], a["scale"], None, None) == want


def test_pack_wants_its_operands(lib):
    for args in ((None, 64, 64, 64), (64, None, 64, 64), (64, 64, 64, None), (64, 64, 64, 72)):
        assert lib.lapis_b200_int4_pack(ref(WEIGHTS), *args, None) == BADARG
    assert lib.lapis_b200_int4_pack(ref(changed(WEIGHTS, zeros=1)), 64, 64, None, 64, None) == BADARG


# ---- the calls over torch tensors -----------------------------------------------------


@pytest.fixture(scope="module")
def X():
    from lapis_b200 import experts
    return experts


def on_cpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_tensors_of_another_kind(X):
    for logits in (None, 3, on_cpu(4, 8), on_cpu(4, 8, dtype=torch.float64)):
        with pytest.raises(TypeError, match="logits"):
            X.route(logits, 2)
        with pytest.raises(TypeError, match="logits"):
            X.route_backward(on_cpu(4, 2), logits, on_cpu(4, 2, dtype=torch.int32))
    with pytest.raises(TypeError):
        X.route(on_cpu(4, 8), "2")
    for expert in (None, on_cpu(4, 2, dtype=torch.int32), on_cpu(4, 2)):
        with pytest.raises(TypeError, match="expert"):
            X.ExpertLists(expert, 4)
    for codes in (None, on_cpu(4, 8, dtype=torch.uint8)):
        with pytest.raises(TypeError, match="codes"):
            X.Int4Matrix(codes, on_cpu(4, 1), columns=16)
    with pytest.raises(TypeError, match="w must"):
        X.quantise_int4(on_cpu(4, 64))


def lists_of(X, tokens=4, k=2, experts=4):
    lists = X.ExpertLists.__new__(X.ExpertLists)
    lists.pos, lists.crd, lists.place = (on_cpu(*s, dtype=torch.int32) for s in ((experts + 1,), (tokens * k,), (tokens, k)))
    return lists


def test_rows_of_another_kind(X):
    lists = lists_of(X)
    for rows in (None, on_cpu(4, 16), on_cpu(4, 16, dtype=torch.int32)):
        with pytest.raises(TypeError, match="x must"):
            lists.gather(rows)
        with pytest.raises(TypeError, match="rows must"):
            lists.combine(rows, on_cpu(4, 2))
        with pytest.raises(TypeError, match="drows must"):
            lists.gather_backward(rows)
        with pytest.raises(TypeError, match="rows must"):
            lists.combine_backward(on_cpu(4, 16), rows, on_cpu(4, 2))
    with pytest.raises(TypeError, match="weights"):
        lists.combine(on_cpu(8, 16), None)
    assert lists.experts == 4
