"""Performance cases of the operators around experts: what a program that serves or trains a model with routed experts calls.

``listed()`` holds the named cases, ``draw()`` makes further ones over the same ranges.  A case is a dict of plain values;
``prepare()`` builds what a caller holds before the call, ``run()`` is one pass.  ``own`` false: the plain form, elementary
torch operations in 32 bits, each result rounded once; ``own`` true: the calls of ``lapis_b200.experts``.

Operations (``op``):
  route     the largest k of a token's logits, their experts and weights (a softmax of all logits or of the chosen), or the
            gradient of the logits
  spread    tokens listed by expert and their rows copied into that order, or the gradient of that copy
  combine   rows of the experts back to their tokens, with weights applied, or its gradients
  product   few rows times 4-bit weights with a scale (and a zero) for every group of columns; for all rows the same
            weights, or those of the row's expert; ``gated``: silu of the first half of the outputs times the second half
  layer     a serving step's layer: route, list, gated product, product, combine
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new token of one request: latency
        {"name": "route_1x64_bf16", "op": "route", "backward": False, "tokens": 1, "experts": 64, "k": 6, "normalise": True, "dtype": "bf16",
         "padded": False},
        # a training step's batch, router in full precision, some experts switched off for some tokens, a few tokens of padding
        {"name": "route_16384x256_f32", "op": "route", "backward": False, "tokens": 16384, "experts": 256, "k": 8, "normalise": True,
         "dtype": "f32", "padded": True},
        # its backward pass, weights of the softmax over all experts
        {"name": "route_8191x130_bf16_bwd", "op": "route", "backward": True, "tokens": 8191, "experts": 130, "k": 5, "normalise": False,
         "dtype": "bf16", "padded": True},
        # a small serving batch: latency
        {"name": "spread_40_f16", "op": "spread", "backward": False, "tokens": 40, "experts": 60, "k": 4, "dim": 2048, "split": 1, "index": "i64",
         "dtype": "f16", "strided": False},
        # a training step's batch
        {"name": "spread_16384_bf16", "op": "spread", "backward": False, "tokens": 16384, "experts": 128, "k": 8, "dim": 2048, "split": 1,
         "index": "i32", "dtype": "bf16", "strided": False},
        # gradient in full precision, odd sizes, half of the experts held by another process
        {"name": "spread_5003_f32_bwd", "op": "spread", "backward": True, "tokens": 5003, "experts": 31, "k": 3, "dim": 1001, "split": 2,
         "index": "i32", "dtype": "f32", "strided": True},
        # back to the tokens of a training step
        {"name": "combine_16384_bf16", "op": "combine", "backward": False, "tokens": 16384, "experts": 128, "k": 8, "dim": 2048, "split": 1,
         "index": "i32", "dtype": "bf16", "strided": False},
        # its gradients, wider rows
        {"name": "combine_8192_bf16_bwd", "op": "combine", "backward": True, "tokens": 8192, "experts": 60, "k": 6, "dim": 5120, "split": 1,
         "index": "i32", "dtype": "bf16", "strided": False},
        # a projection for one new token: latency
        {"name": "product_1x4096x4096_bf16", "op": "product", "rows": 1, "outputs": 4096, "columns": 4096, "group": 128, "zeros": False, "gated": False,
         "dtype": "bf16", "scale": "bf16"},
        # a gated layer for 64 requests, groups with zeros
        {"name": "product_64x14336x4096_f16", "op": "product", "rows": 64, "outputs": 14336, "columns": 4096, "group": 64, "zeros": True, "gated": True,
         "dtype": "f16", "scale": "f16"},
        # gated experts for 48 requests, rows fetched from their tokens
        {"name": "product_48x8of128_bf16", "op": "product", "tokens": 48, "experts": 128, "k": 8, "fetch": True, "outputs": 2048, "columns": 2048, "group": 32,
         "zeros": False, "gated": True, "dtype": "bf16", "scale": "bf16", "split": 1, "index": "i32"},
        # all of a serving step's layer for 32 requests
        {"name": "layer_32x6of64_bf16", "op": "layer", "tokens": 32, "experts": 64, "k": 6, "dim": 2048, "hidden": 1408, "group": 128, "zeros": False,
         "dtype": "bf16", "scale": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Mostly what models have, a multiple of 64 or 16; one in four anything."""
    n, step = _log(rng, lo, hi), rng.choice([64, 64, 16, 1])
    return max(lo, n // step * step)


def draw(rng):
    op = rng.choice(["route", "spread", "combine", "product", "product", "layer"])
    experts = rng.choice([4, 8, 16, 31, 60, 64, 128, 130, 256, 384, 512])
    k = min(experts, rng.choice([1, 2, 3, 4, 5, 6, 8, 8, 10, 16]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    c = {"op": op, "dtype": dtype}
    if op == "route":
        return c | {"backward": rng.random() < 0.5, "tokens": _log(rng, 1, min(65536, 2 ** 23 // experts)), "experts": experts, "k": k,
                    "normalise": rng.random() < 0.6, "padded": rng.random() < 0.5}
    if op in ("spread", "combine"):
        dim = _size(rng, 16, 8192)
        most = min(65536, 9 * 10 ** 8 // ((1 + 2 * k) * dim * SIZE[dtype]), 2 ** 25 // (k * experts))
        return c | {"backward": rng.random() < 0.5, "tokens": _log(rng, 1, max(2, most)), "experts": experts, "k": k, "dim": dim,
                    "split": rng.choice([1, 1, 1, 2, 4]), "index": rng.choice(["i32", "i64"]), "strided": rng.random() < 0.3}
    group, zeros = rng.choice([32, 64, 128]), rng.random() < 0.4
    scale = rng.choice([dtype, dtype, "f32"])
    if op == "layer":
        experts, k = min(experts, 128), min(k, 8)
        tokens, dim = _log(rng, 1, 64), _size(rng, 64, 4096)
        most = min(2 ** 28 // experts, 18 * 10 ** 8 // (tokens * k))
        return c | {"tokens": tokens, "experts": experts, "k": k, "dim": dim, "hidden": _size(rng, 32, max(64, min(2048, most // (2 * dim)))),
                    "group": group, "zeros": zeros, "scale": scale}
    columns, gated = _size(rng, 32, 16384), rng.random() < 0.4
    c |= {"columns": columns, "group": group, "zeros": zeros, "gated": gated, "scale": scale}
    if rng.random() < 0.5:
        rows = _log(rng, 1, 256)
        return c | {"rows": rows, "outputs": 2 * _size(rng, 16, max(32, min(16384, 2 ** 27 // columns, 18 * 10 ** 8 // (rows * columns))))}
    experts, k = min(experts, 128), min(k, 8)
    tokens = _log(rng, 1, 128)
    most = min(2 ** 28 // experts, 2 ** 37 // (tokens * k * experts), 18 * 10 ** 8 // (tokens * k)) // columns
    return c | {"tokens": tokens, "experts": experts, "k": k, "fetch": rng.random() < 0.5, "outputs": 2 * _size(rng, 16, max(32, min(16384, most // 2))),
                "split": rng.choice([1, 1, 2]), "index": rng.choice(["i32", "i64"])}


def _weights_bytes(case, outputs, columns, of_experts):
    """Codes, scales and zeros of the experts that get a row, as many as that is on average where all are equally popular."""
    each = outputs * (columns / 2 + -(-columns // case["group"]) * (SIZE[case["scale"]] + (0.5 if case["zeros"] else 0)))
    if not of_experts:
        return each
    experts = case["experts"]
    return each * experts * (1 - (1 - case["k"] / (experts * case.get("split", 1))) ** case["tokens"])


def work(case):
    op, s = case["op"], SIZE[case["dtype"]]
    if op == "product" and "rows" in case:
        rows, n, cols = case["rows"], case["outputs"], case["columns"]
        out = n // 2 if case["gated"] else n
        return {"bytes": int(_weights_bytes(case, n, cols, False) + rows * (cols + out) * s), "flops": 2 * rows * n * cols}
    t, e, k = case["tokens"], case["experts"], case["k"]
    if op == "route":
        if case["backward"]:
            return {"bytes": t * e * s * (1 if case["normalise"] else 2) + t * k * (8 + (s if case["normalise"] else 0)), "flops": t * e * (1 if case["normalise"] else 5)}
        return {"bytes": t * e * s + t * k * 8, "flops": t * e * 5}
    if op == "layer":
        dim, hidden, rows = case["dim"], case["hidden"], t * k
        return {"bytes": int(_weights_bytes(case, 2 * hidden, dim, True) + _weights_bytes(case, dim, hidden, True) + 2 * t * dim * s + t * e * s),
                "flops": 6 * rows * dim * hidden}
    held = t * k // case["split"]  # slots whose expert is here
    if op == "product":
        n, cols = case["outputs"], case["columns"]
        out = n // 2 if case["gated"] else n
        return {"bytes": int(_weights_bytes(case, n, cols, True) + ((t if case["fetch"] else held) * cols + t * k * out) * s + (e + 1 + t * k) * 4),
                "flops": 2 * held * n * cols}
    dim, lists = case["dim"], t * k * 4
    if op == "spread":
        if case["backward"]:
            return {"bytes": (held + t) * dim * s + lists, "flops": held * dim}
        return {"bytes": (t + t * k) * dim * s + t * k * (4 if case["index"] == "i32" else 8) + 2 * lists + (e + 1) * 4, "flops": t * k}
    if case["backward"]:
        return {"bytes": (t + held + t * k) * dim * s + lists + 2 * t * k * 4, "flops": 3 * held * dim}
    return {"bytes": (held + t) * dim * s + lists + t * k * 4, "flops": 2 * held * dim}


# ---- inputs -----------------------------------------------------------------


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _uniform(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _logits(gen, tokens, experts, dtype):
    """Some experts are more popular than others."""
    return (1.5 * _normal(gen, tokens, experts) + 0.7 * _normal(gen, experts)).to(TYPES[dtype])


def _chosen(case, gen):
    """Experts of the tokens' slots as a router chose them; with ``split`` those of other processes are numbers outside [0, experts)."""
    experts, split = case["experts"], case["split"]
    first = (split // 2) * experts
    expert = _logits(gen, case["tokens"], experts * split, "f32").topk(case["k"], -1).indices - first
    return expert.to(torch.int32 if case["index"] == "i32" else torch.int64)


def _codes(case, gen, outputs, columns, experts=None):
    """4-bit weights: codes [.., outputs, ceil(columns / 2)], the even column in the low half of a byte, with a scale and perhaps a zero
    for every group of columns."""
    lead = (outputs,) if experts is None else (experts, outputs)
    half = (columns + 1) // 2
    low, high = ((2.7 * _normal(gen, *lead, half) + 8).round_().clamp_(0, 15).to(torch.uint8) for _ in range(2))
    groups = -(-columns // case["group"])
    scale = ((0.5 + _uniform(gen, *lead, groups)) * (0.37 * columns ** -0.5)).to(TYPES[case["scale"]])
    zero = (8 + 1.5 * _normal(gen, *lead, groups)).round_().clamp_(0, 15).to(torch.uint8) if case["zeros"] else None
    return {"codes": low | high << 4, "scale": scale, "zero": zero, "columns": columns, "group": case["group"]}


def _held(weights, gated=False):
    """What a program keeps of its weights."""
    if not own:
        return weights
    from lapis_b200 import experts
    return experts.Int4Matrix(weights["codes"], weights["scale"], weights["zero"], columns=weights["columns"], group=weights["group"], gated=gated)


def _rows(gen, rows, dim, dtype, strided=False):
    """Rows of a layer's input: a few channels are large.  ``strided``: part of wider rows."""
    x = _normal(gen, rows, dim + (24 if strided else 0)) * (1 + 4 * (_uniform(gen, dim + (24 if strided else 0)) < 0.02))
    return x.to(TYPES[dtype])[:, 16:16 + dim] if strided else x.to(TYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    op, dtype = case["op"], case["dtype"]
    s = {"case": case}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        s["logits"] = _logits(gen, t, e, dtype)
        if case["padded"]:
            s["logits"][_uniform(gen, t, e) < 0.1] = -math.inf
            s["logits"][t - t // 16:] = -math.inf
        if case["backward"]:
            s["dweights"] = _normal(gen, t, k)
            s["expert"] = _plain_route(s["logits"], k, case["normalise"])[1]
        return s
    if op == "layer":
        s["x"], s["logits"] = _rows(gen, case["tokens"], case["dim"], dtype), _logits(gen, case["tokens"], case["experts"], "f32")
        s["up"] = _held(_codes(case, gen, 2 * case["hidden"], case["dim"], case["experts"]), gated=True)
        s["down"] = _held(_codes(case, gen, case["dim"], case["hidden"], case["experts"]))
        return s
    if op == "product" and "rows" in case:
        s["x"] = _rows(gen, case["rows"], case["columns"], dtype)
        s["weights"] = _held(_codes(case, gen, case["outputs"], case["columns"]), case["gated"])
        return s
    t, k, slots = case["tokens"], case["k"], case["tokens"] * case["k"]
    s["expert"] = _chosen(case, gen)
    if op == "product":
        s["x"] = _rows(gen, t if case["fetch"] else slots, case["columns"], dtype)
        s["weights"] = _held(_codes(case, gen, case["outputs"], case["columns"], case["experts"]), case["gated"])
    elif op == "spread" and not case["backward"]:
        s["x"] = _rows(gen, t, case["dim"], dtype, case["strided"])
        return s
    else:
        s["rows"] = _rows(gen, slots, case["dim"], dtype, case["strided"])
        if op == "combine":
            w = _uniform(gen, t, k) + 0.1
            s["weights"] = w / w.sum(-1, keepdim=True)
            if case["backward"]:
                s["dout"] = _rows(gen, t, case["dim"], dtype, case["strided"])
    if own:
        from lapis_b200 import experts
        s["lists"] = experts.ExpertLists(s["expert"], case["experts"])
    else:
        s["lists"] = _plain_lists(s["expert"], case["experts"])
    return s


# ---- one pass ---------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from lapis_b200 import experts as E
    c = s["case"]
    op = c["op"]
    if op == "route":
        if c["backward"]:
            return {"dlogits": E.route_backward(s["dweights"], s["logits"], s["expert"], normalise=c["normalise"])}
        weights, expert = E.route(s["logits"], c["k"], normalise=c["normalise"])
        return {"weights": weights, "expert": expert}
    if op == "layer":
        weights, expert = E.route(s["logits"], c["k"])
        lists = E.ExpertLists(expert, c["experts"])
        rows = s["down"].matmul(s["up"].matmul(s["x"], lists, fetch=True), lists)
        return {"out": lists.combine(rows, weights), "expert": expert}
    if op == "product":
        return {"y": s["weights"].matmul(s["x"], s["lists"], fetch=c["fetch"]) if "lists" in s else s["weights"].matmul(s["x"])}
    if op == "spread":
        if c["backward"]:
            return {"dx": s["lists"].gather_backward(s["rows"])}
        lists = E.ExpertLists(s["expert"], c["experts"])
        return {"pos": lists.pos, "crd": lists.crd, "place": lists.place, "rows": lists.gather(s["x"])}
    if c["backward"]:
        drows, dweights = s["lists"].combine_backward(s["dout"], s["rows"], s["weights"])
        return {"drows": drows, "dweights": dweights}
    return {"out": s["lists"].combine(s["rows"], s["weights"])}


def _plain_route(logits, k, normalise):
    x = logits.float()
    number = torch.arange(x.shape[1], device=DEV)
    left, expert = x.clone(), []
    for _ in range(k):  # the largest that is left, of equal ones the first
        most = left.amax(-1, keepdim=True)
        at = torch.where((left == most) & (most > -math.inf), number, x.shape[1]).amin(-1)
        expert.append(torch.where(at < x.shape[1], at, -1))
        left = torch.where(number == at[:, None], -math.inf, left)
    expert = torch.stack(expert, -1)
    chosen = expert >= 0
    most = x.amax(-1, keepdim=True)
    most = torch.where(most > -math.inf, most, 0.0)
    e = torch.where(chosen, torch.exp(x.gather(-1, expert.clamp(min=0)) - most), 0.0)
    total = (e if normalise else torch.exp(x - most)).sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), expert.int()


def _plain_route_backward(dweights, logits, expert, normalise):
    x, chosen, at = logits.float(), expert >= 0, expert.clamp(min=0).long()
    most = x.amax(-1, keepdim=True)
    most = torch.where(most > -math.inf, most, 0.0)
    e = torch.exp(x - most)
    mine = torch.where(chosen, e.gather(-1, at), 0.0)
    total = (mine if normalise else e).sum(-1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    w = mine / total
    inner = (w * dweights).sum(-1, keepdim=True)
    if normalise:
        dx, of_chosen = torch.zeros_like(x), w * (dweights - inner)
    else:
        dx, of_chosen = -(e / total) * inner, w * dweights
    return dx.scatter_add(-1, at, torch.where(chosen, of_chosen, 0.0))


def _plain_lists(expert, experts):
    """Slots (token * k + j) sorted by expert, those of no expert here last: where each expert's begin, the slots, and each slot's place."""
    e = expert.flatten()
    bucket = torch.where((e >= 0) & (e < experts), e, experts).long()
    upto = (bucket == torch.arange(experts + 1, device=DEV)[:, None]).cumsum(-1, dtype=torch.int32)
    count = upto[:, -1].long()
    begin = count.cumsum(0) - count
    place = begin[bucket] + upto.gather(0, bucket[None])[0] - 1
    crd = torch.empty_like(place)
    crd[place] = torch.arange(len(e), device=DEV)
    return {"pos": begin.int(), "crd": crd.int(), "place": place.int().view(expert.shape)}


def _dense(weights):
    """[.., outputs, columns] in 32 bits."""
    codes = torch.stack([weights["codes"] & 15, weights["codes"] >> 4], -1).flatten(-2)[..., :weights["columns"]].float()
    scale, zero = (t if t is None else t.float().repeat_interleave(weights["group"], -1)[..., :weights["columns"]] for t in (weights["scale"], weights["zero"]))
    return (codes - (8.0 if zero is None else zero)) * scale


def _plain_product(x, weights, gated, lists=None):
    """Rows x in 32 bits; ``lists``: each row times the weights of its expert, zeros for rows of no expert here."""
    if lists is None:
        y = x @ _dense(weights).T
    else:
        row = torch.arange(len(x), device=DEV)
        y = torch.zeros(len(x), weights["codes"].shape[1], device=DEV)
        for e in range(weights["codes"].shape[0]):
            w = _dense({n: t[e] if isinstance(t, torch.Tensor) else t for n, t in weights.items()})
            y = torch.where(((row >= lists["pos"][e]) & (row < lists["pos"][e + 1]))[:, None], x @ w.T, y)
    if gated:
        a, b = y.chunk(2, -1)
        y = a / (1 + torch.exp(-a)) * b
    return y


def _plain_combine(rows, weights, lists):
    """Sums in 32 bits of the rows that are here."""
    place = lists["place"].long()
    got = torch.where((place < lists["pos"][-1])[..., None], rows[place].float(), 0.0)
    return (got if weights is None else got * weights[..., None]).sum(1)


def _plain(s):
    c = s["case"]
    op, dt = c["op"], TYPES[c["dtype"]]
    if op == "route":
        if c["backward"]:
            return {"dlogits": _plain_route_backward(s["dweights"], s["logits"], s["expert"], c["normalise"]).to(dt)}
        weights, expert = _plain_route(s["logits"], c["k"], c["normalise"])
        return {"weights": weights, "expert": expert}
    if op == "layer":
        weights, expert = _plain_route(s["logits"], c["k"], True)
        lists = _plain_lists(expert, c["experts"])
        h = _plain_product(s["x"].float()[lists["crd"].long() // c["k"]], s["up"], True, lists).to(dt)
        return {"out": _plain_combine(_plain_product(h.float(), s["down"], False, lists).to(dt), weights, lists).to(dt), "expert": expert}
    if op == "product":
        x, lists = s["x"].float(), s.get("lists")
        if lists is not None and c["fetch"]:
            x = x[lists["crd"].long() // c["k"]]
        return {"y": _plain_product(x, s["weights"], c["gated"], lists).to(dt)}
    if op == "spread":
        if c["backward"]:
            return {"dx": _plain_combine(s["rows"], None, s["lists"]).to(dt)}
        lists = _plain_lists(s["expert"], c["experts"])
        here = torch.arange(len(lists["crd"]), device=DEV) < lists["pos"][-1]
        return lists | {"rows": torch.where(here[:, None], s["x"][lists["crd"].long() // c["k"]], 0.0)}
    if not c["backward"]:
        return {"out": _plain_combine(s["rows"], s["weights"], s["lists"]).to(dt)}
    place, dout = s["lists"]["place"].long(), s["dout"].float()
    here = place < s["lists"]["pos"][-1]
    drows = torch.zeros(s["rows"].shape, device=DEV)
    drows[place] = torch.where(here[..., None], dout[:, None] * s["weights"][..., None], 0.0)
    dweights = torch.where(here, (s["rows"][place].float() * dout[:, None]).sum(-1), 0.0)
    return {"drows": drows.to(dt), "dweights": dweights}


# ---- the same from the definitions, in 64 bits --------------------------------


def _exact_weights(w):
    """4-bit weights as numbers of 64 bits."""
    columns = torch.arange(w["columns"], device=DEV)
    code = (w["codes"][..., columns // 2] >> (4 * (columns % 2)).to(torch.uint8)) & 15
    of = columns // w["group"]
    return (code.double() - (8 if w["zero"] is None else w["zero"].double()[..., of])) * w["scale"].double()[..., of]


def _exact_route(logits, k, normalise):
    x = logits.double()
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    none = order.values[:, :k] == -math.inf
    if normalise:
        p = torch.softmax(order.values[:, :k], -1)
    else:
        p = torch.exp(order.values[:, :k] - torch.logsumexp(x, -1, keepdim=True))
    return torch.where(none, 0.0, p), torch.where(none, -1, order.indices[:, :k])


def _exact_lists(expert, experts):
    e = expert.cpu().numpy().reshape(-1).astype(np.int64)
    e[(e < 0) | (e >= experts)] = experts
    crd = np.argsort(e, kind="stable")
    place = np.empty_like(crd)
    place[crd] = np.arange(len(crd))
    return np.concatenate([[0], np.cumsum(np.bincount(e, minlength=experts + 1))])[:experts + 1], crd, place.reshape(expert.shape)


def _exact_product(x, weights, gated, pos=None):
    def act(y):
        half = y.shape[-1] // 2
        return y[..., :half] * torch.sigmoid(y[..., :half]) * y[..., half:] if gated else y
    if pos is None:
        return act(x @ _exact_weights(weights).T)
    outputs = weights["codes"].shape[1]
    y = torch.zeros(len(x), outputs // 2 if gated else outputs, dtype=torch.float64, device=DEV)
    for e in range(len(pos) - 1):
        if pos[e] < pos[e + 1]:
            y[pos[e]:pos[e + 1]] = act(x[pos[e]:pos[e + 1]] @ _exact_weights({n: t[e] if isinstance(t, torch.Tensor) else t for n, t in weights.items()}).T)
    return y


def exact(case, seed):
    global own
    before, own = own, False  # the weights as they were given
    try:
        s = prepare(case, seed)
    finally:
        own = before
    op = case["op"]
    if op == "route":
        if not case["backward"]:
            weights, expert = _exact_route(s["logits"], case["k"], case["normalise"])
            return {"weights": weights, "expert": expert.int()}
        x = s["logits"].double()
        chosen, at = s["expert"] >= 0, s["expert"].clamp(min=0).long()
        dead = (x == -math.inf).all(-1)
        if case["normalise"]:
            kept = torch.full_like(x, -math.inf).scatter(-1, torch.where(chosen, at, at[:, :1]), x.gather(-1, torch.where(chosen, at, at[:, :1])))
        else:
            kept = x
        p = torch.softmax(torch.where(dead[:, None], 0.0, kept), -1)
        g = torch.zeros_like(x).scatter_add(-1, at, torch.where(chosen, s["dweights"].double(), 0.0))
        return {"dlogits": torch.where(dead[:, None], 0.0, p * (g - (g * p).sum(-1, keepdim=True)))}
    if op == "product" and "rows" in case:
        return {"y": _exact_product(s["x"].double(), s["weights"], case["gated"])}
    if op == "layer":
        weights, expert = _exact_route(s["logits"], case["k"], True)
    else:
        weights, expert = s.get("weights"), s["expert"]
    pos, crd, place = _exact_lists(expert, case["experts"])
    token = torch.from_numpy(crd // case["k"]).to(DEV)
    at, here = torch.from_numpy(place).to(DEV), torch.from_numpy(place < pos[-1]).to(DEV)
    pos = pos.tolist()
    if op == "product":
        x = s["x"].double()
        return {"y": _exact_product(x[token] if case["fetch"] else x, s["weights"], case["gated"], pos)}
    if op == "layer":
        rows = _exact_product(_exact_product(s["x"].double()[token], s["up"], True, pos), s["down"], False, pos)
        return {"out": torch.einsum("tk,tkd->td", weights, rows[at]), "expert": expert.int()}
    if op == "spread" and not case["backward"]:
        rows = s["x"].double()[token]
        rows[pos[-1]:] = 0
        return {"pos": torch.tensor(pos, device=DEV, dtype=torch.int32), "crd": torch.from_numpy(crd).to(DEV, torch.int32), "place": at.int(), "rows": rows}
    got, weight = {}, here.double() if op == "spread" else torch.where(here, weights.double(), 0.0)
    if op == "combine" and case["backward"]:
        got = {"drows": torch.zeros(s["rows"].shape, dtype=torch.float64, device=DEV), "dweights": torch.zeros(weights.shape, dtype=torch.float64, device=DEV)}
    else:
        out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device=DEV)
    for j in range(case["k"]):  # one slot of every token at a time
        if got:
            dout = s["dout"].double()
            got["drows"][at[:, j]] = dout * weight[:, j, None]
            got["dweights"][:, j] = torch.where(here[:, j], (s["rows"][at[:, j]].double() * dout).sum(-1), 0.0)
        else:
            out += s["rows"][at[:, j]].double() * weight[:, j, None]
    return got or {"dx" if op == "spread" else "out": out}
