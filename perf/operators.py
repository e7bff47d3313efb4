"""Performance cases of the operators around attention: what a program that serves or trains a model calls, at its sizes.

``listed()`` holds the named cases, ``draw()`` makes further ones over the same ranges.  A case is a dict of plain values;
``prepare()`` builds what a caller holds before the call, ``run()`` is one pass.  ``own`` false: the plain form, elementary
torch operations in 32 bits, rounded once at the end; ``own`` true: the calls of ``lapis_b200.attention``.

Operations (``op``):
  rotate    norms of the queries and keys of each head and their rotation by position, forward or backward
  store     new keys and values written to the pages of a cache (``fused``: normalised and rotated on their way, with the
            queries), then read back as the values that the cache holds
  attend    attention of one new token per request over the pages of the cache
  step      both as a serving step has them: one token per request normalised, rotated, written and attended with
"""
import functools
import math

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
LARGEST = {"i8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # a training step's layer, forward: 8192 tokens, 32 query and 8 key heads that share them
        {"name": "rotate_8k_bf16", "op": "rotate", "backward": False, "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "pairs": "halves", "dtype": "bf16"},
        # its backward pass, over a longer batch
        {"name": "rotate_16k_bf16_bwd", "op": "rotate", "backward": True, "tokens": 16384, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "pairs": "halves", "dtype": "bf16"},
        # backward in full precision, a ragged batch, half of each head rotated, neighbouring pairs
        {"name": "rotate_1021_f32_bwd", "op": "rotate", "backward": True, "tokens": 1021, "q_heads": 12, "kv_heads": 4, "dim": 96,
         "rot": 48, "pairs": "neighbours", "dtype": "f32"},
        # one new token of one request: latency
        {"name": "store_1_bf16", "op": "store", "fused": True, "tokens": 1, "requests": 1, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "pairs": "halves", "page": 16, "dtype": "bf16", "store": "bf16"},
        # prompts of 32,768 tokens in all written to an 8-bit cache
        {"name": "store_32k_i8", "op": "store", "fused": True, "tokens": 32768, "requests": 12, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "pairs": "halves", "page": 64, "dtype": "bf16", "store": "i8"},
        # keys and values as they are, odd numbers of tokens, heads and slots of a page
        {"name": "store_5003_e4m3", "op": "store", "fused": False, "tokens": 5003, "requests": 7, "q_heads": 5, "kv_heads": 5, "dim": 80,
         "rot": 80, "pairs": "halves", "page": 24, "dtype": "f16", "store": "e4m3"},
        # a short chat of one user: latency
        {"name": "attend_1x129_bf16", "op": "attend", "requests": 1, "longest": 129, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "window": 0, "dtype": "bf16", "store": "bf16"},
        # one request with a long document: a single row, work only along the cache
        {"name": "attend_1x131072_bf16", "op": "attend", "requests": 1, "longest": 131072, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "dtype": "bf16", "store": "bf16"},
        # a full server: 128 requests of ragged lengths, 8-bit cache
        {"name": "attend_128x8192_i8", "op": "attend", "requests": 128, "longest": 8192, "q_heads": 64, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "dtype": "bf16", "store": "i8"},
        # a model with narrow heads and a window, odd sizes
        {"name": "attend_23x20011_e4m3", "op": "attend", "requests": 23, "longest": 20011, "q_heads": 48, "kv_heads": 3, "dim": 64,
         "page": 16, "window": 4096, "dtype": "f16", "store": "e4m3"},
        # full precision, a head for each query head, head size 72, pages of 24
        {"name": "attend_16x2047_f32", "op": "attend", "requests": 16, "longest": 2047, "q_heads": 8, "kv_heads": 8, "dim": 72,
         "page": 24, "window": 0, "dtype": "f32", "store": "f32"},
        # a serving step of 48 requests: write the token, attend with it
        {"name": "step_48x4096_bf16", "op": "step", "requests": 48, "longest": 4096, "q_heads": 32, "kv_heads": 4, "dim": 128, "rot": 128,
         "pairs": "halves", "page": 32, "window": 0, "dtype": "bf16", "store": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8, 16])
    return kv * rng.choice([1, 2, 3, 4, 6, 8, 16] if kv <= 4 else [1, 2, 4, 8] if kv <= 8 else [1, 2]), kv


def draw(rng):
    op = rng.choice(["rotate", "store", "attend", "attend", "step"])
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice([32, 64, 72, 80, 96, 112, 128, 128, 192, 256])
    rot = dim if rng.random() < 0.7 else dim // 2
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    # a computed f32 value on the edge between two codes may take either: with f32 what is quantised is the input itself
    store = rng.choice([dtype, "i8", "e4m3"])
    c = {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if op in ("rotate", "store"):
        most = max(2, int(24576 * 48 * 128 / ((q_heads + 2 * kv_heads) * dim)) // (1 if dtype != "f32" else 2))
        c |= {"tokens": _log(rng, 1, min(most, 40000)), "rot": rot, "pairs": rng.choice(["halves", "neighbours"])}
    if op == "rotate":
        return c | {"backward": rng.random() < 0.5}
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    if op == "store":
        fused = dtype != "f32" and rng.random() < 0.6
        return c | {"fused": fused, "requests": min(c["tokens"], _log(rng, 1, 64)), "page": page, "store": store}
    requests = _log(rng, 1, 128)
    most = int(2 ** 30 / (requests * kv_heads * dim * SIZE[store]))
    c |= {"requests": requests, "longest": _log(rng, 1, max(2, min(131072, most))), "page": page,
          "window": rng.choice([0, 0, 0, 128, 1000]), "store": store}
    return c if op == "attend" else c | {"rot": rot, "pairs": rng.choice(["halves", "neighbours"]), "dtype": "bf16" if dtype == "f32" else dtype,
                                         "store": "bf16" if store == "f32" else store}


def _lengths(case):
    """Tokens of each request: the longest first, the others ragged; of eight requests or more one is an empty place in the batch."""
    n, longest = case["requests"], case["longest"]
    r = np.random.RandomState(n * 7919 + longest)
    lens = r.randint(1, longest + 1, n)
    lens[0] = longest
    if n >= 8 and case["op"] == "attend":
        lens[n // 2] = 0
    return lens


def work(case):
    t, hq, hkv, d, s = case.get("tokens"), case["q_heads"], case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    if case["op"] == "rotate":
        tables = t * (case["rot"] * 4 + 4)
        return {"bytes": (3 if case["backward"] else 2) * t * (hq + hkv) * d * s + tables, "flops": t * (hq + hkv) * d * (16 if case["backward"] else 7)}
    held = 2 * hkv * (d * SIZE[case["store"]] + (4 if case["store"] in LARGEST else 0))  # bytes of one token in the cache
    if case["op"] == "store":
        through = t * (2 * hkv * d * s + held) + t * (held + 2 * hkv * d * s)
        if case["fused"]:
            through += 2 * t * hq * d * s + t * case["rot"] * 4
        return {"bytes": through + 8 * t, "flops": t * (hq + 4 * hkv) * d * 7}
    lens = _lengths(case)
    seen = int(np.minimum(lens, case["window"]).sum() if case["window"] else lens.sum())
    n = case["requests"]
    moved = seen * held + 2 * n * hq * d * s + 4 * n * hq
    if case["op"] == "step":
        moved += n * (2 * hkv * d * s + hq * d * s + held)
    return {"bytes": moved, "flops": 4 * seen * hq * d}


# ---- inputs -----------------------------------------------------------------


@functools.lru_cache(maxsize=4)
def _tables(places, rot):
    angle = torch.arange(places, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEV) / (rot // 2))
    return angle.cos().float(), angle.sin().float()


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _quantised(x, store):
    """Codes and scales of the rows of x."""
    most = x.abs().amax(-1, keepdim=True)
    big = torch.full_like(most, LARGEST[store])  # a tensor: torch divides by a number by way of its reciprocal
    code = torch.where(most > 0, x * (big / most), 0.0).clamp(-LARGEST[store], LARGEST[store])
    code = code.round().to(torch.int8) if store == "i8" else code.to(torch.float8_e4m3fn)
    return code, (most / big).squeeze(-1)


def _pages(case, lens, gen):
    """Page lists as CSR rows (pos, crd): the pages of a request lie anywhere in the cache."""
    each = -(-lens // case["page"])
    pos = np.concatenate([[0], np.cumsum(each)])
    total = int(pos[-1])
    crd = torch.randperm(total + 3, generator=gen, device=DEV)[:total].to(torch.int32)
    return torch.from_numpy(pos.astype(np.int32)).to(DEV), crd, total + 3


def _cache(case, pages, gen, filled):
    """k, v [pages, heads, slots of a page, dim] and their scales."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    kind, got = case["store"], []
    for which in range(2):
        if not filled:
            got.append((torch.zeros(shape, device=DEV, dtype=torch.uint8 if kind == "e4m3" else TYPES[kind]),
                        torch.zeros(shape[:3], device=DEV) if kind in LARGEST else None))
            if kind == "e4m3":
                got[-1] = (got[-1][0].view(torch.float8_e4m3fn), got[-1][1])
            continue
        x = _normal(gen, *shape)
        if which == 0:
            x += 0.5 * _normal(gen, 1, case["kv_heads"], 1, case["dim"])  # keys of a head have a direction in common
        else:
            x *= 1 + 4 * (torch.rand(case["dim"], generator=gen, device=DEV) < 0.03)  # values have a few large channels
        got.append(_quantised(x, kind) if kind in LARGEST else (x.to(TYPES[kind]), None))
    (k, ks), (v, vs) = got
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    hq, hkv, d, dt = case["q_heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
    s = {"case": case, "op": case["op"]}
    if case["op"] == "attend":
        lens = _lengths(case)
        s["pos"], s["crd"], pages = _pages(case, lens, gen)
        s |= _cache(case, pages, gen, True)
        s["q"] = (1.5 * _normal(gen, case["requests"], hq, d)).to(dt)
        s["length"] = torch.from_numpy(lens.astype(np.int32)).to(DEV)
    else:
        t = case["requests"] if case["op"] == "step" else case["tokens"]
        # one projection's output holds the queries, keys and values of a token next to one another
        qkv = _normal(gen, t, hq + 2 * hkv, d).to(dt)
        s["q"], s["k_new"], s["v_new"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["q_weight"], s["k_weight"] = (1 + 0.2 * _normal(gen, 2, d)).to(dt)
        if case["op"] == "step":
            lens = _lengths(case)
            row, place = torch.arange(t, device=DEV, dtype=torch.int32), torch.from_numpy((lens - 1).astype(np.int32)).to(DEV)
            s["length"] = torch.from_numpy(lens.astype(np.int32)).to(DEV)
        elif case["op"] == "store":
            n = case["requests"]
            lens = np.full(n, t // n)
            lens[:t % n] += 1
            row = torch.from_numpy(np.repeat(np.arange(n), lens).astype(np.int32)).to(DEV)
            place = torch.from_numpy(np.concatenate([np.arange(x) for x in lens]).astype(np.int32)).to(DEV)
        else:  # packed sequences of up to 4096 tokens
            place = torch.arange(t, device=DEV, dtype=torch.int32) % 4096
            if case["backward"]:
                s["dq"], s["dk"] = _normal(gen, t, hq, d).to(dt), _normal(gen, t, hkv, d).to(dt)
        s["cos"], s["sin"] = _tables(int(place.max()) + 1, case["rot"])
        s["place"] = place
        if case["op"] != "rotate":
            s["row"] = row
            s["pos"], s["crd"], pages = _pages(case, lens, gen)
            s |= _cache(case, pages, gen, case["op"] == "step")
    if own and "k" in s:
        from lapis_b200 import attention
        s["cache"] = attention.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ---- one pass ---------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from lapis_b200 import attention as A
    c, op = s["case"], s["op"]
    near = c.get("pairs") == "neighbours"
    if op == "rotate":
        if not c["backward"]:
            q, k = A.qk_norm_rope(s["q"], s["k_new"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["place"], eps=EPS, interleaved=near)
            return {"q": q, "k": k}
        dq, dk, dqw, dkw = A.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k_new"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                                                   s["place"], eps=EPS, interleaved=near)
        return {"dq": dq, "dk": dk, "dq_weight": dqw, "dk_weight": dkw}
    if op == "attend":
        out, lse = A.paged_attention(s["q"], s["cache"], s["pos"], s["crd"], s["length"], window=c["window"], return_lse=True)
        return {"out": out, "lse": lse}
    got = {}
    if op == "step" or c["fused"]:
        got["q"] = s["cache"].append_norm_rope(s["q"], s["k_new"], s["v_new"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["pos"],
                                               s["crd"], s["row"], s["place"], eps=EPS, interleaved=near)
    else:
        s["cache"].append(s["k_new"], s["v_new"], s["pos"], s["crd"], s["row"], s["place"])
    if op == "store":
        got["k"], got["v"] = s["cache"].read(s["pos"], s["crd"], s["row"], s["place"], dtype=s["k_new"].dtype)
        return got
    out = A.paged_attention(got["q"], s["cache"], s["pos"], s["crd"], s["length"], window=c["window"])
    return {"out": out} | ({"k": s["k"], "v": s["v"]} if c["store"] not in LARGEST else {})


def _rotation(cos, sin, near):
    """Pairs of the rotated dimensions as (first, second) halves of the last axis, and back."""
    if near:
        return lambda x: (x[..., 0::2], x[..., 1::2]), lambda a, b: torch.stack([a, b], -1).flatten(-2)
    return lambda x: (x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]), lambda a, b: torch.cat([a, b], -1)


def _norm_rope(x, weight, s, near):
    x = x.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    cos, sin = (s[w][s["place"].long()][:, None] for w in ("cos", "sin"))
    rot = 2 * cos.shape[-1]
    apart, together = _rotation(cos, sin, near)
    a, b = apart(n[..., :rot])
    return torch.cat([together(a * cos - b * sin, b * cos + a * sin), n[..., rot:]], -1)


def _norm_rope_backward(dy, x, weight, s, near):
    x, dy = x.float(), dy.float()
    cos, sin = (s[w][s["place"].long()][:, None] for w in ("cos", "sin"))
    rot = 2 * cos.shape[-1]
    apart, together = _rotation(cos, sin, near)
    a, b = apart(dy[..., :rot])
    dn = torch.cat([together(a * cos + b * sin, b * cos - a * sin), dy[..., rot:]], -1)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    g = dn * weight.float()
    return r * (g - x * (r * r * (g * x).mean(-1, keepdim=True))), (dn * x * r).sum((0, 1))


def _where(s):
    """Page and slot of the new tokens."""
    page, place = s["case"]["page"], s["place"].long()
    return s["crd"][s["pos"][s["row"].long()].long() + place // page].long(), place % page


def _write(s, which, x):
    page, slot = _where(s)
    kind = s["case"]["store"]
    if kind in LARGEST:
        code, scale = _quantised(x, kind)
        s[which + "_scale"][page, :, slot] = scale
        if kind == "e4m3":
            s[which].view(torch.uint8)[page, :, slot] = code.view(torch.uint8)
        else:
            s[which][page, :, slot] = code
    else:
        s[which][page, :, slot] = x.to(TYPES[kind])


def _held(s, which, page, slot):
    """[..., heads, dim] in 32 bits of the given pages and slots."""
    if s["case"]["store"] == "e4m3":
        x = s[which].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn).float()
    else:
        x = s[which][page, :, slot].float()
    return x * s[which + "_scale"][page, :, slot][..., None] if s["case"]["store"] in LARGEST else x


def _attend(s, q):
    c = s["case"]
    n, hq, hkv, d, page = c["requests"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    length = s["length"].long()
    at = torch.arange(c["longest"], device=DEV)
    seen = at[None] < length[:, None]
    if c["window"]:
        seen &= at[None] >= length[:, None] - c["window"]
    entry = torch.where(seen, s["pos"][:-1].long()[:, None] + at[None] // page, 0)
    pages, slot = s["crd"][entry].long(), (at % page).expand(n, -1)
    k, v = (_held(s, w, pages, slot).permute(0, 2, 1, 3) for w in ("k", "v"))  # [n, hkv, longest, d]
    score = (q.float().view(n, hkv, hq // hkv, d) @ k.transpose(-1, -2)) * d ** -0.5
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(most == -math.inf, 0.0, most))
    total = weight.sum(-1, keepdim=True)
    v = torch.where(seen[:, None, :, None], v, 0.0)
    out = (weight @ v) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, most + torch.log(total), -math.inf)
    return out.reshape(n, hq, d), lse.reshape(n, hq)


def _plain(s):
    c, op = s["case"], s["op"]
    dt, near = TYPES[c["dtype"]], c.get("pairs") == "neighbours"
    if op == "rotate":
        if not c["backward"]:
            return {"q": _norm_rope(s["q"], s["q_weight"], s, near).to(dt), "k": _norm_rope(s["k_new"], s["k_weight"], s, near).to(dt)}
        dq, dqw = _norm_rope_backward(s["dq"], s["q"], s["q_weight"], s, near)
        dk, dkw = _norm_rope_backward(s["dk"], s["k_new"], s["k_weight"], s, near)
        return {"dq": dq.to(dt), "dk": dk.to(dt), "dq_weight": dqw, "dk_weight": dkw}
    if op == "attend":
        out, lse = _attend(s, s["q"])
        return {"out": out.to(dt), "lse": lse}
    got, k = {}, s["k_new"].float()
    if op == "step" or c["fused"]:
        got["q"], k = _norm_rope(s["q"], s["q_weight"], s, near).to(dt), _norm_rope(s["k_new"], s["k_weight"], s, near)
    _write(s, "k", k)
    _write(s, "v", s["v_new"].float())
    if op == "store":
        page, slot = _where(s)
        got["k"], got["v"] = (_held(s, w, page, slot).to(dt) for w in ("k", "v"))
        return got
    out = _attend(s, got["q"])[0].to(dt)
    return {"out": out} | ({"k": s["k"], "v": s["v"]} if c["store"] not in LARGEST else {})


# ---- the same from the definitions, in 64 bits --------------------------------


def _exact_rotated(x, weight, s, backward_of=None):
    """Rotation as a product with complex numbers of modulus one; its gradient is the product with the conjugates."""
    c = s["case"]
    x, w, half = x.double(), weight.double(), c["rot"] // 2
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["place"].long()].unsqueeze(1)
    first = torch.arange(half, device=DEV) * (2 if c["pairs"] == "neighbours" else 1)
    second = first + (1 if c["pairs"] == "neighbours" else half)

    def turned(y, by):
        z, y = torch.complex(y[..., first], y[..., second]) * by, y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    norm = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    if backward_of is None:
        return turned(x / norm * w, turn)
    dn = turned(backward_of.double(), turn.conj())
    unit = x / norm
    inner = (dn * w * unit).sum(-1, keepdim=True) / x.shape[-1]
    return (dn * w - unit * inner) / norm, torch.einsum("thd,thd->d", dn, unit)


def _exact_held(x, kind):
    if kind not in LARGEST:
        return x
    big = LARGEST[kind]
    most = x.abs().max(-1, keepdim=True).values
    code = x * big / torch.where(most == 0, 1.0, most)
    return (code.round() if kind == "i8" else code.float().to(torch.float8_e4m3fn).double()) * (most / big).float().double()


def exact(case, seed):
    s = prepare(case, seed)
    op, page, lens = case["op"], case["page"] if "page" in case else 1, s["length"].tolist() if "length" in s else []
    if op == "rotate":
        if not case["backward"]:
            return {"q": _exact_rotated(s["q"], s["q_weight"], s), "k": _exact_rotated(s["k_new"], s["k_weight"], s)}
        dq, dqw = _exact_rotated(s["q"], s["q_weight"], s, s["dq"])
        dk, dkw = _exact_rotated(s["k_new"], s["k_weight"], s, s["dk"])
        return {"dq": dq, "dk": dk, "dq_weight": dqw, "dk_weight": dkw}
    got = {}
    if op != "attend":
        fused = op == "step" or case["fused"]
        q = _exact_rotated(s["q"], s["q_weight"], s) if fused else None
        k = _exact_held(_exact_rotated(s["k_new"], s["k_weight"], s) if fused else s["k_new"].double(), case["store"])
        v = _exact_held(s["v_new"].double(), case["store"])
        if op == "store":
            return ({"q": q} if fused else {}) | {"k": k, "v": v}
    else:
        q = s["q"].double()
    group, outs, lses = case["q_heads"] // case["kv_heads"], [], []
    pos = s["pos"].tolist()
    for b, n in enumerate(lens):
        lo = max(0, n - case["window"]) if case["window"] else 0
        mine = s["crd"][pos[b]:pos[b + 1]].long()
        kv = []
        for w in ("k", "v"):
            x = s[w].view(torch.uint8)[mine].view(TYPES["e4m3"]) if case["store"] == "e4m3" else s[w][mine]
            x = x.double()
            if case["store"] in LARGEST:
                x = x * s[w + "_scale"][mine].double().unsqueeze(-1)
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, lo:n])  # [heads, tokens, dim]
        kb, vb = kv
        if op == "step":  # the token that this step writes
            kb[:, -1], vb[:, -1] = k[b], v[b]
        score = torch.einsum("hgd,hnd->hgn", q[b].view(-1, group, case["dim"]), kb) / math.sqrt(case["dim"])
        lse = torch.logsumexp(score, -1)
        outs.append(torch.einsum("hgn,hnd->hgd", torch.exp(score - lse.unsqueeze(-1)), vb).flatten(0, 1) if n else torch.zeros_like(q[b]))
        lses.append(lse.flatten() if n else torch.full((case["q_heads"],), -math.inf, device=DEV, dtype=torch.float64))
    got["out"] = torch.stack(outs)
    if op == "attend":
        got["lse"] = torch.stack(lses)
    elif case["store"] not in LARGEST:
        got |= {"k": None, "v": None}  # the cache: all but one token of a request is as it was
    return got
