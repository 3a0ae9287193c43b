"""The mixture-of-experts operators over 4-bit weights, as cases to measure.

Four operators that a quantised mixture-of-experts layer is made of:

* ``q4_gemm``: C = A dequant(W)^T with 4-bit codes and one scale (and, where given, one zero
  point) per row and group of the reduction; one activation row (a matrix-vector product) up to
  prompt-sized blocks.
* ``expert_route``: the router: softmax or sigmoid scores, a bias that only steers the choice,
  groups of experts, top-k, renormalised weights.
* ``expert_route_backward``: the gradient of the router's logits from its weights' gradient.
* ``expert_q4_ffn``: the chosen experts' gated feed-forward products over 4-bit weights, summed
  with the router's weights.

``run`` computes them in plain torch operations, or (``own``) through the library's binding.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FFN_MOST = 2 * 8192 * 3 * 2048 * 1024  # operations of the largest listed feed-forward case
Q4_MOST = 2 * 2048 * 8192 * 8192


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one token through a square projection: the smallest serving call, where latency counts
        {"name": "q4 1x4096x4096", "op": "q4", "m": 1, "n": 4096, "k": 4096, "group": 128,
         "type": "bf16", "out": "bf16", "scales": "bf16", "zeros": False},
        # one token through a wide layer (the benchmark's narrow shape), asymmetric codes
        {"name": "q4 1x8192x8192 zeros", "op": "q4", "m": 1, "n": 8192, "k": 8192, "group": 64,
         "type": "f16", "out": "f16", "scales": "f16", "zeros": True},
        # a small batch with ragged sizes: tiles, groups and vectors all end inside
        {"name": "q4 13x5003x4008 ragged", "op": "q4", "m": 13, "n": 5003, "k": 4008, "group": 32,
         "type": "bf16", "out": "f32", "scales": "f32", "zeros": True},
        # a prompt through a wide layer (the benchmark's codec shape)
        {"name": "q4 2048x8192x8192", "op": "q4", "m": 2048, "n": 8192, "k": 8192, "group": 128,
         "type": "bf16", "out": "bf16", "scales": "bf16", "zeros": False},
        # one token's choice among 64 experts: a decoding step
        {"name": "route 1x64", "op": "route", "t": 1, "experts": 64, "top_k": 6, "score": "softmax",
         "groups": 1, "top_groups": 1, "bias": False, "renormalize": True, "scale": 1.0,
         "type": "f32", "masked": 0.0},
        # a prompt's tokens, softmax without renormalisation, an odd number of experts, some masked
        {"name": "route 4099x60", "op": "route", "t": 4099, "experts": 60, "top_k": 4,
         "score": "softmax", "groups": 1, "top_groups": 1, "bias": False, "renormalize": False,
         "scale": 1.0, "type": "bf16", "masked": 0.1},
        # a training batch: sigmoid scores, balance bias, 4 of 8 groups of 32 experts
        {"name": "route 16384x256 groups", "op": "route", "t": 16384, "experts": 256, "top_k": 8,
         "score": "sigmoid", "groups": 8, "top_groups": 4, "bias": True, "renormalize": True,
         "scale": 2.5, "type": "f32", "masked": 0.0},
        # the same batch's gradient
        {"name": "route back 16384x256", "op": "back", "t": 16384, "experts": 256, "top_k": 8,
         "score": "sigmoid", "groups": 8, "top_groups": 4, "bias": True, "renormalize": True,
         "scale": 2.5, "type": "f32", "masked": 0.0},
        # a ragged batch's gradient through the whole softmax
        {"name": "route back 4099x60", "op": "back", "t": 4099, "experts": 60, "top_k": 4,
         "score": "softmax", "groups": 1, "top_groups": 1, "bias": False, "renormalize": False,
         "scale": 1.0, "type": "bf16", "masked": 0.1},
        # one token through 8 of 64 experts: a decoding step
        {"name": "ffn 1 token 8/64", "op": "ffn", "t": 1, "experts": 64, "top_k": 8, "d": 2048,
         "f": 1024, "group": 128, "type": "bf16", "scales": "bf16", "zeros": False, "dropped": 0.0},
        # a small batch, odd sizes, zero points, choices that were dropped
        {"name": "ffn 37 tokens ragged", "op": "ffn", "t": 37, "experts": 12, "top_k": 3, "d": 1000,
         "f": 344, "group": 32, "type": "f16", "scales": "f16", "zeros": True, "dropped": 0.2},
        # a prompt through 4 of 32 experts
        {"name": "ffn 2048 tokens 4/32", "op": "ffn", "t": 2048, "experts": 32, "top_k": 4, "d": 2048,
         "f": 1024, "group": 128, "type": "bf16", "scales": "bf16", "zeros": False, "dropped": 0.0},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A layer's width: mostly a multiple of 128, 64 or 8, as layers have them; any number at times."""
    by = rng.choice([1, 8, 64, 64, 128, 128])
    return max(low, _log(rng, low, high) // by * by)


def _draw_q4(rng):
    kind = rng.choice(["bf16", "f16"])
    return {"op": "q4", "m": _log(rng, 1, 2048), "n": _width(rng, 64, 8192), "k": _width(rng, 96, 8192),
            "group": rng.choice([32, 64, 128, 256]), "type": kind, "out": rng.choice([kind, "f32"]),
            "scales": rng.choice([kind, "f32"]), "zeros": rng.random() < 0.5}


def _draw_router(rng, op):
    groups = rng.choice([1, 1, 2, 4, 8])
    experts = groups * _log(rng, max(2, 8 // groups), 256 // groups)
    top_groups = rng.randint(1, groups)
    top_k = rng.randint(1, min(8, experts // groups * top_groups))
    return {"op": op, "t": _log(rng, 1, 16384), "experts": experts,
            "top_k": top_k, "score": rng.choice(["softmax", "sigmoid"]), "groups": groups,
            "top_groups": top_groups, "bias": rng.random() < 0.5, "renormalize": rng.random() < 0.7,
            "scale": rng.choice([1.0, 2.5]), "type": rng.choice(["f32", "bf16", "f16"]),
            "masked": rng.choice([0.0, 0.1]) if groups == 1 else 0.0}


def _draw_ffn(rng):
    experts = _log(rng, 4, 64)
    kind = rng.choice(["bf16", "f16"])
    return {"op": "ffn", "t": _log(rng, 1, 2048), "experts": experts,
            "top_k": rng.randint(1, min(8, experts)), "d": _width(rng, 256, 2048),
            "f": _width(rng, 96, 1024), "group": rng.choice([32, 64, 128]), "type": kind,
            "scales": rng.choice([kind, "f32"]), "zeros": rng.random() < 0.5,
            "dropped": rng.choice([0.0, 0.2])}


def draw(rng):
    while True:
        op = rng.choice(["q4", "q4", "route", "back", "ffn", "ffn"])
        if op == "q4":
            c = _draw_q4(rng)
            if 2 * c["m"] * c["n"] * c["k"] <= Q4_MOST // 2:
                return c
        elif op == "ffn":
            c = _draw_ffn(rng)
            # the plain form lays out every expert's weights: as many as the largest listed case
            if (2 * c["t"] * c["top_k"] * 3 * c["d"] * c["f"] <= FFN_MOST
                    and c["experts"] * c["d"] * c["f"] <= 32 * 2048 * 1024):
                return c
        else:
            return _draw_router(rng, op)


# ------------------------------------------------------------------ the inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _quantise(g, rows, cols, group, spread, zeros, scale_type):
    """Gaussian weights brought to 4 bits group by group: packed codes (low nibble first), scales
    and, for asymmetric codes, zero points; the last group of a row may be short."""
    groups = -(-cols // group)
    w = _normal(g, rows, groups * group) * spread
    w[:, cols:] = 0
    w = w.view(rows, groups, group)
    if zeros:
        low, high = w.amin(2).clamp_(max=0), w.amax(2).clamp_(min=0)
        scale = ((high - low) / 15).clamp_(min=1e-6).to(scale_type)
        point = torch.round(-low / scale.float()).clamp_(0, 15)
    else:
        scale = (w.abs().amax(2) / 7).clamp_(min=1e-6).to(scale_type)
        point = torch.full_like(scale, 8, dtype=torch.float32)
    w.div_(scale.float()[:, :, None]).round_().add_(point[:, :, None]).clamp_(0, 15)
    code = w.view(rows, groups * group)[:, : cols + cols % 2].to(torch.uint8)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    return packed.contiguous(), scale.contiguous(), point.to(torch.uint8) if zeros else None


def _undecided(case, logits, bias):
    """Rows in which two scores that decide the choice are so near that 32 bits cannot order them
    (equal ones can be: the lowest index comes first)."""
    t, k = logits.shape[0], case["top_k"]
    score = logits.double()
    score = torch.softmax(score, 1).nan_to_num(0.0) if case["score"] == "softmax" else torch.sigmoid(score)
    key = score if bias is None else score + bias.double()
    key = torch.where(torch.isinf(logits), torch.full_like(key, -math.inf), key)
    near = torch.zeros(t, dtype=torch.bool, device=logits.device)
    if case["top_groups"] < case["groups"]:
        by = key.view(t, case["groups"], -1)
        total, at = by.topk(min(2, by.shape[2]), 2).values.sum(2).sort(dim=1, descending=True, stable=True)
        kept = case["top_groups"]
        gap = total[:, kept - 1] - total[:, kept]
        near = (gap > 0) & (gap < 4e-6 * (total[:, kept - 1].abs() + 2 * score.amax(1)))
        chosen = torch.zeros_like(total, dtype=torch.bool).scatter_(1, at[:, :kept], True)
        key = torch.where(chosen[:, :, None], by, torch.full_like(by, -math.inf)).flatten(1)
    top, at = key.sort(dim=1, descending=True, stable=True)
    gap = (top[:, :-1] - top[:, 1:])[:, :k]
    least = 4e-6 * (top.abs() + score.gather(1, at))[:, : gap.shape[1]]
    return near | ((gap > 0) & (gap < least)).any(1)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["op"] == "q4":
        kind = TYPES[case["type"]]
        s["x"] = _normal(g, case["m"], case["k"]).to(kind)
        s["codes"], s["scales"], s["zeros"] = _quantise(
            g, case["n"], case["k"], case["group"], case["k"] ** -0.5, case["zeros"], TYPES[case["scales"]])
        s["y"] = torch.empty(case["m"], case["n"], device="cuda", dtype=TYPES[case["out"]])
        return s
    if case["op"] in ("route", "back"):
        t, e, k, kind = case["t"], case["experts"], case["top_k"], TYPES[case["type"]]
        spread = 0.05 if case["score"] == "sigmoid" else 0.2 / e
        s["bias"] = _normal(g, e) * spread if case["bias"] else None
        keep = torch.rand(t, e, generator=g, device="cuda") >= case["masked"]
        if case["masked"]:
            keep[::97] = False  # and rows whose mask leaves nothing
        shut = torch.full((t, e), -math.inf, device="cuda", dtype=kind)
        s["logits"] = torch.where(keep, (_normal(g, t, e) * 1.5).to(kind), shut)
        for _ in range(4):  # the rows that 32 bits cannot order are drawn again: their choice is anybody's
            fresh = torch.where(keep, (_normal(g, t, e) * 1.5).to(kind), shut)
            s["logits"] = torch.where(_undecided(case, s["logits"], s["bias"])[:, None], fresh, s["logits"])
        s["ids"] = torch.empty(t, k, device="cuda", dtype=torch.int32)
        s["weights"] = torch.empty(t, k, device="cuda", dtype=torch.float32)
        if case["op"] == "back":
            s["ids"] = _route_plain(case, s["logits"], s["bias"])[0]
            s["dweights"] = _normal(g, t, k)
            s["dlogits"] = torch.empty_like(s["logits"])
        return s
    t, e, k, d, f = (case[n] for n in ("t", "experts", "top_k", "d", "f"))
    kind, kept = TYPES[case["type"]], TYPES[case["scales"]]
    s["x"] = _normal(g, t, d).to(kind)
    # popular and unpopular experts, as a trained router has them
    score = _normal(g, t, e) + 0.5 * _normal(g, 1, e)
    s["ids"] = score.topk(k, 1).indices.to(torch.int32).contiguous()
    s["weights"] = torch.softmax(_normal(g, t, k), 1)
    if case["dropped"]:  # choices beyond an expert's capacity, or of experts that live elsewhere
        lost = torch.rand(t, k, generator=g, device="cuda") < case["dropped"]
        s["ids"] = torch.where(lost, torch.full_like(s["ids"], -1), s["ids"])
    s["up"] = _quantise(g, e * 2 * f, d, case["group"], d ** -0.5, case["zeros"], kept)
    s["down"] = _quantise(g, e * d, f, case["group"], f ** -0.5, case["zeros"], kept)
    s["y"] = torch.empty(t, d, device="cuda", dtype=kind)
    return s


# ------------------------------------------------------------------ the plain forms

def _dequantise(codes, scales, zeros, group, cols):
    """float32 weights (..., cols) of packed codes (..., ceil(cols / 2))."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :cols].float()
    wide = lambda x: x.float().repeat_interleave(group, -1)[..., :cols]  # noqa: E731
    return (code - (8.0 if zeros is None else wide(zeros))) * wide(scales)


def _q4_plain(s):
    c = s["case"]
    w = _dequantise(s["codes"], s["scales"], s["zeros"], c["group"], c["k"])
    return (s["x"].float() @ w.t()).to(TYPES[c["out"]])


def _scores(case, logits):
    """float32 scores; an expert of logit -inf has score 0 and cannot be chosen."""
    x = logits.float()
    if case["score"] == "sigmoid":
        return torch.reciprocal(1 + torch.exp(-x))
    top = x.amax(1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return p / p.sum(1, keepdim=True).clamp(min=1e-38)


def _route_plain(case, logits, bias):
    score = _scores(case, logits)
    open_ = torch.isfinite(logits)
    shut = torch.full_like(score, -math.inf)
    key = torch.where(open_, score if bias is None else score + bias, shut)
    if case["top_groups"] < case["groups"]:
        by = key.view(key.shape[0], case["groups"], -1)
        two = by.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        kept = two.sort(dim=1, descending=True, stable=True).indices[:, : case["top_groups"]]
        chosen = torch.zeros_like(two, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(chosen[:, :, None], by, shut.view_as(by)).flatten(1)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, : case["top_k"]]
    held = torch.isfinite(key.gather(1, ids))
    w = torch.where(held, score.gather(1, ids), torch.zeros_like(score[:, :1]))
    if case["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return torch.where(held, ids, torch.full_like(ids, -1)).to(torch.int32), w * case["scale"]


def _back_plain(s):
    c, ids = s["case"], s["ids"].long()
    held, at = ids >= 0, ids.clamp(min=0)
    score = _scores(c, s["logits"])
    mine = torch.where(held, score.gather(1, at), torch.zeros_like(score[:, :1]))
    g = torch.where(held, s["dweights"], torch.zeros_like(s["dweights"])) * c["scale"]
    if c["renormalize"]:
        total = mine.sum(1, keepdim=True)
        w = torch.where(total > 0, mine / total, torch.zeros_like(mine))
        g = torch.where(total > 0, (g - (g * w).sum(1, keepdim=True)) / total, torch.zeros_like(g))
    d = torch.zeros_like(score).scatter_add_(1, at, torch.where(held, g, torch.zeros_like(g)))
    if c["score"] == "sigmoid":
        d = d * score * (1 - score)
    else:
        d = score * (d - (d * score).sum(1, keepdim=True))
    return d.to(s["logits"].dtype)


def _ffn_plain(s):
    """Pairs of a token and an expert sorted by expert into blocks of one expert each, so that
    both products are batched ones; a block is about an expert's usual share."""
    c = s["case"]
    t, e, k, d, f = (c[n] for n in ("t", "experts", "top_k", "d", "f"))
    pairs = t * k
    block = 1 << max(0, (pairs // e).bit_length() - 1)
    blocks = pairs if block == 1 else pairs // block + e
    ids = s["ids"].reshape(-1).long()
    held = (ids >= 0) & (ids < e)
    ids = torch.where(held, ids, torch.full_like(ids, e))
    order = ids.sort(stable=True).indices
    sorted_ids = ids[order]
    place = torch.arange(pairs, device=ids.device)
    if block > 1:  # each expert's pairs begin at a block of their own
        count = torch.zeros(e + 1, dtype=torch.long, device=ids.device).scatter_add_(0, ids, torch.ones_like(ids))
        padded = (count[:e] + block - 1) // block * block
        begin = torch.cumsum(padded, 0) - padded
        first = torch.cumsum(count, 0) - count
        inside = sorted_ids < e
        place = torch.where(inside, begin[sorted_ids.clamp(max=e - 1)] + place - first[sorted_ids],
                            torch.full_like(place, blocks * block))
        of = torch.full((blocks * block + 1,), 0, dtype=torch.long, device=ids.device)
        of[place] = sorted_ids.clamp(max=e - 1)
        of = of[:-1].view(blocks, block).amax(1)
    else:
        of = sorted_ids.clamp(max=e - 1)
    x = torch.zeros(blocks * block + 1, d, device=ids.device)
    x[place] = s["x"].float()[order // k]
    x = x[:-1].view(blocks, block, d)
    zero = lambda z, rows: None if z is None else z.view(e, rows, -1)  # noqa: E731

    def weights(q, rows, cols):
        codes, scales, zeros = q[0].view(e, rows, -1), q[1].view(e, rows, -1), zero(q[2], rows)
        if pairs <= e:  # few pairs: only the chosen experts' weights are laid out
            return _dequantise(codes[of], scales[of], None if zeros is None else zeros[of], c["group"], cols)
        return _dequantise(codes, scales, zeros, c["group"], cols)[of]

    h = torch.bmm(x, weights(s["up"], 2 * f, d).transpose(1, 2))
    gate, up = h[..., :f], h[..., f:]
    h = gate / (1 + torch.exp(-gate)) * up
    out = torch.bmm(h, weights(s["down"], d, f).transpose(1, 2)).view(blocks * block, d)
    out = torch.cat((out, torch.zeros_like(out[:1])))
    y = torch.zeros(pairs, d, device=ids.device)
    y[order] = out[place]
    w = torch.where(held, s["weights"].reshape(-1), torch.zeros_like(s["weights"].reshape(-1)))
    return (y * w[:, None]).view(t, k, d).sum(1).to(s["x"].dtype)


# ------------------------------------------------------------------ the library's calls

_library = None


def _lib():
    """The binding and a context on torch's current stream, as a program makes them once."""
    global _library
    if _library is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "uor-matmul_b200"))
        import uor_b200 as U
        ctx = U.Context(torch.cuda.current_device())
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        _library = U, ctx, {"bf16": U.BF16, "f16": U.F16, "f32": U.F32}
    return _library


def _q4_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    if "w" not in s:  # the weights' descriptor, which a program keeps
        s["w"] = U.Q4(s["codes"], s["scales"], tag[c["scales"]], c["n"], c["k"], c["group"], zeros=s["zeros"])
    U.q4_gemm(tag[c["type"]], tag[c["out"]], s["x"], (c["m"], c["k"]), s["w"], s["y"], (c["m"], c["n"]),
              ctx=ctx, asynchronous=True)
    return s["y"]


def _router(U, c):
    return U.Router(c["experts"], c["top_k"], U.SOFTMAX if c["score"] == "softmax" else U.SIGMOID,
                    groups=c["groups"], top_groups=c["top_groups"], renormalize=c["renormalize"],
                    scale=c["scale"])


def _route_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    if "router" not in s:
        s["router"] = _router(U, c)
    t, e, k = c["t"], c["experts"], c["top_k"]
    U.expert_route(tag[c["type"]], s["router"], s["logits"], (t, e), s["bias"], s["ids"], (t, k),
                   s["weights"], (t, k), ctx=ctx, asynchronous=True)
    return s["ids"], s["weights"]


def _back_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    if "router" not in s:
        s["router"] = _router(U, c)
    t, e, k = c["t"], c["experts"], c["top_k"]
    U.expert_route_backward(tag[c["type"]], s["router"], s["logits"], (t, e), s["ids"], (t, k),
                            s["dweights"], (t, k), s["dlogits"], (t, e), ctx=ctx, asynchronous=True)
    return s["dlogits"]


def _ffn_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    t, e, k, d, f = (c[n] for n in ("t", "experts", "top_k", "d", "f"))
    if "w" not in s:
        s["w"] = (U.Q4(s["up"][0], s["up"][1], tag[c["scales"]], e * 2 * f, d, c["group"], zeros=s["up"][2]),
                  U.Q4(s["down"][0], s["down"][1], tag[c["scales"]], e * d, f, c["group"], zeros=s["down"][2]))
    U.expert_q4_ffn(tag[c["type"]], tag[c["type"]], e, s["x"], (t, d), s["ids"], (t, k), s["weights"], (t, k),
                    s["w"][0], s["w"][1], s["y"], (t, d), ctx=ctx, asynchronous=True)
    return s["y"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"q4": _q4_own, "route": _route_own, "back": _back_own, "ffn": _ffn_own}[op](state)
    if op == "q4":
        return _q4_plain(state)
    if op == "route":
        return _route_plain(state["case"], state["logits"], state["bias"])
    return _back_plain(state) if op == "back" else _ffn_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def _size(name):
    return 4 if name == "f32" else 2


def _q4_bytes(rows, cols, group, scales, zeros):
    return rows * ((cols + 1) // 2 + -(-cols // group) * (_size(scales) + (1 if zeros else 0)))


def work(case):
    c = case
    if c["op"] == "q4":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k * 2 + _q4_bytes(n, k, c["group"], c["scales"], c["zeros"]) + m * n * _size(c["out"]),
                "flops": 2 * m * n * k}
    if c["op"] in ("route", "back"):
        t, e, k = c["t"], c["experts"], c["top_k"]
        if c["op"] == "route":
            return {"bytes": t * e * _size(c["type"]) + (4 * e if c["bias"] else 0) + 8 * t * k, "flops": 4 * t * e}
        return {"bytes": 2 * t * e * _size(c["type"]) + 8 * t * k, "flops": 6 * t * e}
    t, e, k, d, f = (c[n] for n in ("t", "experts", "top_k", "d", "f"))
    live = 1 - c["dropped"]
    used = e * (1 - (1 - live * k / e) ** t)  # experts that some token chose
    bytes_ = (_q4_bytes(2 * f, d, c["group"], c["scales"], c["zeros"]) + _q4_bytes(d, f, c["group"], c["scales"], c["zeros"]))
    return {"bytes": used * bytes_ + 2 * t * d * 2 + 8 * t * k, "flops": 2 * live * t * k * 3 * d * f}


# ------------------------------------------------------------------ the definitions, in 64 bits

def _exact_weights(q, row0, rows, cols, group):
    """float64 weights of rows row0 .. row0 + rows, straight from w = scale * (code - zero)."""
    codes, scales, zeros = q
    at = torch.arange(cols, device=codes.device)
    byte = codes[row0:row0 + rows].long().index_select(1, at // 2)
    code = (byte >> ((at % 2) * 4)) & 15
    zero = 8 if zeros is None else zeros[row0:row0 + rows].long().index_select(1, at // group)
    return (code - zero).double() * scales[row0:row0 + rows].double().index_select(1, at // group)


def _exact_choice(c, x, score, bias):
    """The experts by repeated search for the largest, the lowest index first among equals."""
    t, e = x.shape
    key = score + (0.0 if bias is None else bias.double())
    key = key.masked_fill(torch.isinf(x), -math.inf)

    def best(v):
        return torch.argmax((v == v.amax(1, keepdim=True)).to(torch.int8) * torch.arange(v.shape[1], 0, -1, device=v.device), 1)

    if c["top_groups"] < c["groups"]:
        size = e // c["groups"]
        sums = torch.stack([key[:, i * size:(i + 1) * size].topk(min(2, size), 1).values.sum(1) for i in range(c["groups"])], 1)
        open_ = torch.zeros(t, e, dtype=torch.bool, device=x.device)
        for _ in range(c["top_groups"]):
            at = best(sums)
            sums.scatter_(1, at[:, None], -math.inf)
            open_ |= (torch.arange(e, device=x.device)[None, :] // size) == at[:, None]
        key = key.masked_fill(~open_, -math.inf)
    ids = []
    for _ in range(c["top_k"]):
        at = best(key)
        there = torch.isfinite(key.gather(1, at[:, None]))[:, 0]
        ids.append(torch.where(there, at, -1))
        key = key.scatter(1, at[:, None], -math.inf)
    return torch.stack(ids, 1)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "q4":
        w = _exact_weights((s["codes"], s["scales"], s["zeros"]), 0, c["n"], c["k"], c["group"])
        return torch.einsum("mk,nk->mn", s["x"].double(), w)
    if c["op"] == "ffn":
        t, e, d, f = c["t"], c["experts"], c["d"], c["f"]
        y = torch.zeros(t, d, dtype=torch.float64, device="cuda")
        for one in range(e):
            token, slot = torch.nonzero(s["ids"] == one, as_tuple=True)
            if not token.numel():
                continue
            x = s["x"][token].double()
            both = x @ _exact_weights(s["up"], one * 2 * f, 2 * f, d, c["group"]).T
            h = torch.nn.functional.silu(both[:, :f]) * both[:, f:]
            out = h @ _exact_weights(s["down"], one * d, d, f, c["group"]).T
            y.index_add_(0, token, out * s["weights"][token, slot].double()[:, None])
        return y
    x = s["logits"].double()
    score = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, 1).nan_to_num(0.0)
    ids = s["ids"] if c["op"] == "back" else _exact_choice(c, x, score, s["bias"])
    picked = torch.zeros_like(score)  # 1 where an expert was chosen
    token, slot = torch.nonzero(ids >= 0, as_tuple=True)
    expert = ids[token, slot].long()
    picked[token, expert] = 1.0
    total = (score * picked).sum(1).clamp(min=1e-300)
    if c["op"] == "route":
        w = torch.zeros(ids.shape, dtype=torch.float64, device="cuda")
        value = score[token, expert] / total[token] if c["renormalize"] else score[token, expert]
        w[token, slot] = value * c["scale"]
        return None, w
    grad = torch.zeros_like(score)  # the weights' gradient, by expert
    grad[token, expert] = s["dweights"][token, slot].double() * c["scale"]
    own_slope = score * (1 - score)
    if c["renormalize"]:
        part = score * picked / total[:, None]
        dscore = picked * (grad - (grad * part).sum(1, keepdim=True)) / total[:, None]
    else:
        dscore = grad
    if c["score"] == "sigmoid":
        return dscore * own_slope
    return score * dscore - score * (score * dscore).sum(1, keepdim=True)
