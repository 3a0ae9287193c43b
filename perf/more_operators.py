"""The attention half of a decoder layer over 4-bit weights and a 4-bit cache, as cases to measure.

Three operators, next to the products and experts of ``operators.py``:

* ``append``: keys and values of new tokens, rotated by their positions, are brought to 4 bits and
  put into a paged cache (``kv4_append``); queries are rotated on the way. The pass ends with
  ``kv4_read``, so its outputs are what the cache now holds of them.
* ``attend``: attention of new tokens' queries over the cache (``kv4_attention``): one token, a few
  drafted ones or whole prompts a sequence; causal, optionally within a window and first tokens.
* ``linear``: ``q4_linear``, the product with 4-bit weights with bias, activation and residual.

``run`` computes them in plain torch operations, or (``own``) through the library's binding.

A page of the cache holds, for each key-value head, blocks of 16 tokens: the keys' codes, their
scales and middles, then the values'. ``_key_bytes``, ``_value_bytes`` and ``_scale_bytes`` say where
each lies.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LINEAR_MOST = 2 * 2048 * 8192 * 8192
ATTEND_MOST = 4 * 128 * 32 * 8192 * 4096  # operations of a prompt of 8192 tokens, 32 heads of 128
CACHE_MOST = 64 * 8192 * 8 * 128          # tokens x heads x channels of a cache


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # an attention output's way back into the stream for one token: where latency counts
        {"name": "linear 1x4096x4096 residual", "op": "linear", "m": 1, "n": 4096, "k": 4096, "group": 128,
         "type": "bf16", "out": "bf16", "zeros": False, "bias": False, "act": "none", "residual": True},
        # a small batch's hidden layer, ragged in every direction
        {"name": "linear 27x4001x1192 ragged", "op": "linear", "m": 27, "n": 4001, "k": 1192, "group": 32,
         "type": "f16", "out": "f32", "zeros": True, "bias": True, "act": "gelu", "residual": True},
        # a prompt through a wide layer (the benchmark's codec shape)
        {"name": "linear 2048x8192x8192", "op": "linear", "m": 2048, "n": 8192, "k": 8192, "group": 128,
         "type": "bf16", "out": "bf16", "zeros": False, "bias": True, "act": "silu", "residual": True},
        # one token of one sequence: a decoding step
        {"name": "append 1 token", "op": "append", "seqs": 1, "new": 1, "context": 4096, "ragged": False, "pad": 0,
         "heads": 8, "share": 4, "dim": 128, "group": 32, "page": 16, "type": "bf16", "rotated": 128,
         "interleaved": False},
        # 13 sequences' prompt chunks of odd lengths, behind them rows of a padded batch; half of a
        # head's channels rotated, pairs side by side
        {"name": "append 13 ragged chunks", "op": "append", "seqs": 13, "new": 90, "context": 700, "ragged": True,
         "pad": 5, "heads": 3, "share": 2, "dim": 96, "group": 32, "page": 32, "type": "f16", "rotated": 48,
         "interleaved": True},
        # a prompt
        {"name": "append 8192 tokens", "op": "append", "seqs": 1, "new": 8192, "context": 8192, "ragged": False,
         "pad": 0, "heads": 8, "share": 4, "dim": 128, "group": 32, "page": 64, "type": "bf16", "rotated": 128,
         "interleaved": False},
        # one token of one sequence
        {"name": "attend 1 token in 4096", "op": "attend", "seqs": 1, "new": 1, "context": 4096, "ragged": False,
         "pad": 0, "heads": 8, "share": 4, "dim": 128, "group": 32, "page": 16, "type": "bf16", "out": "bf16",
         "window": 0, "sinks": 0},
        # a full batch's decoding step in long contexts
        {"name": "attend 64 tokens in 8192", "op": "attend", "seqs": 64, "new": 1, "context": 8192, "ragged": False,
         "pad": 0, "heads": 8, "share": 8, "dim": 128, "group": 32, "page": 64, "type": "bf16", "out": "bf16",
         "window": 0, "sinks": 0},
        # drafted tokens of sequences of odd lengths, within a window and the first tokens, in a padded batch
        {"name": "attend 29 drafts windowed", "op": "attend", "seqs": 29, "new": 5, "context": 5000, "ragged": True,
         "pad": 3, "heads": 4, "share": 3, "dim": 64, "group": 64, "page": 16, "type": "f16", "out": "f32",
         "window": 1000, "sinks": 4},
        # prompt chunks of several sequences behind what they have cached
        {"name": "attend 6 ragged chunks", "op": "attend", "seqs": 6, "new": 300, "context": 2500, "ragged": True,
         "pad": 0, "heads": 2, "share": 5, "dim": 128, "group": 128, "page": 32, "type": "f16", "out": "f16",
         "window": 0, "sinks": 0},
        # a prompt's second quarter
        {"name": "attend 2048 in 4096", "op": "attend", "seqs": 1, "new": 2048, "context": 4096, "ragged": False,
         "pad": 0, "heads": 8, "share": 4, "dim": 128, "group": 32, "page": 64, "type": "bf16", "out": "bf16",
         "window": 0, "sinks": 0},
        # a whole prompt
        {"name": "attend 8192 in 8192", "op": "attend", "seqs": 1, "new": 8192, "context": 8192, "ragged": False,
         "pad": 0, "heads": 8, "share": 4, "dim": 128, "group": 32, "page": 64, "type": "bf16", "out": "bf16",
         "window": 0, "sinks": 0},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A layer's width: mostly a multiple of 128, 64 or 8, as layers have them; any number at times."""
    by = rng.choice([1, 8, 64, 64, 128, 128])
    return max(low, _log(rng, low, high) // by * by)


def _draw_linear(rng):
    kind = rng.choice(["bf16", "f16"])
    return {"op": "linear", "m": _log(rng, 1, 2048), "n": _width(rng, 64, 8192), "k": _width(rng, 96, 8192),
            "group": rng.choice([32, 64, 128]), "type": kind, "out": rng.choice([kind, "f32"]),
            "zeros": rng.random() < 0.5, "bias": rng.random() < 0.7,
            "act": rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]), "residual": rng.random() < 0.7}


def _draw_cache(rng, op):
    dim = rng.choice([64, 96, 128, 128, 192, 256])
    group = rng.choice([g for g in (32, 64, 128, 256) if dim % g == 0])
    new = rng.choice([1, 1, _log(rng, 2, 8), _log(rng, 8, 2048)])
    return {"op": op, "seqs": _log(rng, 1, 64), "new": new, "context": _log(rng, new, 8192), "ragged": rng.random() < 0.6,
            "pad": rng.choice([0, 0, 3]), "heads": _log(rng, 1, 8), "share": rng.choice([1, 2, 3, 4, 5, 8, 16]), "dim": dim,
            "group": group, "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["bf16", "f16"])}


def draw(rng):
    while True:
        op = rng.choice(["linear", "append", "attend", "attend"])
        if op == "linear":
            c = _draw_linear(rng)
            if work(c)["flops"] <= LINEAR_MOST:
                return c
            continue
        c = _draw_cache(rng, op)
        if op == "append":
            c["rotated"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, 0])
            c["interleaved"] = rng.random() < 0.4
            rows = c["seqs"] * c["new"] * c["heads"] * (c["share"] + 2) * c["dim"]
            if rows <= 8192 * 8 * 6 * 128 and c["seqs"] * c["context"] * c["heads"] * c["dim"] <= CACHE_MOST:
                return c
            continue
        c["out"] = rng.choice([c["type"], "f32"])
        c["window"] = rng.choice([0, 0, _log(rng, 1, 4096)])
        c["sinks"] = rng.choice([0, rng.randint(1, 64)]) if c["window"] else 0
        if work(c)["flops"] <= ATTEND_MOST and c["seqs"] * c["context"] * c["heads"] * c["dim"] <= CACHE_MOST:
            return c


def _lengths(case):
    """Each sequence's (new tokens, tokens in the cache with them): the case's, or spread below them."""
    if not case["ragged"]:
        return [(case["new"], case["context"])] * case["seqs"]
    rng = random.Random(case["seqs"] * 100003 + case["context"])
    found = []
    for _ in range(case["seqs"]):
        length = rng.randint(max(1, case["context"] // 8), case["context"])
        found.append((min(length, rng.randint(1, case["new"])), length))
    return found


# ------------------------------------------------------------------ the cache's layout

def _block_bytes(case):
    return 16 * case["dim"] + 128 * (case["dim"] // case["group"])


def _key_bytes(case, device):
    """(16, dim / 2): where in a block the byte of a token's channels 2 i, 2 i + 1 lies (the lower one
    in the lower nibble). A token's words of 8 channels go by (channel / 8) % 4, then channel / 32."""
    i = torch.arange(case["dim"] // 2, device=device)
    word, byte, groups = i // 4, i % 4, case["dim"] // 32
    at = ((word % 4) * groups + word // 4) * 4 + byte
    return torch.arange(16, device=device)[:, None] * (case["dim"] // 2) + at


def _value_bytes(case, device):
    """The same for values. A word has four channels of two neighbouring tokens, 16 bits each; words go
    by the token's half of the block, (channel / 4) % 8, its pair in the half, then channel / 32."""
    i = torch.arange(case["dim"] // 2, device=device) * 2
    t = torch.arange(16, device=device)[:, None]
    word = ((t // 8 * 8 + i // 4 % 8) * 4 + t // 2 % 4) * (case["dim"] // 32) + i // 32
    base = 8 * case["dim"] + 64 * (case["dim"] // case["group"])
    return base + word * 4 + t % 2 * 2 + i // 2 % 2


def _scale_bytes(case, values, device):
    """(16, groups, 2): where the 16 bits of a token's scale and middle of each group lie."""
    t = torch.arange(16, device=device)[:, None, None]
    g = torch.arange(case["dim"] // case["group"], device=device)[None, :, None]
    which = torch.arange(2, device=device)[None, None, :]
    groups = case["dim"] // case["group"]
    base = 8 * case["dim"] + (8 * case["dim"] + 64 * groups if values else 0)
    return base + (t // 2 * groups + g) * 8 + which * 4 + t % 2 * 2


def _rounded(x, kind):
    return x.to(kind).float()


def _quantised(r, group):
    """Codes, scales and middles of values r (.., dim) of a 16-bit type, in f32 steps."""
    kind = r.dtype
    x = r.float().unflatten(-1, (-1, group))
    high, low = x.amax(-1), x.amin(-1)
    mid = _rounded(high * 0.5 + low * 0.5, kind)
    scale = _rounded((high * 0.5 - low * 0.5) / 7.5, kind)
    code = torch.round((x - mid[..., None]) / scale[..., None] + 7.5).clamp(0, 15)
    code = torch.where(scale[..., None] > 0, code, torch.zeros_like(code))
    return code.flatten(-2).to(torch.uint8), scale.to(kind), mid.to(kind)


def _held(codes, scale, mid, group):
    """f32 values of codes (.., dim)."""
    x = codes.float().unflatten(-1, (-1, group)) - 7.5
    return (x * scale.float()[..., None] + mid.float()[..., None]).flatten(-2)


def _put(case, pool, base, t, codes, scale, mid, values):
    """Codes, scales and middles (rows, heads, ..) into the blocks at byte `base` (rows, heads), as
    their tokens t (rows) of 16."""
    device = pool.device
    where = (_value_bytes if values else _key_bytes)(case, device)[t]
    pool[base[:, :, None] + where[:, None, :]] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    where = _scale_bytes(case, values, device)[t].flatten(1)
    halves = torch.stack((scale, mid), -1).contiguous().view(torch.int16).int().flatten(-2)
    pool[base[:, :, None] + where[:, None, :]] = (halves & 255).to(torch.uint8)
    pool[base[:, :, None] + where[:, None, :] + 1] = (halves >> 8 & 255).to(torch.uint8)


def _take(case, pool, base, t, values):
    """f32 values (rows, heads, dim) of the tokens t (rows) of the blocks at `base` (rows, heads)."""
    device, kind = pool.device, TYPES[case["type"]]
    where = (_value_bytes if values else _key_bytes)(case, device)[t]
    byte = pool[base[:, :, None] + where[:, None, :]]
    codes = torch.stack((byte & 15, byte >> 4), -1).flatten(-2)
    where = _scale_bytes(case, values, device)[t].flatten(1)
    halves = torch.stack((pool[base[:, :, None] + where[:, None, :]], pool[base[:, :, None] + where[:, None, :] + 1]), -1)
    halves = halves.contiguous().view(kind).squeeze(-1).unflatten(-1, (-1, 2))
    return _held(codes, halves[..., 0], halves[..., 1], case["group"])


def _places(case, table, seq, position):
    """Bytes (rows, heads) of the blocks of the tokens at `position` of sequences `seq`, and their
    places in them."""
    page, heads = case["page"], case["heads"]
    blocks = page // 16
    number = table[seq, position // page].long()
    head = torch.arange(heads, device=table.device)
    at = (number[:, None] * heads + head) * blocks + (position % page // 16)[:, None]
    return at * _block_bytes(case), position % 16


# ------------------------------------------------------------------ the inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _quantise_weights(g, rows, cols, group, spread, zeros, scale_type):
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


def _prepare_linear(case, g):
    m, n, k, kind, out = case["m"], case["n"], case["k"], TYPES[case["type"]], TYPES[case["out"]]
    s = {"case": case, "x": _normal(g, m, k).to(kind)}
    s["codes"], s["scales"], s["zeros"] = _quantise_weights(g, n, k, case["group"], k ** -0.5, case["zeros"], kind)
    s["bias"] = (_normal(g, n) * 0.3).to(kind) if case["bias"] else None
    s["residual"] = _normal(g, m, n).to(out) if case["residual"] else None
    s["y"] = torch.empty(m, n, device="cuda", dtype=out)
    return s


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "linear":
        return _prepare_linear(case, g)
    kind = TYPES[case["type"]]
    heads, share, dim, page = case["heads"], case["share"], case["dim"], case["page"]
    lengths = _lengths(case)
    s = {"case": case}
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for new, _ in lengths:
        starts.append(starts[-1] + new)
    s["live"], rows = starts[-1], starts[-1] + case["pad"]
    s["starts"], s["lengths"] = int32(starts), int32([length for _, length in lengths])
    # each sequence's pages lie anywhere in the pool; entries behind its last are not read
    pages = [-(-length // page) for _, length in lengths]
    s["pages"], wide = sum(pages) + 3, max(pages)
    order = torch.randperm(s["pages"], generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.full((len(pages), wide), -1, dtype=torch.int32, device="cuda")
    first = 0
    for i, count in enumerate(pages):
        s["table"][i, :count] = order[first:first + count]
        first += count
    seq = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor([new for new, _ in lengths]))
    position = torch.cat([torch.arange(length - new, length) for new, length in lengths])
    s["seq"], s["position"] = seq.cuda(), position.cuda()
    s["pool"] = torch.zeros(s["pages"] * heads * (page // 16) * _block_bytes(case), dtype=torch.uint8, device="cuda")
    # keys have channels that stand out and lie off zero, as rotated models' do
    shift, size = _normal(g, heads, dim) * 0.5, 1 + 2 * (torch.rand(heads, dim, generator=g, device="cuda") < 0.05)
    if case["op"] == "append":
        wide = heads * (share + 2) * dim  # a projection's rows: queries, keys, values
        x = _normal(g, rows, wide).view(rows, heads * (share + 2), dim)
        keys = x[:, heads * share:heads * (share + 1)]
        keys.mul_(size).add_(shift)
        s["qkv"] = x.view(rows, wide).to(kind)
        at, rotated = wide_positions(case), case["rotated"]
        if rotated:
            angle = torch.arange(at, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
                -torch.arange(0, rotated, 2, device="cuda", dtype=torch.float64) / rotated)
            s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        s["q"] = torch.zeros(rows, heads * share * dim, device="cuda", dtype=kind)
        s["k"], s["v"] = (torch.zeros(rows, heads * dim, device="cuda", dtype=kind) for _ in range(2))
        return s
    # fill the cache, a few thousand tokens at a time
    all_seq = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor([length for _, length in lengths])).cuda()
    all_at = torch.cat([torch.arange(length) for _, length in lengths]).cuda()
    step = max(1, (1 << 25) // (heads * dim))
    for i in range(0, all_at.numel(), step):
        base, t = _places(case, s["table"], all_seq[i:i + step], all_at[i:i + step])
        k = _normal(g, t.numel(), heads, dim) * size + shift
        _put(case, s["pool"], base, t, *_quantised(k.to(kind), case["group"]), False)
        v = _normal(g, t.numel(), heads, dim)
        _put(case, s["pool"], base, t, *_quantised(v.to(kind), case["group"]), True)
    s["q"] = (_normal(g, rows, heads * share * dim) * 1.5).to(kind)
    s["scale"] = dim ** -0.5
    s["y"] = torch.zeros(rows, heads * share * dim, device="cuda", dtype=TYPES[case["out"]])
    s["lse"] = torch.zeros(rows, heads * share, device="cuda", dtype=torch.float32)
    return s


def wide_positions(case):
    """Positions that a rotation's tables have: all of the page table's."""
    return -(-case["context"] // case["page"]) * case["page"]


# ------------------------------------------------------------------ the plain forms

def _activate(x, act):
    if act == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _linear_plain(s):
    c = s["case"]
    code = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).flatten(-2)[..., :c["k"]].float()
    wide = lambda x: x.float().repeat_interleave(c["group"], -1)[..., :c["k"]]  # noqa: E731
    w = (code - (8.0 if s["zeros"] is None else wide(s["zeros"]))) * wide(s["scales"])
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[c["out"]])


def _rotate_plain(s, x):
    """Rows of heads (rows, heads, dim): in 64 bits, where a product of a 16-bit value and an f32 is
    exact, then rounded to f32 and to the type."""
    c = s["case"]
    n = c["rotated"]
    if not n:
        return x
    cos, sin = (s[name].double()[s["position"]][:, None, :] for name in ("cos", "sin"))
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if c["interleaved"] else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a.double(), b.double()
    a, b = (a * cos - b * sin).float().to(x.dtype), (b * cos + a * sin).float().to(x.dtype)
    head = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((head, x[..., n:]), -1)


def _append_plain(s):
    c = s["case"]
    heads, share, dim, live = c["heads"], c["share"], c["dim"], s["live"]
    x = s["qkv"][:live].view(live, -1, dim)
    q, k, v = x[:, :heads * share], x[:, heads * share:heads * (share + 1)], x[:, heads * (share + 1):]
    s["q"][:live] = _rotate_plain(s, q).flatten(1)
    base, t = _places(c, s["table"], s["seq"], s["position"])
    _put(c, s["pool"], base, t, *_quantised(_rotate_plain(s, k), c["group"]), False)
    _put(c, s["pool"], base, t, *_quantised(v, c["group"]), True)
    s["k"][:live] = _take(c, s["pool"], base, t, False).flatten(1).to(s["k"].dtype)
    s["v"][:live] = _take(c, s["pool"], base, t, True).flatten(1).to(s["v"].dtype)
    return s["q"], s["k"], s["v"]


def _attend_plain(s):
    c = s["case"]
    heads, share, dim = c["heads"], c["share"], c["dim"]
    device = s["pool"].device
    start = 0
    for i, (new, length) in enumerate(_lengths(c)):
        at = torch.arange(length, device=device)
        base, t = _places(c, s["table"], torch.full_like(at, i), at)
        k, v = (_take(c, s["pool"], base, t, values).transpose(0, 1) for values in (False, True))  # heads, length, dim
        step = max(1, (1 << 28) // (length * heads * share))
        for first in range(0, new, step):
            count = min(step, new - first)
            rows = slice(start + first, start + first + count)
            q = s["q"][rows].float().view(count, heads, share, dim).permute(1, 0, 2, 3).reshape(heads, count * share, dim)
            score = (q @ k.transpose(1, 2)).view(heads, count, share, length) * s["scale"]
            here = (length - new + first + torch.arange(count, device=device))[:, None]
            seen = at <= here
            if c["window"]:
                seen = seen & ((at > here - c["window"]) | (at < c["sinks"]))
            score = torch.where(seen[None, :, None, :], score, torch.full_like(score, -math.inf))
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - top)
            total = p.sum(-1, keepdim=True)
            y = (p / total).view(heads, count * share, length) @ v
            y = y.view(heads, count, share, dim).permute(1, 0, 2, 3)
            s["y"][rows] = y.reshape(count, -1).to(s["y"].dtype)
            s["lse"][rows] = (top + torch.log(total))[..., 0].permute(1, 0, 2).reshape(count, -1)
        start += new
    return s["y"], s["lse"]


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


def _linear_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    m, n, k = c["m"], c["n"], c["k"]
    if "w" not in s:  # the weights' descriptor, which a program keeps
        s["w"] = U.Q4(s["codes"], s["scales"], tag[c["type"]], n, k, c["group"], zeros=s["zeros"])
    act = {"none": U.IDENTITY, "relu": U.RELU, "gelu": U.GELU, "gelu_tanh": U.GELU_TANH, "silu": U.SILU}[c["act"]]
    U.q4_linear(tag[c["type"]], tag[c["out"]], s["x"], (m, k), s["w"], s["y"], (m, n), bias=s["bias"], activation=act,
                residual=s["residual"], rv=(m, n), ctx=ctx, asynchronous=True)
    return s["y"]


def _cache(s):
    """The cache's and the batch's descriptors, which a program keeps."""
    U, _, tag = _lib()
    c = s["case"]
    if "cache" not in s:
        s["cache"] = U.KV4(s["pool"], s["pages"], c["page"], c["heads"], c["dim"], c["group"], tag[c["type"]])
        s["batch"] = U.Batch(s["starts"], s["lengths"], s["table"], c["seqs"], s["table"].shape[1])
    return s["cache"], s["batch"]


def _append_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    cache, batch = _cache(s)
    heads, share, dim, rows = c["heads"], c["share"], c["dim"], s["qkv"].shape[0]
    wide = heads * (share + 2) * dim
    if "turn" not in s:
        s["turn"] = U.Rotation(s["cos"], s["sin"], wide_positions(c), c["rotated"], c["interleaved"]) if c["rotated"] else None
    q, k, v = s["qkv"], s["qkv"].view(-1)[heads * share * dim:], s["qkv"].view(-1)[heads * (share + 1) * dim:]
    U.kv4_append(tag[c["type"]], cache, batch, k, (rows, heads * dim, wide), v, (rows, heads * dim, wide),
                 q=q, qv=(rows, heads * share * dim, wide), q_out=s["q"], ov=(rows, heads * share * dim),
                 rotation=s["turn"], ctx=ctx, asynchronous=True)
    U.kv4_read(tag[c["type"]], cache, batch, s["k"], (rows, heads * dim), s["v"], (rows, heads * dim), ctx=ctx,
               asynchronous=True)
    return s["q"], s["k"], s["v"]


def _attend_own(s):
    U, ctx, tag = _lib()
    c = s["case"]
    cache, batch = _cache(s)
    rows, wide = s["q"].shape
    U.kv4_attention(tag[c["type"]], tag[c["out"]], cache, batch, s["q"], (rows, wide), s["y"], (rows, wide),
                    scale=s["scale"], window=c["window"], sinks=c["sinks"], lse=s["lse"],
                    lv=(rows, c["heads"] * c["share"]), ctx=ctx, asynchronous=True)
    return s["y"], s["lse"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _linear_own, "append": _append_own, "attend": _attend_own}[op](state)
    return {"linear": _linear_plain, "append": _append_plain, "attend": _attend_plain}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without

def _size(name):
    return 4 if name == "f32" else 2


def _seen(case):
    """(pairs of a new token and a token that it sees, tokens that some new token sees)."""
    pairs = tokens = 0
    w, sinks = case["window"], case["sinks"]
    for new, length in _lengths(case):
        for p in (range(length - new, length) if w else ()):
            low = max(0, p - w + 1)
            pairs += p + 1 - low + min(sinks, low)
        if not w:
            pairs += new * (2 * length - new + 1) // 2
        low = max(0, length - new - w + 1) if w else 0
        tokens += length - low + min(sinks, low)
    return pairs, tokens


def work(case):
    c = case
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        weights = n * ((k + 1) // 2 + -(-k // c["group"]) * (2 + (1 if c["zeros"] else 0)))
        outs = m * n * _size(c["out"]) * (2 if c["residual"] else 1) + (2 * n if c["bias"] else 0)
        return {"bytes": m * k * 2 + weights + outs, "flops": 2 * m * n * k}
    heads, share, dim = c["heads"], c["share"], c["dim"]
    held = dim + 8 * (dim // c["group"])  # bytes of a token's keys and values, per head
    lengths = _lengths(c)
    rows = sum(new for new, _ in lengths)
    if c["op"] == "append":
        turned = 8 * (c["rotated"] // 2) * len({p for new, length in lengths for p in range(length - new, length)})
        through = heads * (share * 2 + 2 + 2) * dim * 2  # queries in and out, keys and values in and out again
        return {"bytes": rows * (through + 2 * heads * held) + turned,
                "flops": rows * heads * (share + 2) * dim * 6}
    pairs, tokens = _seen(c)
    return {"bytes": tokens * heads * held + rows * heads * share * (dim * (2 + _size(c["out"])) + 4),
            "flops": 4 * pairs * heads * share * dim}


# ------------------------------------------------------------------ the definitions, in 64 bits

def _exact_linear(case, s):
    k = torch.arange(case["k"], device="cuda")
    rows = []
    for j in range(0, case["n"], 1024):
        byte = s["codes"][j:j + 1024].long().index_select(1, k // 2)
        zero = 8 if s["zeros"] is None else s["zeros"][j:j + 1024].long().index_select(1, k // case["group"])
        w = (((byte >> ((k % 2) * 4)) & 15) - zero).double() * s["scales"][j:j + 1024].double().index_select(1, k // case["group"])
        rows.append(torch.einsum("mk,nk->mn", s["x"].double(), w))
    y = torch.cat(rows, 1)
    if s["bias"] is not None:
        y += s["bias"].double()
    f = torch.nn.functional
    y = {"none": lambda v: v, "relu": f.relu, "silu": f.silu, "gelu": f.gelu,
         "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[case["act"]](y)
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_held(r, group):
    """What the cache holds of r (.., dim): the steps that the definition rounds to f32 and to the type
    are rounded here too, all else is in 64 bits."""
    kind = r.dtype
    step = lambda v: v.float().double()  # noqa: E731
    out = []
    for part in r.double().split(group, -1):
        high, low = part.max(-1, keepdim=True).values, part.min(-1, keepdim=True).values
        mid = step((high + low) / 2).to(torch.float32).to(kind).double()
        scale = step((high / 2 - low / 2) / 7.5).to(torch.float32).to(kind).double()
        code = step(step(step(part - mid) / scale) + 7.5)
        code = torch.where(scale > 0, code.round().clamp(0, 15), torch.zeros_like(code))
        out.append(mid + scale * (code - 7.5))
    return torch.cat(out, -1)


def _exact_append(case, s):
    rows, live = s["qkv"].shape[0], s["live"]
    heads, share, dim, n = case["heads"], case["share"], case["dim"], case["rotated"]
    x = s["qkv"][:live].double().view(live, -1, dim)
    first = torch.arange(0, n, 2, device="cuda") if case["interleaved"] else torch.arange(n // 2, device="cuda")
    second = first + (1 if case["interleaved"] else n // 2)
    turned = x.clone()
    if n:
        cos, sin = s["cos"][s["position"]].double()[:, None], s["sin"][s["position"]].double()[:, None]
        turned[..., first] = x[..., first] * cos - x[..., second] * sin
        turned[..., second] = x[..., second] * cos + x[..., first] * sin
    cut = heads * share
    found = [turned[:, :cut]]
    kind = TYPES[case["type"]]
    for part in (turned[:, cut:cut + heads], x[:, cut + heads:]):
        found.append(_exact_held(part.float().to(kind), case["group"]))
    whole = []
    for part in found:
        full = torch.zeros(rows, part.shape[1] * dim, dtype=torch.float64, device="cuda")
        full[:live] = part.reshape(live, -1)
        whole.append(full)
    return tuple(whole)


def _exact_attend(case, s):
    heads, share, dim, group, page = case["heads"], case["share"], case["dim"], case["group"], case["page"]
    y, lse = s["y"].double(), s["lse"].double()
    kind, blocks = TYPES[case["type"]], page // 16
    groups = dim // group
    pool = s["pool"].view(s["pages"], heads, blocks, -1)
    cut = [8 * dim, 64 * groups, 8 * dim, 64 * groups]
    start = 0
    for i, (new, length) in enumerate(_lengths(case)):
        count = -(-length // page)
        mine = pool[s["table"][i, :count].long()].transpose(0, 1).reshape(heads, count * blocks, -1)
        kc, kp, vc, vp = mine.split(cut, -1)
        n = count * blocks
        nibbles = lambda b: torch.stack((b & 15, b >> 4), -1).flatten(-2)  # noqa: E731
        # keys: token, word of the quarter, 32 channels; values: half, four channels, pair, 32 channels, token
        kc = nibbles(kc).view(heads, n, 16, 4, dim // 32, 8).permute(0, 1, 2, 4, 3, 5).reshape(heads, n * 16, dim)
        vc = nibbles(vc).view(heads, n, 2, 8, 4, dim // 32, 2, 4).permute(0, 1, 2, 4, 6, 5, 3, 7).reshape(heads, n * 16, dim)

        def value(codes, params):
            p = params.contiguous().view(kind).view(heads, n, 8, groups, 2, 2).permute(0, 1, 2, 5, 3, 4)
            p = p.reshape(heads, n * 16, groups, 2).double()
            wide = p.repeat_interleave(group, 2)
            return ((codes.double() - 7.5) * wide[..., 0] + wide[..., 1])[:, :length]

        k, v = value(kc, kp), value(vc, vp)
        here = torch.arange(length - new, length, device="cuda")[:, None]
        at = torch.arange(length, device="cuda")[None, :]
        hidden = at > here
        if case["window"]:
            hidden = hidden | ((at <= here - case["window"]) & (at >= case["sinks"]))
        for h in range(heads * share):
            q = s["q"][start:start + new, h * dim:(h + 1) * dim].double()
            for a in range(0, new, 2048):
                score = (q[a:a + 2048] @ k[h // share].T * s["scale"]).masked_fill(hidden[a:a + 2048], -math.inf)
                lse[start + a:start + min(new, a + 2048), h] = torch.logsumexp(score, 1)
                y[start + a:start + min(new, a + 2048), h * dim:(h + 1) * dim] = torch.softmax(score, 1) @ v[h // share]
        start += new
    return y, lse


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)
