"""Caches, 64-bit references and error bounds for the tests of the 4-bit keys and values.

The bounds are derived, not fitted. A held value is x = mid + scale (code - 7.5); in a group whose
largest is M in size, |mid| <= M and scale <= 2 M / 14, so every term that the kernels' sums hold of it
(mid, 16 scale u, 23.5 scale with u < 2) is at most 6 M.

Scores: sums of dim products in f32, none chained more than dim / 8 + 16 times: off by at most
(dim / 8 + 16) 2^-23 scale sum |q| 6 M. Weights carry that and 2^-20 for the exponential, twice (their
sum divides them). Values: weights times scales travel as two bfloat16, 2^-17 together, and f32 sums
chain at most a block of 16 tokens at a time: (n / 16 + 64) 2^-23.

For a 16-bit result the products of codes run with offsets of up to 4 |q| until a group's end: terms
of 16 * 5 scale |q| <= 12 M |q|, in sums of 32 channels that are added eight times at most, 8 2^-23
of them more. Queries are float16 then, of 2^-25 of a row's largest where they are less than 2^-14 of
it. And weights times scales are rounded twice to bfloat16, 2 2^-8 of scale |code - 7.5| <= 1.1 M, and
once, half a unit, beside the middles.

Where values and weights are rounded to 16 bits (many rows), half a unit of that type is added to each. The
keys' codes times their scales are exact there; the middles multiply a group's sum of queries in two parts of
16 bits, which is off by 2^-17 of it, and queries below 2 lose 2^-25 of a row's largest in float16, as do the
parts and the products' second ones. The output's own rounding is half a unit more."""
import math

import numpy as np

import uor_b200 as U
from q4_data import TORCH, UNIT, round_bound

try:
    import torch
except Exception:  # pragma: no cover
    torch = None

MOST = {U.BF16: 3.3895313892515355e38, U.F16: 65504.0}


def held(x, group):
    """What the cache holds of x (.., dim) of a 16-bit type, in float64: every step that the definition
    rounds to f32 is one of f32."""
    kind = x.dtype
    most = MOST[U.BF16 if kind == torch.bfloat16 else U.F16]
    v = torch.nan_to_num(x.float(), nan=0.0, posinf=most, neginf=-most).unflatten(-1, (-1, group))
    high, low = v.amax(-1, keepdim=True), v.amin(-1, keepdim=True)
    mid = (high * 0.5 + low * 0.5).to(kind).float()
    scale = ((high * 0.5 - low * 0.5) / 7.5).to(kind)
    past = 7.5 * scale.double() + mid.abs().double() > most
    scale = torch.where(past, (scale.view(torch.int16) - 1).view(kind), scale).float()
    code = ((v - mid) / scale + 7.5).round().clamp(0, 15)
    code = torch.where(scale > 0, code, torch.zeros_like(code))
    return (mid.double() + scale.double() * (code.double() - 7.5)).flatten(-2)


def rotated(x, cos, sin, dims, interleaved):
    """x (rows, heads, dim) with rows of cos, sin (rows, dims / 2), rounded as the library rounds."""
    if not dims:
        return x
    first = torch.arange(dims // 2, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else dims // 2)
    a, b, c, s = x[..., first].double(), x[..., second].double(), cos.double()[:, None], sin.double()[:, None]
    y = x.clone()
    y[..., first] = (a * c - b * s).float().to(x.dtype)
    y[..., second] = (b * c + a * s).float().to(x.dtype)
    return y


class Cache:
    """A cache of `lengths` tokens per sequence in pages strewn over a pool of random bytes, and the
    batch of each sequence's newest `news` tokens, with `pad` rows behind the last."""

    def __init__(self, lengths, news, page=16, heads=2, dim=64, group=32, elem=U.BF16, pad=0, spare=2, seed=0,
                 extra_pages=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.lengths, self.news, self.page, self.heads, self.dim, self.group, self.elem = (
            lengths, news, page, heads, dim, group, elem)
        self.kind, self.g = TORCH[elem], g
        counts = [-(-n // page) for n in lengths]
        self.pages, self.cols = sum(counts) + spare, max(max(counts) + extra_pages, 1)
        order = torch.randperm(self.pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lengths), self.cols), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(counts):
            self.table[i, :n] = order[at:at + n]
            at += n
        size = U.kv4_page_bytes(page, heads, dim, group, elem)
        self.pool = torch.randint(0, 256, (self.pages * size,), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
        self.kv = U.KV4(self.pool, self.pages, page, heads, dim, group, elem)
        self.batch = self.batch_of(news)
        self.rows = sum(news) + pad

    def batch_of(self, news, lengths=None):
        starts = np.concatenate([[0], np.cumsum(news)])
        as_ints = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        return U.Batch(as_ints(starts), as_ints(self.lengths if lengths is None else lengths), self.table, len(news), self.cols)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def fill(self, ctx=None, size=1.0, shift=0.0):
        """Appends whole sequences of random keys and values; keeps what the cache then holds of them
        (per sequence (length, heads, dim), float64)."""
        rows, wide = sum(self.lengths), self.heads * self.dim
        k = (self.normal(rows, wide) * size + shift).to(self.kind)
        v = (self.normal(rows, wide) * size + shift).to(self.kind)
        U.kv4_append(self.elem, self.kv, self.batch_of(self.lengths), k, (rows, wide), v, (rows, wide), ctx=ctx)
        cut = lambda x: torch.split(held(x.view(rows, self.heads, self.dim), self.group), self.lengths)  # noqa: E731
        self.k, self.v = cut(k), cut(v)
        return self

    def queries(self, share, size=1.5):
        return (self.normal(self.rows, self.heads * share * self.dim) * size).to(self.kind)


def seen_by(at, keys, window, sinks, device="cuda"):
    """Which of the positions 0 .. keys - 1 a row at position `at` (a column of them) sees."""
    j = torch.arange(keys, device=device)[None]
    ok = j <= at[:, None]
    if window:
        ok = ok & ((j > at[:, None] - window) | (j < sinks))
    return ok


def attention(cache, q, share, scale, out, window=0, sinks=0, rounded=False, keys_of=None):
    """(y, y's bound, lse, lse's bound) in float64; rows that no sequence has are NaN in y. keys_of:
    per sequence, the keys that are there at all (default: its length)."""
    rows, dim = q.shape[0], cache.dim
    nan = lambda *s: torch.full(s, math.nan, dtype=torch.float64, device="cuda")  # noqa: E731
    y, y_off = nan(rows, cache.heads * share, dim), nan(rows, cache.heads * share, dim)
    lse, lse_off = nan(rows, cache.heads * share), nan(rows, cache.heads * share)
    unit = UNIT[cache.elem]
    start = 0
    biggest = lambda x: 6 * x.abs().unflatten(-1, (-1, cache.group)).amax(-1).repeat_interleave(cache.group, -1)  # noqa: E731
    for i, (n, length) in enumerate(zip(cache.news, cache.lengths)):
        there = cache.k[i].shape[0]
        at = torch.arange(length - n, length, device="cuda")
        ok = seen_by(at, there, window, sinks)
        if keys_of is not None:
            ok = ok & keys_of[i][None]
        for h in range(cache.heads * share):
            k, v = cache.k[i][:, h // share], cache.v[i][:, h // share]
            x = q[start:start + n].double().view(n, -1, dim)[:, h]
            s = (x @ k.T * scale).masked_fill(~ok, -math.inf)
            empty = ~ok.any(1)
            top = s.amax(1, keepdim=True).masked_fill(empty[:, None], 0.0) if there else torch.zeros(n, 1, device="cuda").double()
            p = torch.exp(s - top)
            total = p.sum(1, keepdim=True)
            share_of = torch.where(total > 0, p / total.clamp(min=1e-300), torch.zeros_like(p))
            y[start:start + n, h] = share_of @ v
            lse[start:start + n, h] = (top + torch.log(total))[:, 0]
            off = (dim / 8 + 16) * 2.0 ** -23 * abs(scale) * (x.abs() @ biggest(k).T)
            if out != U.F32:
                off = off + abs(scale) * (8 * 2.0 ** -23 * (x.abs() @ (2 * biggest(k)).T)
                                          + 2.0 ** -25 * x.abs().amax(1, keepdim=True) * biggest(k).sum(1)[None])
            if rounded:
                off = off + abs(scale) * (2.0 ** -17 * (x.abs() @ (biggest(k) / 6).T)
                                          + 3 * 2.0 ** -25 * x.abs().amax(1, keepdim=True) * (biggest(k) / 6).sum(1)[None])
            off = off.masked_fill(~ok, 0.0) + s.abs().masked_fill(~ok, 0.0) * 2.0 ** -22
            worst = off.amax(1, keepdim=True) if there else torch.zeros(n, 1, device="cuda").double()
            by = 2 * torch.expm1(worst) + 2.0 ** -19 + 2.0 ** -16 + (there / 16 + 64) * 2.0 ** -23 + (3 * unit if rounded else 0.0)
            y_off[start:start + n, h] = by * (share_of @ biggest(v))
            if out != U.F32 and not rounded:
                y_off[start:start + n, h] += (2.2 * 2.0 ** -8 + unit) * (share_of @ (biggest(v) / 6))
            if rounded:  # a score's own error is as a rule far below the worst; values and weights 3 units of what they hold
                y_off[start:start + n, h] = ((2 * torch.expm1(worst) + 3 * unit) * (share_of @ v.abs())
                                             + (2.0 ** -16 + (there / 16 + 64) * 2.0 ** -23) * (share_of @ biggest(v)))
            lse_off[start:start + n, h] = (worst[:, 0] + 2.0 ** -18 + (there / 16 + 64) * 2.0 ** -23
                                           + 2.0 ** -22 * lse[start:start + n, h].abs().nan_to_num(0, 0, 0))
        start += n
    y, y_off = y.view(rows, -1), y_off.view(rows, -1)
    return y, y_off + round_bound(y.abs() + y_off, out), lse, lse_off
