"""Inputs, 64-bit references and error bounds for the 4-bit family's tests.

The bounds are derived, not fitted. A sum held in f32 with at most D additions one after another
is off by at most D 2^-23 times the sum of its terms' magnitudes (an addition, truncated or
rounded, is off by at most 2^-23 of a partial sum, which that sum bounds). No kernel chains more
than a term per 8 positions of the reduction and 64 joins, so D = k / 8 + 64. Rounding to the
output adds half a unit: 2^-8 of the value for bfloat16, 2^-11 for float16 (2^-25 absolute below
its normal range), 2^-24 for float32."""
import numpy as np

import uor_b200 as U

try:
    import torch
except Exception:  # pragma: no cover
    torch = None

TORCH = {} if torch is None else {U.BF16: torch.bfloat16, U.F16: torch.float16, U.F32: torch.float32}
UNIT = {U.BF16: 2.0 ** -8, U.F16: 2.0 ** -11, U.F32: 2.0 ** -24}


def generator(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


class Weights:
    """rows x cols random 4-bit weights: the library's descriptor and their float64 values.
    pad: bytes between rows of codes; groups_pad: elements between rows of scales; shift: bytes by
    which the codes begin past an aligned address."""

    def __init__(self, rows, cols, group, scale_type=None, zeros=True, seed=0, pad=0, groups_pad=0, shift=0,
                 spread=None, device="cuda"):
        scale_type = U.F32 if scale_type is None else scale_type
        g = generator(seed, device)
        groups = -(-cols // group)
        width = (cols + 1) // 2
        spread = cols ** -0.5 / 4 if spread is None else spread
        span = max(rows - 1, 0) * (width + pad) + width
        store = torch.randint(0, 256, (span + shift,), generator=g, device=device, dtype=torch.int32).to(torch.uint8)
        codes = store[shift:]
        gspan = max(rows - 1, 0) * (groups + groups_pad) + groups
        scales = ((torch.rand(gspan, generator=g, device=device) + 0.5) * spread).to(TORCH[scale_type])
        zero = torch.randint(0, 256, (gspan,), generator=g, device=device, dtype=torch.int32).to(torch.uint8) if zeros else None
        self.q = U.Q4(codes, scales, scale_type, rows, cols, group, zeros=zero, row_bytes=width + pad,
                      groups_rs=groups + groups_pad)
        by_row = codes.as_strided((rows, width), (width + pad, 1)).long()
        code = torch.stack((by_row & 15, by_row >> 4), 2).view(rows, 2 * width)[:, :cols]
        at = torch.arange(cols, device=device) // group
        pick = lambda v: v.as_strided((rows, groups), (groups + groups_pad, 1))[:, at]  # noqa: E731
        z = (pick(zero).long() & 15) if zeros else 8
        self.value = (code - z).double() * pick(scales).double()


def dot_bound(x, w, k):
    """The f32 sums' bound for x w^T in float64."""
    return (k / 8 + 64) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def round_bound(y, out):
    return UNIT[out] * y.abs() + (2.0 ** -25 if out == U.F16 else 0.0)


def assert_within(got, want, bound, what=""):
    """Element by element; what is not finite in `want` has to be the same in `got`."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine] - bound[fine]
    if off.numel():
        assert float(off.max()) <= 0, f"{what}: {float(off.max())} past its bound"


def ffn_reference(x, ids, weights, up, down, experts, elem, out):
    """(y, bound) in float64 of the experts' layer. With dg, du the bounds of the two inner sums,
    the inner activation h = silu(g) u (silu's slope is below 1.1 in size) is off by at most
    1.1 |u| dg + |silu(g)| du + 1.1 dg du, 8 2^-23 |h| for its own arithmetic and half a unit of
    `elem`; the outer sum carries that through |W| and adds its own."""
    t, d = x.shape
    f = down.shape[1]
    y = torch.zeros(t, d, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    size = torch.zeros_like(y)
    for e in range(experts):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if not token.numel():
            continue
        rows = x[token]
        wg, wu = up[e * 2 * f:e * 2 * f + f], up[e * 2 * f + f:(e + 1) * 2 * f]
        g, u = rows @ wg.T, rows @ wu.T
        dg, du = dot_bound(rows, wg, d), dot_bound(rows, wu, d)
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * u.abs() * dg + s.abs() * du + 1.1 * dg * du + 8 * 2.0 ** -23 * h.abs()
        dh = dh + round_bound(h.abs() + dh, elem)
        wd = down[e * d:(e + 1) * d]
        w = weights[token, slot].double()[:, None]
        part = h @ wd.T
        y.index_add_(0, token, part * w)
        off = dh @ wd.abs().T + dot_bound(h.abs() + dh, wd, f)
        bound.index_add_(0, token, off * w.abs())
        size.index_add_(0, token, part.abs() * w.abs())
    bound = bound + (ids.shape[1] + 4) * 2.0 ** -23 * (size + bound)
    return y, bound + round_bound(y.abs() + bound, out)
