"""The router and its gradient against the formulas in 64 bits.

Weights are held to (128 + |logit - top|) 2^-24 of their value: exp is within 2 units, its argument's
rounding moves it by |logit - top| 2^-24, a row's sum of up to 1024 terms is joined in at most 37
steps, and the divisions and products add a few units each. A gradient is a difference of such
terms, so its bound is that share of the terms' magnitudes."""
import numpy as np
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, UNIT, generator

pytestmark = [pytest.mark.gpu, needs_gpu]
INF = float("inf")
SHARE = 128 * 2.0 ** -24


def scores(logits, router):
    x = logits.double()
    open_ = x > -INF  # False for NaN
    if router.score == U.SIGMOID:
        return torch.where(open_, torch.sigmoid(x), torch.zeros_like(x)), open_
    top = torch.where(open_, x, torch.full_like(x, -INF)).amax(1, keepdim=True)
    p = torch.where(open_, torch.where(x == top, torch.ones_like(x), torch.exp(x - top)), torch.zeros_like(x))
    total = p.sum(1, keepdim=True)
    return torch.where(total > 0, p / total, torch.zeros_like(p)), open_


def choose(logits, router, bias):
    """(ids, rows decided beyond f32's rounding) by stable sorts of the float64 keys."""
    s, open_ = scores(logits, router)
    key = s if bias is None else s + bias.double()
    key = torch.where(open_ & (key > -INF), key, torch.full_like(key, -INF))
    sure = torch.ones(key.shape[0], dtype=torch.bool, device=key.device)

    def gaps(v, upto):
        v = v[:, :upto]
        d = v[:, :-1] - v[:, 1:]
        return ((d == 0) | (d > 1e-5 * (v[:, :-1].abs() + 1e-3)) | torch.isnan(d)).all(1)

    if router.top_groups < router.groups:
        by = key.view(key.shape[0], router.groups, -1)
        two = by.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        v, at = two.sort(dim=1, descending=True, stable=True)
        sure &= gaps(v, router.groups)
        keep = torch.zeros_like(two, dtype=torch.bool).scatter_(1, at[:, :router.top_groups], True)
        key = torch.where(keep[:, :, None], by, torch.full_like(by, -INF)).flatten(1)
    v, at = key.sort(dim=1, descending=True, stable=True)
    sure &= gaps(v, router.top_k + 1)
    at, v = at[:, :router.top_k], v[:, :router.top_k]
    return torch.where(v > -INF, at, torch.full_like(at, -1)), sure


def weights_of(logits, router, ids):
    s, _ = scores(logits, router)
    w = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0).long()), torch.zeros(1, dtype=torch.float64, device=s.device))
    if router.renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return w * router.scale


def gradient(logits, router, ids, dweights):
    """The formula, with the bound of its terms."""
    s, open_ = scores(logits, router)
    held, at = ids >= 0, ids.clamp(min=0).long()
    zero = torch.zeros(1, dtype=torch.float64, device=s.device)
    mine = torch.where(held, s.gather(1, at), zero)
    g = torch.where(held, dweights.double(), zero) * router.scale
    size = g.abs()
    if router.renormalize:
        total = mine.sum(1, keepdim=True)
        w = torch.where(total > 0, mine / total, zero)
        size = torch.where(total > 0, (size + (size * w).sum(1, keepdim=True)) / total, zero)
        g = torch.where(total > 0, (g - (g * w).sum(1, keepdim=True)) / total, zero)
    d = torch.zeros_like(s).scatter_add_(1, at, torch.where(held, g, zero))
    z = torch.zeros_like(s).scatter_add_(1, at, torch.where(held, size, zero))
    if router.score == U.SIGMOID:
        return d * s * (1 - s), z * s
    return s * (d - (d * s).sum(1, keepdim=True)), s * (z + (z * s).sum(1, keepdim=True))


def spread_logits(t, e, elem, seed):
    """Rows of distinct, well separated logits in random order (exact in bfloat16 for e <= 256)."""
    order = torch.rand(t, e, generator=generator(seed), device="cuda").argsort(1)
    return ((order - e // 2).float() * (8.0 / e if e & (e - 1) else 2.0 ** (3 - (e.bit_length() - 1)))).to(TORCH[elem])


def route(logits, router, bias=None, elem=U.F32, iv=None, wv=None, lv=None, **more):
    t, k = logits.shape[0], router.top_k
    ids = torch.full((t, k), -9, device="cuda", dtype=torch.int32)
    w = torch.full((t, k), -9.0, device="cuda")
    r = U.Route()
    U.expert_route(elem, router, logits, lv or (t, router.experts), bias, ids, iv or (t, k), w, wv or (t, k), route=r, **more)
    assert r.kernel == 9
    return ids, w


def check(logits, router, bias=None, elem=U.F32, least=0.9):
    ids, w = route(logits, router, bias, elem)
    want, sure = choose(logits, router, bias)
    assert float(sure.double().mean()) >= least
    assert torch.equal(ids[sure].long(), want[sure])
    value = weights_of(logits, router, ids)
    reach = torch.nan_to_num(logits.double(), nan=0, posinf=0, neginf=0)
    reach = (reach.amax(1) - reach.amin(1))[:, None] * 2.0 ** -24
    assert bool(((w.double() - value).abs() <= (SHARE + reach) * value.abs() + 1e-37).all())
    return ids, w


@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 1), (5, 5), (31, 7), (32, 32), (33, 4), (60, 4), (64, 6), (100, 9),
                                           (128, 8), (160, 6), (256, 8), (384, 8), (512, 10), (1000, 3), (1024, 32)])
@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
def test_choice_and_weights(experts, top_k, score):
    for t in (1, 9, 257):
        for renormalize in (False, True):
            r = U.Router(experts, top_k, score, renormalize=renormalize, scale=1.5)
            check(spread_logits(t, experts, U.F32, experts + t), r)


@pytest.mark.parametrize("elem", [U.F32, U.BF16, U.F16])
@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
def test_types(elem, score):
    for e in (16, 64, 256):
        check(spread_logits(100, e, elem, e), U.Router(e, 4, score), elem=elem)


@pytest.mark.parametrize("experts,groups,top_groups", [(256, 8, 4), (64, 4, 1), (60, 6, 2), (32, 32, 5), (32, 16, 3),
                                                       (160, 8, 3), (96, 3, 2), (1024, 32, 4), (8, 2, 1), (256, 8, 8),
                                                       (128, 1, 1), (64, 2, 1)])
@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
def test_groups_and_bias(experts, groups, top_groups, score):
    g = generator(experts + groups)
    for biased in (False, True):
        bias = torch.randn(experts, generator=g, device="cuda") * (0.05 if score == U.SIGMOID else 0.2 / experts) if biased else None
        top_k = min(6, experts // groups * top_groups)
        r = U.Router(experts, top_k, score, groups, top_groups, True, 2.5)
        logits = torch.randn(300, experts, generator=g, device="cuda") * 1.5
        check(logits, r, bias, least=0.8)


@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
@pytest.mark.parametrize("groups", [1, 4])
def test_ties_go_to_the_lowest_index(score, groups):
    e = 64
    r = U.Router(e, 6, score, groups, max(1, groups // 2))
    same = torch.zeros(3, e, device="cuda")
    ids, w = check(same, r)
    assert torch.equal(ids.cpu(), torch.arange(6, dtype=torch.int32).expand(3, 6))
    few = torch.randint(-2, 3, (500, e), generator=generator(4), device="cuda").float()
    check(few, r, least=1.0)


@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
@pytest.mark.parametrize("renormalize", [False, True])
def test_masks(score, renormalize):
    """Rows with everything, all but one and all but a few experts closed; the type's lowest value."""
    e = 70
    r = U.Router(e, 5, score, renormalize=renormalize)
    logits = spread_logits(40, e, U.F32, 1)
    logits[0] = -INF
    logits[1, 1:] = -INF
    logits[2, 3:] = float("nan")
    logits[3, ::2] = -INF
    logits[4] = float("nan")
    logits[5, 10] = INF
    logits[6, 10] = logits[6, 60] = INF
    logits[7] = torch.finfo(torch.float32).min
    logits[8, 5:] = torch.finfo(torch.float32).min
    logits[9] = logits[9] * 0 - 200.0
    ids, w = check(logits, r, least=0.0)
    want, _ = choose(logits, r, None)
    assert torch.equal(ids[:10].long(), want[:10])
    assert bool((ids[0] == -1).all()) and bool((w[0] == 0).all())
    assert ids[1].tolist() == [0, -1, -1, -1, -1]
    assert sorted(ids[2, :3].tolist()) == [0, 1, 2] and ids[2, 3:].tolist() == [-1, -1]
    assert ids[5, 0] == 10 and ids[6, :2].tolist() == [10, 60]
    assert bool(torch.isfinite(w).all())


def test_bias_that_shuts_and_forces():
    e = 40
    bias = torch.zeros(e, device="cuda")
    bias[:10] = -INF
    bias[11] = float("nan")
    bias[33] = INF
    logits = spread_logits(50, e, U.F32, 3)
    ids, _ = route(logits, U.Router(e, 4, U.SIGMOID), bias)
    assert bool((ids[:, 0] == 33).all()) and bool((ids[:, 1:] >= 10).all()) and not bool((ids == 11).any())
    rest = torch.where(torch.isinf(bias) | torch.isnan(bias), torch.full_like(bias, -INF), bias)
    want, _ = choose(logits, U.Router(e, 3, U.SIGMOID), rest)
    assert torch.equal(ids[:, 1:].long(), want)


def test_strides():
    t, e, k = 37, 48, 5
    r = U.Router(e, k, U.SIGMOID)
    base = spread_logits(t, e, U.F32, 6)
    want, _ = route(base, r)
    wide = torch.full((t, e + 5), 9.0, device="cuda")
    wide[:, :e] = base
    turned = base.t().contiguous()
    for buf, lv in ((wide, (t, e, e + 5, 1)), (turned, (t, e, 1, t))):
        ids = torch.full((k, t + 2), -9, device="cuda", dtype=torch.int32)
        w = torch.full((t, 2 * k), -9.0, device="cuda")
        U.expert_route(U.F32, r, buf, lv, None, ids, (t, k, 1, t + 2), w, (t, k, 2 * k, 2))
        assert torch.equal(ids[:, :t].t(), want) and bool((ids[:, t:] == -9).all())
        assert bool((w[:, 1::2] == -9).all())


def test_host_arrays_and_no_tokens():
    t, e, k = 11, 24, 3
    r = U.Router(e, k)
    logits = spread_logits(t, e, U.F32, 2)
    bias = torch.linspace(0, 0.01, e, device="cuda")
    ids, w = route(logits, r, bias)
    hi, hw = np.zeros((t, k), np.int32), np.zeros((t, k), np.float32)
    U.expert_route(U.F32, r, logits.cpu().numpy(), (t, e), bias.cpu().numpy(), hi, (t, k), hw, (t, k))
    assert np.array_equal(hi, ids.cpu().numpy()) and np.array_equal(hw, w.cpu().numpy())
    none = torch.empty(0, e, device="cuda")
    U.expert_route(U.F32, r, none, (0, e), None, ids, (0, k), w, (0, k))


def back(logits, router, ids, dweights, elem=U.F32):
    t, e, k = logits.shape[0], router.experts, router.top_k
    d = torch.full((t, e), 5.0, device="cuda", dtype=TORCH[elem])
    U.expert_route_backward(elem, router, logits, (t, e), ids, (t, k), dweights, (t, k), d, (t, e))
    return d


@pytest.mark.parametrize("experts,top_k", [(1, 1), (5, 2), (32, 32), (60, 4), (64, 6), (200, 8), (256, 8), (1024, 32)])
@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("elem", [U.F32, U.BF16, U.F16])
def test_gradient(experts, top_k, score, renormalize, elem):
    for t in (1, 130):
        r = U.Router(experts, top_k, score, renormalize=renormalize, scale=2.5)
        logits = spread_logits(t, experts, elem, t + experts)
        logits[::7, ::5] = -INF
        ids, _ = route(logits, r, elem=elem)
        dw = torch.randn(t, top_k, generator=generator(8), device="cuda")
        got = back(logits, r, ids, dw, elem).double()
        want, size = gradient(logits, r, ids, dw)
        bound = 2 * SHARE * size + (UNIT[elem] * want.abs() + (2.0 ** -25 if elem == U.F16 else 0)) * 1.01 + 1e-37
        assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_against_differences(score, renormalize):
    """Central differences of the forward kernel's own weights, the choice unchanged by the step:
    off by h^2 / 6 of a third derivative (below 1 for these scores) and 2^-22 / h of rounding."""
    e, k, h = 12, 4, 2.0 ** -6
    r = U.Router(e, k, score, renormalize=renormalize)
    logits = spread_logits(6, e, U.F32, 5)
    ids, _ = route(logits, r)
    dw = torch.randn(6, k, generator=generator(1), device="cuda")
    got = back(logits, r, ids, dw).double()
    for i in range(e):
        step = torch.zeros_like(logits)
        step[:, i] = h
        (up_ids, up), (down_ids, down) = route(logits + step, r), route(logits - step, r)
        assert torch.equal(up_ids, ids) and torch.equal(down_ids, ids)
        slope = ((up.double() - down.double()) / (2 * h) * dw.double()).sum(1)
        bound = (h * h / 6 + 2.0 ** -22 / h) * dw.double().abs().sum(1) * 2
        assert bool(((got[:, i] - slope).abs() <= bound).all())


def test_gradient_of_odd_choices():
    """Ids outside the experts take no part, an expert chosen twice gets both gradients, a masked
    row's gradient is zero, infinities and NaN among the closed logits reach nothing."""
    e, k = 40, 4
    logits = spread_logits(8, e, U.F32, 7)
    logits[1] = -INF
    logits[2, 30:] = float("nan")
    ids = torch.tensor([[0, 1, 2, 3], [-1, -1, -1, -1], [4, 4, 9, -1], [40, 5, -7, 5], [1, 1, 1, 1], [39, 38, 0, 2],
                        [7, 8, 9, 10], [3, -1, -1, -1]], device="cuda", dtype=torch.int32)
    dw = torch.randn(8, k, generator=generator(2), device="cuda")
    for score in (U.SOFTMAX, U.SIGMOID):
        for renormalize in (False, True):
            r = U.Router(e, k, score, renormalize=renormalize)
            got = back(logits, r, ids, dw).double()
            kept = torch.where((ids >= 0) & (ids < e), ids, torch.full_like(ids, -1))
            want, size = gradient(logits, r, kept, dw)
            assert bool((got[1] == 0).all()) and bool(torch.isfinite(got).all())
            assert bool((got[2, 30:] == 0).all())
            assert bool(((got - want).abs() <= 2 * SHARE * size + 2.0 ** -23 * want.abs() + 1e-37).all())


def test_gradient_strides_and_host():
    t, e, k = 19, 33, 3
    r = U.Router(e, k, U.SIGMOID)
    logits = spread_logits(t, e, U.F32, 1)
    ids, _ = route(logits, r)
    dw = torch.randn(t, k, generator=generator(3), device="cuda")
    want = back(logits, r, ids, dw)
    turned = torch.zeros(e, t + 1, device="cuda")
    U.expert_route_backward(U.F32, r, logits.t().contiguous(), (t, e, 1, t), ids, (t, k), dw.t().contiguous(), (t, k, 1, t),
                            turned, (t, e, 1, t + 1))
    assert torch.equal(turned[:, :t].t(), want) and bool((turned[:, t] == 0).all())
    host = np.zeros((t, e), np.float32)
    U.expert_route_backward(U.F32, r, logits.cpu().numpy(), (t, e), ids.cpu().numpy(), (t, k), dw.cpu().numpy(), (t, k),
                            host, (t, e))
    assert np.array_equal(host, want.cpu().numpy())
