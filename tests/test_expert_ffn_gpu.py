"""The experts' gated feed-forward layer over 4-bit weights against the formula in 64 bits."""
import numpy as np
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, Weights, assert_within, ffn_reference, generator

pytestmark = [pytest.mark.gpu, needs_gpu]


class Layer:
    def __init__(self, experts, d, f, group=32, scale_type=None, zeros=True, seed=0, **more):
        self.experts, self.d, self.f = experts, d, f
        self.up = Weights(experts * 2 * f, d, group, scale_type, zeros, seed=seed + 1, **more)
        self.down = Weights(experts * d, f, group, scale_type, zeros, seed=seed + 2, **more)

    def run(self, x, ids, weights, elem=U.BF16, out=None, **more):
        out = elem if out is None else out
        t, k = ids.shape
        y = torch.full((t, self.d), 7.0, device="cuda", dtype=TORCH[out])
        r = U.Route()
        U.expert_q4_ffn(elem, out, self.experts, x, (t, self.d), ids, (t, k), weights, (t, k), self.up.q, self.down.q, y,
                        (t, self.d), route=r, **more)
        assert r.kernel == 8
        return y

    def check(self, x, ids, weights, elem=U.BF16, out=None):
        out = elem if out is None else out
        y = self.run(x, ids, weights, elem, out)
        want, bound = ffn_reference(x.double(), ids, weights, self.up.value, self.down.value, self.experts, elem, out)
        assert_within(y, want, bound, f"{tuple(ids.shape)} {self.experts} {self.d} {self.f}")
        return y


def tokens(t, d, experts, k, elem=U.BF16, seed=0, dropped=0.0):
    g = generator(seed)
    x = torch.randn(t, d, generator=g, device="cuda").to(TORCH[elem])
    ids = torch.rand(t, experts, generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32).contiguous()
    w = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), 1)
    lost = torch.rand(t, k, generator=g, device="cuda") < dropped
    return x, torch.where(lost, torch.full_like(ids, -1), ids), w


@pytest.mark.parametrize("t", [1, 2, 5, 8, 9, 16, 23, 32, 33, 50, 100, 300])
@pytest.mark.parametrize("experts,k", [(8, 2), (16, 8), (3, 1), (1, 1)])
def test_tokens(t, experts, k):
    layer = Layer(experts, 192, 96)
    layer.check(*tokens(t, 192, experts, k, seed=t))


@pytest.mark.parametrize("d,f,group", [(1, 1, 32), (2, 3, 32), (33, 17, 32), (64, 64, 64), (130, 129, 128), (200, 8, 64),
                                       (8, 200, 32), (256, 130, 128), (257, 255, 64), (1000, 344, 32), (640, 512, 256),
                                       (96, 160, 96)])
@pytest.mark.parametrize("t", [1, 7, 40, 150])
def test_sizes(d, f, group, t):
    layer = Layer(6, d, f, group)
    layer.check(*tokens(t, d, 6, 3, seed=d))


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("scale_type", [U.F32, U.BF16, U.F16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("t", [1, 30, 90])
def test_types(elem, scale_type, zeros, t):
    layer = Layer(5, 128, 160, 64, scale_type, zeros)
    x, ids, w = tokens(t, 128, 5, 2, elem)
    for out in (elem, U.F32):
        layer.check(x, ids, w, elem, out)


@pytest.mark.parametrize("t", [1, 6, 30, 120])
def test_dropped_choices(t):
    """Ids outside the experts are skipped, whatever weight and activation stand beside them."""
    layer = Layer(9, 160, 64)
    x, ids, w = tokens(t, 160, 9, 4, dropped=0.4, seed=t)
    ids[0] = torch.tensor([-1, 9, 1000000, -2147483648])
    w[0, 0], w[0, 1] = float("nan"), float("inf")
    y = layer.check(x, ids, torch.where((ids < 0) | (ids >= 9), torch.zeros_like(w), w))
    again = layer.run(x, ids, w)
    assert torch.equal(y, again) and bool((y[0] == 0).all())


@pytest.mark.parametrize("t", [1, 3, 20, 140])
def test_one_expert_for_all_and_none_for_the_rest(t):
    layer = Layer(7, 96, 128)
    x, ids, w = tokens(t, 96, 7, 1, seed=t)
    ids[:] = 5
    layer.check(x, ids, w)
    ids[:] = -1
    assert bool((layer.run(x, ids, w) == 0).all())


@pytest.mark.parametrize("t", [2, 17, 90])
def test_expert_chosen_twice(t):
    layer = Layer(4, 64, 96)
    x, ids, w = tokens(t, 64, 4, 3, seed=t)
    ids[:, 2] = ids[:, 0]
    layer.check(x, ids, w)


@pytest.mark.parametrize("t", [4, 60])
def test_not_finite_stays_with_its_token(t):
    layer = Layer(6, 128, 64)
    x, ids, w = tokens(t, 128, 6, 2, seed=t)
    clean = layer.run(x, ids, w)
    x[1, 3] = float("inf")
    w2 = w.clone()
    w2[2, 0] = float("nan")
    y = layer.run(x, ids, w2)
    rest = torch.ones(t, dtype=torch.bool, device="cuda")
    rest[1] = rest[2] = False
    assert torch.equal(y[rest], clean[rest])
    assert bool(torch.isnan(y[2]).all()) and not bool(torch.isfinite(y[1]).all())
    # an expert with a NaN scale reaches its own tokens alone
    scales = layer.up.q.arrays[1]
    groups = 4
    scales[(3 * 128) * groups] = float("nan")
    y = layer.run(x, ids, w)
    mine = (ids == 3).any(1)
    rest = ~mine
    rest[1] = False
    assert torch.equal(y[rest], clean[rest])
    mine[1] = False
    assert bool(torch.isnan(y[mine].float()).all())


def test_strided_and_unaligned():
    experts, d, f, t, k = 5, 72, 40, 21, 3
    for pad, shift in ((0, 0), (3, 1), (4, 4), (8, 16)):
        layer = Layer(experts, d, f, 32, pad=pad, shift=shift, groups_pad=pad % 2)
        x, ids, w = tokens(t, d, experts, k)
        want = layer.check(x, ids, w, out=U.F32)
        wide = torch.zeros(t, d + 7, device="cuda", dtype=torch.bfloat16)
        wide[:, :d] = x
        y = torch.full((d, t + 2), 3.0, device="cuda")
        U.expert_q4_ffn(U.BF16, U.F32, experts, wide, (t, d, d + 7, 1), ids.t().contiguous(), (t, k, 1, t), w.t().contiguous(),
                        (t, k, 1, t), layer.up.q, layer.down.q, y, (t, d, 1, t + 2))
        assert torch.equal(y[:, :t].t(), want) and bool((y[:, t:] == 3).all())


def test_no_choices_no_tokens_and_host():
    layer = Layer(4, 64, 32, scale_type=U.F16)
    x, ids, w = tokens(6, 64, 4, 2, U.F16)
    y = torch.full((6, 64), 3.0, device="cuda")
    U.expert_q4_ffn(U.F16, U.F32, 4, x, (6, 64), ids, (6, 0, 1, 1), w, (6, 0, 1, 1), layer.up.q, layer.down.q, y, (6, 64))
    assert bool((y == 0).all())
    U.expert_q4_ffn(U.F16, U.F32, 4, x, (0, 64), ids, (0, 2), w, (0, 2), layer.up.q, layer.down.q, y, (0, 64))
    want = layer.run(x, ids, w, U.F16)
    host = [U.Q4(q.arrays[0].cpu().numpy(), q.arrays[1].cpu().numpy(), U.F16, q.rows, q.cols, q.group,
                 zeros=q.arrays[2].cpu().numpy()) for q in (layer.up.q, layer.down.q)]
    hy = np.zeros((6, 64), np.float16)
    U.expert_q4_ffn(U.F16, U.F16, 4, x.cpu().numpy(), (6, 64), ids.cpu().numpy(), (6, 2), w.cpu().numpy(), (6, 2), *host, hy,
                    (6, 64))
    assert np.array_equal(hy, want.cpu().numpy())


def test_same_bytes_every_time():
    layer = Layer(8, 256, 128)
    for t in (3, 40, 200):
        x, ids, w = tokens(t, 256, 8, 4, seed=t)
        first = layer.run(x, ids, w)
        assert all(torch.equal(first, layer.run(x, ids, w)) for _ in range(3))
