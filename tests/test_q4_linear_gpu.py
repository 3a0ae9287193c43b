"""q4_linear against 64 bits: bias, activation and residual behind each of the product's kernels, in
place, strided, of odd sizes; without any of them it is q4_gemm to the byte."""
import math

import numpy as np
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, Weights, assert_within, dot_bound, generator, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]

ACTS = [U.IDENTITY, U.RELU, U.GELU, U.GELU_TANH, U.SILU]


def _act(v, act):
    f = torch.nn.functional
    if act == U.GELU:  # the tails included: 1 + erf and 1 + tanh are off by 2^-54 in 64 bits too
        return 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    if act == U.GELU_TANH:
        return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return {U.IDENTITY: lambda x: x, U.RELU: f.relu, U.SILU: f.silu}[act](v)


def _want(x, w, bias, act, residual, out):
    """Every activation's slope is below 1.13 in size; its own f32 arithmetic is off by at most 2^-18 of
    its result (an exponent of up to 100 with a relative error of a few 2^-24) and of the value where
    both are small."""
    v = x.double() @ w.T
    off = dot_bound(x.double(), w, w.shape[1])
    if bias is not None:
        v = v + bias.double()
        off = off + 2.0 ** -23 * v.abs()
    y = _act(v, act)
    off = 1.13 * off + (2.0 ** -18 * y.abs() + 2.0 ** -24 if act else 0.0)
    if residual is not None:
        y = y + residual.double()
        off = off + 2.0 ** -23 * (y.abs() + off)
    return y, off + round_bound(y.abs() + off, out)


# few rows read directly, through shared memory, many rows, many with a split reduction, no reduction
SIZES = [(1, 256, 512, 64), (1, 4096, 1024, 128), (5, 77, 520, 32), (13, 130, 1001, 32), (40, 300, 256, 128), (700, 520, 1000, 64), (700, 1040, 1000, 64),
         (300, 200, 4096, 128), (130, 1000, 128, 32), (3, 33, 0, 32)]


@pytest.mark.parametrize("m,n,k,group", SIZES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("elem,out", [(U.BF16, U.BF16), (U.F16, U.F32)])
def test_against_64_bits(m, n, k, group, act, elem, out):
    g = generator(m + n + act)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = Weights(n, k, group, seed=n, zeros=act % 2 == 0, spread=max(k, 1) ** -0.5 / 4)
    x = normal(m, k).to(TORCH[elem])
    for bias, residual in ((normal(n).to(TORCH[elem]), normal(m, n).to(TORCH[out])), (normal(n), None), (None, normal(m, n).to(TORCH[out]))):
        y = torch.full((m, n), 5.0, device="cuda", dtype=TORCH[out])
        U.q4_linear(elem, out, x, (m, k), w.q, y, (m, n), bias=bias, activation=act, residual=residual)
        want, off = _want(x, w.value, bias, act, residual, out)
        assert_within(y, want, off)
    if act == U.IDENTITY:
        plain, y = torch.empty(m, n, device="cuda", dtype=TORCH[out]), torch.empty(m, n, device="cuda", dtype=TORCH[out])
        U.q4_gemm(elem, out, x, (m, k), w.q, plain, (m, n))
        U.q4_linear(elem, out, x, (m, k), w.q, y, (m, n))
        assert torch.equal(y, plain)


@pytest.mark.parametrize("m,n,k", [(1, 512, 256), (9, 131, 512), (300, 264, 4096), (700, 1100, 1000)])
@pytest.mark.parametrize("elem,out", [(U.F16, U.F16), (U.BF16, U.F32)])
def test_added_in_place(m, n, k, elem, out):
    """The residual is the output: the stream that a projection is added to."""
    g = generator(m)
    w = Weights(n, k, 32, seed=1)
    x = torch.randn(m, k, generator=g, device="cuda").to(TORCH[elem])
    stream = torch.randn(m, n, generator=g, device="cuda").to(TORCH[out])
    want, apart = stream.clone(), torch.empty_like(stream)
    U.q4_linear(elem, out, x, (m, k), w.q, apart, (m, n), activation=U.SILU, residual=want)
    U.q4_linear(elem, out, x, (m, k), w.q, stream, (m, n), activation=U.SILU, residual=stream)
    assert torch.equal(stream, apart)


@pytest.mark.parametrize("m,n,k", [(2, 96, 512), (7, 130, 520), (260, 130, 4096), (700, 1100, 1000)])
def test_strides(m, n, k):
    """A residual and an output of columns down the rows, reversed, with gaps; gaps stay."""
    g = generator(n)
    w = Weights(n, k, 32, seed=2)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    bias = torch.randn(n + 1, generator=g, device="cuda").bfloat16()[1:]
    residual = torch.randn(m * n, generator=g, device="cuda")
    y = torch.full((m * (2 * n + 1),), 5.0, device="cuda")
    U.q4_linear(U.BF16, U.F32, x, (m, k), w.q, y, (m, n, 2 * n + 1, -2), bias=bias, activation=U.GELU, residual=residual, rv=(m, n, 1, m))
    want, off = _want(x, w.value, bias, U.GELU, residual.view(n, m).T, U.F32)
    rows = y.view(m, 2 * n + 1)
    assert_within(rows[:, 0:2 * n:2].flip(1), want, off)
    assert bool((rows[:, 1:2 * n:2] == 5.0).all()) and bool((rows[:, 2 * n] == 5.0).all())


@pytest.mark.parametrize("m,k", [(2, 64), (300, 4096)])
@pytest.mark.parametrize("act", ACTS)
def test_extremes(m, k, act):
    """Large sums of both signs, infinities and NaN through the activations, as their formulas have them."""
    n = 64
    w = Weights(n, k, 32, seed=3)
    x = torch.zeros(m, k, device="cuda").half()
    bias = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 12.0, -12.0, 40.0, -40.0, 90.0, -90.0, 1e4, -1e4, 1e13, -1e13, 3e38,
                         math.inf, math.nan], device="cuda")
    bias = torch.cat((bias, torch.linspace(-15, 15, n - len(bias), device="cuda")))
    y = torch.empty(m, n, device="cuda")
    U.q4_linear(U.F16, U.F32, x, (m, k), w.q, y, (m, n), bias=bias, activation=act)
    want = _act(bias.double(), act)[None].expand(m, n)
    # an exponent z carries 2^-22 |z|, so results below 2^-60 are compared in size alone
    off = 2.0 ** -14 * want.abs() + 2.0 ** -60
    assert_within(y, want, off)


@pytest.mark.parametrize("m", [3, 200])
def test_host_arrays(m):
    g = np.random.default_rng(0)
    n, k = 70, 128
    codes = g.integers(0, 256, n * k // 2, dtype=np.uint8)
    scales = (g.random(n * k // 32, dtype=np.float32) + 0.5) * 0.02
    q = U.Q4(codes, scales, U.F32, n, k, 32)
    x = g.standard_normal((m, k)).astype(np.float16)
    bias, residual = g.standard_normal(n).astype(np.float32), g.standard_normal((m, n)).astype(np.float32)
    y = np.empty((m, n), np.float32)
    U.q4_linear(U.F16, U.F32, x, (m, k), q, y, (m, n), bias=bias, activation=U.RELU, residual=residual)
    c = np.stack((codes & 15, codes >> 4), 1).reshape(n, k).astype(np.float64) - 8
    w = c * np.repeat(scales.reshape(n, -1).astype(np.float64), 32, 1)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a))  # noqa: E731
    want, off = _want(to(x), to(w), to(bias), U.RELU, to(residual), U.F32)
    assert_within(to(y), want, off)
    added = residual.copy()
    U.q4_linear(U.F16, U.F32, x, (m, k), q, added, (m, n), bias=bias, activation=U.RELU, residual=added)
    assert np.array_equal(added, y)
