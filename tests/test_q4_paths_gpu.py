"""The 4-bit family's kernels at the sizes that choose between them, against the formula in 64 bits:
the tensor-memory kernel (route tile of 256 rows) and the one for few rows (16)."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, Weights, assert_within, dot_bound, ffn_reference, generator, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]

MANY, FEW = 256, 16


def _gemm(m, n, k, group, tile, elem=U.BF16, out=None, y_strides=None, x_rs=None, **more):
    out = elem if out is None else out
    w = Weights(n, k, group, seed=n + k, **more)
    rs, cs = (n, 1) if y_strides is None else y_strides
    x = torch.randn((m - 1) * (x_rs or k) + k, generator=generator(m), device="cuda").to(TORCH[elem])
    x64 = x.as_strided((m, k), (x_rs or k, 1)).double()
    y = torch.full(((m - 1) * rs + (n - 1) * cs + 1,), -7.0, device="cuda", dtype=TORCH[out])
    route = U.Route()
    U.q4_gemm(elem, out, x, (m, k, x_rs or k, 1), w.q, y, (m, n, rs, cs), route=route)
    assert route.tile_m == tile
    want = x64 @ w.value.T
    off = dot_bound(x64, w.value, k)
    assert_within(y.as_strided((m, n), (rs, cs)), want, off + round_bound(want.abs() + off, out), f"{m}x{n}x{k} g{group}")


@pytest.mark.parametrize("m", [17, 31, 33, 64, 65, 127, 130, 193, 257, 300, 515])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_row_counts(m, group):
    _gemm(m, 144, 3712, group, MANY)


@pytest.mark.parametrize("n", [1, 2, 15, 17, 63, 127, 129, 250, 257, 1000])
@pytest.mark.parametrize("m", [40, 200])
def test_widths(m, n):
    _gemm(m, n, 3648, 64, MANY, elem=U.F16)


@pytest.mark.parametrize("k", [3585, 3586, 3599, 3601, 3711, 3713, 4104, 9000])
@pytest.mark.parametrize("m", [19, 150])
def test_reductions(m, k):
    _gemm(m, 70, k, 32, MANY)
    _gemm(m, 70, k, 128, MANY, out=U.F32)


@pytest.mark.parametrize("group", [32, 96, 160, 192, 256, 384, 1024, 4096])
@pytest.mark.parametrize("m", [33, 160])
def test_groups(m, group):
    _gemm(m, 100, 3680, group, MANY, zeros=group % 64 == 0, out=U.F32)


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("scale_type", [U.F32, U.BF16, U.F16])
@pytest.mark.parametrize("zeros", [False, True])
def test_types(elem, scale_type, zeros):
    for out in (elem, U.F32):
        _gemm(140, 96, 3840, 64, MANY, elem=elem, out=out, scale_type=scale_type, zeros=zeros)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (2, 4), (4, 0), (12, 16), (16, 16)])
@pytest.mark.parametrize("k", [3616, 3605])
def test_codes_anywhere(pad, shift, k):
    _gemm(133, 130, k, 32, MANY, pad=pad, shift=shift, groups_pad=pad % 3)


@pytest.mark.parametrize("strides", [(161, 1), (1, 70), (320, 2)])
def test_outputs_and_rows_of_x_apart(strides):
    _gemm(65, 150, 3616, 32, MANY, y_strides=strides, x_rs=3624)
    _gemm(65, 150, 3616, 32, MANY, y_strides=strides, x_rs=3617, out=U.F32)


@pytest.mark.parametrize("m,n,k,tile", [
    (2, 60, 60000, FEW), (3, 60, 20000, MANY), (3, 60, 19000, FEW),        # a pass's activations
    (8, 70, 7168, FEW), (8, 70, 7200, MANY), (16, 70, 3584, FEW), (16, 70, 3600, MANY), (17, 70, 3584, FEW),
    (1024, 512, 1024, FEW), (1025, 512, 1024, MANY), (5000, 100, 1000, FEW), (6000, 100, 1000, MANY)])
def test_where_the_kernels_meet(m, n, k, tile):
    _gemm(m, n, k, 64, tile)
    _gemm(m, n, k, 160, tile, elem=U.F16, out=U.F32)


# ------------------------------------------------------------------ experts


def _tokens(t, d, k, elem, seed):
    g = generator(seed)
    x = torch.randn(t, d, generator=g, device="cuda").to(TORCH[elem])
    return x, torch.softmax(torch.randn(t, k, generator=g, device="cuda"), 1), g


def _layer(x, ids, weights, experts, f, group, tile, elem=U.BF16, out=None, **more):
    out = elem if out is None else out
    t, d = x.shape
    k = ids.shape[1]
    up = Weights(experts * 2 * f, d, group, seed=d + 1, **more)
    down = Weights(experts * d, f, group, seed=d + 2, **more)
    y = torch.full((t, d), 7.0, device="cuda", dtype=TORCH[out])
    route = U.Route()
    U.expert_q4_ffn(elem, out, experts, x, (t, d), ids, (t, k), weights, (t, k), up.q, down.q, y, (t, d), route=route)
    assert route.tile_m == tile
    want, bound = ffn_reference(x.double(), ids, weights, up.value, down.value, experts, elem, out)
    assert_within(y, want, bound, f"{t} {experts} {d} {f}")
    again = torch.full_like(y, 3.0)
    U.expert_q4_ffn(elem, out, experts, x, (t, d), ids, (t, k), weights, (t, k), up.q, down.q, again, (t, d))
    assert torch.equal(y, again)


def _choose(g, t, experts, k, skew):
    """k different experts a token, the first ones `skew` times as likely by a step of e-folds."""
    lean = -skew * torch.arange(experts, device="cuda") / max(experts - 1, 1)
    noise = -torch.log(-torch.log(torch.rand(t, experts, generator=g, device="cuda").clamp(1e-6, 1 - 1e-6)))
    return (noise + lean).argsort(1, descending=True)[:, :k].to(torch.int32).contiguous()


@pytest.mark.parametrize("t,k,experts,d,f", [(1100, 1, 4, 64, 64), (600, 2, 64, 192, 600), (300, 4, 40, 200, 96),
                                             (2000, 6, 100, 72, 130), (515, 2, 2, 130, 33), (1030, 1, 1, 96, 257)])
@pytest.mark.parametrize("skew", [0, 4, 12])
def test_sorted_experts(t, k, experts, d, f, skew):
    """Experts with none, a few and most of the pairs, several tiles to a processor pair."""
    x, w, g = _tokens(t, d, k, U.BF16, t + skew)
    _layer(x, _choose(g, t, experts, k, skew), w, experts, f, 32, MANY)


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("scale_type", [U.F32, U.BF16, U.F16])
@pytest.mark.parametrize("group", [32, 64, 128, 160])
def test_sorted_experts_types(elem, scale_type, group):
    x, w, g = _tokens(530, 320, 2, elem, group)
    for out in (elem, U.F32):
        _layer(x, _choose(g, 530, 6, 2, 1), w, 6, 192, group, MANY, elem, out, scale_type=scale_type, zeros=group != 64)


def test_sorted_experts_dropped_twice_and_apart():
    x, w, g = _tokens(700, 161, 3, U.BF16, 5)
    ids = _choose(g, 700, 9, 3, 2)
    ids[:, 2] = ids[:, 0]
    ids[::3, 1] = -1
    ids[5] = 1 << 30
    w[5] = float("nan")
    clean = w.clone()
    clean[5] = 0
    _layer(x, ids, clean, 9, 77, 32, MANY, pad=3, shift=1)
    ids[:] = -1
    _layer(x, ids, clean, 9, 77, 32, MANY)


@pytest.mark.parametrize("t", [17, 40, 100, 250])
@pytest.mark.parametrize("skew", [0, 6])
def test_few_columns_of_experts_shared(t, skew):
    """Experts' columns over several blocks, more than the blocks that share them in the largest."""
    x, w, g = _tokens(t, 264, 4, U.BF16, t)
    _layer(x, _choose(g, t, 12, 4, skew), w, 12, 136, 64, FEW)
    x, w, g = _tokens(t, 131, 4, U.F16, t)
    _layer(x, _choose(g, t, 12, 4, skew), w, 12, 70, 96, FEW, U.F16, U.F32, pad=1)


@pytest.mark.parametrize("t,tile", [(32, FEW), (33, MANY), (64, MANY)])
def test_large_experts(t, tile):
    """Where the weights are the work: few pairs an expert, and more."""
    x, w, g = _tokens(t, 1024, 2, U.BF16, t)
    _layer(x, _choose(g, t, 16, 2, 0), w, 16, 2560, 128, tile)
