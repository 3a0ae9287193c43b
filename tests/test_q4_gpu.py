"""Products with 4-bit weights and group scales against the formula in 64 bits."""
import numpy as np
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, Weights, assert_within, dot_bound, generator, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]


def _x(m, k, elem, seed, rs=None, cs=1):
    """A buffer and its m x k view's (rows, cols, rs, cs) and float64 values."""
    rs = k * cs if rs is None else rs
    span = (m - 1) * rs + (k - 1) * cs + 1 if m and k else 0
    buf = torch.randn(max(span, 1), generator=generator(seed), device="cuda").to(TORCH[elem])
    return buf, (m, k, rs, cs), buf.as_strided((m, k), (rs, cs)).double()


def _run(m, n, k, group, elem=U.BF16, out=None, x_strides=(None, 1), y_strides=None, **more):
    out = elem if out is None else out
    w = Weights(n, k, group, seed=n + k, **more)
    x, xv, x64 = _x(m, k, elem, m, *x_strides)
    rs, cs = (n, 1) if y_strides is None else y_strides
    y = torch.full(((m - 1) * rs + (n - 1) * cs + 1,), -7.0, device="cuda", dtype=TORCH[out])
    route = U.Route()
    U.q4_gemm(elem, out, x, xv, w.q, y, (m, n, rs, cs), route=route)
    assert route.kernel == 8
    want = x64 @ w.value.T
    off = dot_bound(x64, w.value, k)
    got = y.as_strided((m, n), (rs, cs))
    assert_within(got, want, off + round_bound(want.abs() + off, out), f"{m}x{n}x{k} g{group}")
    return y, got


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 130, 257, 300, 515])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_row_counts(m, group):
    """Every row count's tile, ending inside it too."""
    _run(m, 144, 512, group)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 127, 128, 129, 250, 1000])
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_widths(m, n):
    _run(m, n, 384, 64, elem=U.F16)


@pytest.mark.parametrize("k", [1, 2, 3, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 255, 257, 1000, 1001, 4104, 9000])
@pytest.mark.parametrize("m", [1, 4, 19, 150])
def test_reductions(m, k):
    """Reductions that end inside a byte, a vector, a group or a tile."""
    _run(m, 70, k, 32)
    _run(m, 70, k, 128, out=U.F32)


@pytest.mark.parametrize("group", [32, 64, 96, 128, 160, 192, 256, 384, 1024, 4096])
@pytest.mark.parametrize("m", [1, 12, 40, 160])
def test_groups(m, group):
    _run(m, 100, 1056, group, zeros=group % 64 == 0, out=U.F32)


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("scale_type", [U.F32, U.BF16, U.F16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m", [1, 24, 140])
def test_types(elem, scale_type, zeros, m):
    for out in (elem, U.F32):
        _run(m, 96, 320, 64, elem=elem, out=out, scale_type=scale_type, zeros=zeros)


@pytest.mark.parametrize("pad", [0, 1, 2, 4, 12, 16])
@pytest.mark.parametrize("shift", [0, 1, 4, 16])
@pytest.mark.parametrize("m", [1, 20, 133])
def test_codes_anywhere(pad, shift, m):
    """Rows of codes at any byte address and distance, scales with gaps between their rows."""
    _run(m, 130, 256, 32, pad=pad, shift=shift, groups_pad=pad % 3)
    _run(m, 50, 229, 64, pad=pad, shift=shift)


@pytest.mark.parametrize("strides", [(None, 1), (520, 1), (521, 1), (1, 300), (-512, 1), (1030, 2), (0, 1)])
@pytest.mark.parametrize("m", [1, 9, 140])
def test_activation_strides(strides, m):
    rs, cs = strides
    if rs is not None and rs < 0:
        k, n = 512, 40
        w = Weights(n, k, 64, seed=5)
        buf = torch.randn(m * k, generator=generator(3), device="cuda").to(torch.bfloat16)
        y = torch.empty(m * n, device="cuda", dtype=torch.float32)
        U.q4_gemm(U.BF16, U.F32, buf, (m, k, -k, 1), w.q, y, (m, n))
        x = buf.view(m, k).flip(0).double()
        want = x @ w.value.T
        assert_within(y.view(m, n), want, dot_bound(x, w.value, k) + round_bound(want.abs(), U.F32) * 2)
        return
    _run(m, 72, 256 if cs > 1 and rs == 1 else 512, 64, x_strides=(rs, cs))


@pytest.mark.parametrize("m", [1, 6, 70, 200])
def test_output_strides_and_gaps(m):
    """A padded output keeps what is between its rows; a transposed one is written as it lies."""
    n = 45
    y, _ = _run(m, n, 192, 32, out=U.F32, y_strides=(n + 3, 1))
    if m > 1:
        assert bool((y[: (m - 1) * (n + 3)].view(m - 1, n + 3)[:, n:] == -7).all())
    _run(m, n, 192, 32, y_strides=(1, m))


def test_shared_rows_of_codes():
    """A row stride of zero: every output has the same codes and scales."""
    k, n, m = 128, 33, 40
    one = Weights(1, k, 32, seed=9)
    q = U.Q4(one.q.arrays[0], one.q.arrays[1], U.F32, n, k, 32, zeros=one.q.arrays[2], row_bytes=0, groups_rs=0)
    x, xv, x64 = _x(m, k, U.BF16, 4)
    y = torch.empty(m, n, device="cuda")
    U.q4_gemm(U.BF16, U.F32, x, xv, q, y, (m, n))
    want = (x64 @ one.value.T).expand(m, n)
    assert_within(y, want, dot_bound(x64, one.value, k).expand(m, n) + round_bound(want, U.F32) * 2)


def test_empty_products():
    w = Weights(5, 64, 32)
    y = torch.full((4,), 3.0, device="cuda")
    U.q4_gemm(U.BF16, U.F32, torch.empty(0, device="cuda", dtype=torch.bfloat16), (0, 64), w.q, y, (0, 5))
    assert bool((y == 3).all())
    # no reduction: the empty sum
    empty = U.Q4(torch.empty(0, device="cuda", dtype=torch.uint8), torch.empty(0, device="cuda"), U.F32, 2, 0, 32)
    for m in (1, 2):
        y = torch.full((m * 2,), 3.0, device="cuda")
        U.q4_gemm(U.BF16, U.F32, torch.empty(0, device="cuda", dtype=torch.bfloat16), (m, 0), empty, y, (m, 2))
        assert bool((y == 0).all())


@pytest.mark.parametrize("m", [1, 8, 40, 200])
@pytest.mark.parametrize("k", [256, 300])
def test_not_finite(m, k):
    """Infinities and NaN spread to the cells that read them and to no other."""
    n, group = 140, 64
    w = Weights(n, k, group, seed=2)
    x, xv, _ = _x(m, k, U.BF16, 8)
    x2 = x.view(m, k)
    x2[0, 5] = float("inf")
    if m > 3:
        x2[3, k - 1] = float("nan")
        x2[2, 7] = -float("inf")
    scales = w.q.arrays[1]
    groups = -(-k // group)
    scales[9 * groups + 1] = float("inf")
    scales[17 * groups + groups - 1] = float("nan")
    y = torch.empty(m, n, device="cuda")
    U.q4_gemm(U.BF16, U.F32, x, xv, w.q, y, (m, n))
    code = torch.where(torch.isfinite(w.value), w.value, torch.ones_like(w.value))  # the clean columns
    clean_rows = torch.isfinite(x2).all(1)
    clean_cols = torch.ones(n, dtype=torch.bool, device="cuda")
    clean_cols[9] = clean_cols[17] = False
    x64 = torch.where(clean_rows[:, None], x2.double(), torch.zeros(1, device="cuda", dtype=torch.float64))
    want = x64 @ code.T
    at = clean_rows[:, None] & clean_cols[None, :]
    bound = dot_bound(x64, code, k) + round_bound(want.abs(), U.F32) * 2
    assert bool(((y.double() - want).abs() <= bound)[at].all())
    assert not bool(torch.isfinite(y[:, 17]).any())
    assert not bool(torch.isfinite(y[:, 9]).any())
    if m > 3:
        assert bool(torch.isnan(y[3]).all())
    zero = w.value[:, 5] == 0  # inf x 0 is NaN, inf x w the infinity of w's sign
    row = y[0]
    use = clean_cols & ~zero
    assert torch.equal(row[use], torch.sign(w.value[:, 5][use]).float() * float("inf"))
    assert bool(torch.isnan(row[zero]).all())


def test_same_bytes_every_time():
    for m in (1, 11, 100, 300):
        w = Weights(500, 2048, 128, seed=1)
        x, xv, _ = _x(m, 2048, U.BF16, 2)
        runs = []
        for _ in range(3):
            y = torch.empty(m, 500, device="cuda")
            U.q4_gemm(U.BF16, U.F32, x, xv, w.q, y, (m, 500))
            runs.append(y)
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_host_arrays():
    """Host buffers are staged: the same bytes as device ones."""
    m, n, k, group = 5, 37, 200, 32
    w = Weights(n, k, group, scale_type=U.F16, seed=6)
    x, xv, _ = _x(m, k, U.F16, 1)
    y = torch.empty(m * n, device="cuda", dtype=torch.float16)
    U.q4_gemm(U.F16, U.F16, x, xv, w.q, y, (m, n))
    hq = U.Q4(*(a.cpu().numpy() for a in w.q.arrays[:2]), U.F16, n, k, group, zeros=w.q.arrays[2].cpu().numpy())
    hy = np.full(m * n, 5, np.float16)
    U.q4_gemm(U.F16, U.F16, x.cpu().numpy(), xv, hq, hy, (m, n))
    assert np.array_equal(hy, y.cpu().numpy())


def test_on_a_stream_of_its_own():
    """Work queued on the context's stream is ordered with what fills its inputs there."""
    ctx = U.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    w = Weights(256, 1024, 128, seed=3)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        x = torch.zeros(4, 1024, device="cuda", dtype=torch.bfloat16)
        for _ in range(20):
            x.add_(0.125)
        y = torch.empty(4, 256, device="cuda")
        U.q4_gemm(U.BF16, U.F32, x, (4, 1024), w.q, y, (4, 256), ctx=ctx, asynchronous=True)
        twice = y * 2
    assert ctx.sync() == U.OK
    stream.synchronize()
    x64 = torch.full((4, 1024), 2.5, device="cuda", dtype=torch.float64)
    want = 2 * (x64 @ w.value.T)
    assert_within(twice, want, 2 * dot_bound(x64, w.value, 1024) + round_bound(want.abs(), U.F32) * 4)
    ctx.set_stream(None)
    ctx.close()
