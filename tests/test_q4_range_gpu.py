"""Products with 4-bit weights over the whole range of their types: a result that f32 holds is
right also where the activations, before a group's scale, would add up past it."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import Weights, assert_within, dot_bound, ffn_reference, generator, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]
LOWEST = torch.finfo(torch.bfloat16).min if torch is not None else None


@pytest.mark.parametrize("m,tile", [(1, 16), (3, 16), (12, 16), (300, 256)])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("pad", [0, 1])
def test_activations_of_the_types_size(m, tile, group, pad):
    """A few activations of the type's lowest and highest values beside ordinary ones; weights below
    15 2^-9 keep every result within f32. Rows at odd addresses too."""
    n, k = 150, 3712
    w = Weights(n, k, group, seed=group, spread=2.0 ** -10, pad=pad)
    x = torch.randn(m, k, generator=generator(m), device="cuda").bfloat16()
    x[:, 7], x[:, 40], x[:, 41], x[:, 700], x[:, k - 1] = LOWEST, -LOWEST, -LOWEST, LOWEST, LOWEST
    y = torch.full((m, n), -7.0, device="cuda")
    route = U.Route()
    U.q4_gemm(U.BF16, U.F32, x, (m, k), w.q, y, (m, n), route=route)
    assert route.tile_m == tile
    want = x.double() @ w.value.T
    assert float(want.abs().max()) < 3e38
    off = dot_bound(x.double(), w.value, k)
    assert_within(y, want, off + round_bound(want.abs() + off, U.F32))


@pytest.mark.parametrize("t", [1, 6, 600])
def test_experts_of_small_scales(t):
    """Activations near 2^126 and scales near 2^-125, as if the layer before had kept its own."""
    experts, d, f, k = 4, 192, 96, 2
    up = Weights(experts * 2 * f, d, 32, seed=1, spread=2.0 ** -125)
    down = Weights(experts * d, f, 32, seed=2)
    g = generator(t)
    x = ((torch.rand(t, d, generator=g, device="cuda") - 0.5) * 2.0 ** 127).bfloat16()
    ids = torch.rand(t, experts, generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32).contiguous()
    w = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), 1)
    y = torch.full((t, d), 7.0, device="cuda")
    U.expert_q4_ffn(U.BF16, U.F32, experts, x, (t, d), ids, (t, k), w, (t, k), up.q, down.q, y, (t, d))
    want, bound = ffn_reference(x.double(), ids, w, up.value, down.value, experts, U.BF16, U.F32)
    assert bool(torch.isfinite(want).all())
    assert_within(y, want, bound)
