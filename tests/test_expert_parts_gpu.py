"""Up to 4 tokens an inner activation is two 16-bit parts: what is lost of it is a rounding of the
second part, not of the first.

Activations are small integers and the up product's scales powers of two, so that its sums are
exact in f32 and the bound holds only the inner activation's own arithmetic (8 2^-23), its two
parts' rounding (unit^2, and half a unit of float16's denormals) and the down product's sums."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, UNIT, Weights, dot_bound, generator, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("f", [8, 12, 24])
@pytest.mark.parametrize("t", [1, 2, 3, 4])
def test_second_part(elem, f, t):
    experts, d, k = 3, 64, 2
    up = Weights(experts * 2 * f, d, 32, seed=f)
    up.q.arrays[1].fill_(2.0 ** -7)
    codes, _, zeros = up.q.arrays
    code = torch.stack((codes & 15, codes >> 4), 1).view(experts * 2 * f, d).double()
    up_value = (code - (zeros.view(-1, d // 32)[:, torch.arange(d, device="cuda") // 32] & 15).double()) * 2.0 ** -7
    down = Weights(experts * d, f, 32, seed=f + 1)
    g = generator(t + f)
    x = torch.randint(-2, 3, (t, d), generator=g, device="cuda").to(TORCH[elem])
    ids = torch.rand(t, experts, generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32).contiguous()
    w = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), 1)
    y = torch.full((t, d), 7.0, device="cuda")
    U.expert_q4_ffn(elem, U.F32, experts, x, (t, d), ids, (t, k), w, (t, k), up.q, down.q, y, (t, d))

    want, bound, once = (torch.zeros(t, d, dtype=torch.float64, device="cuda") for _ in range(3))
    size = torch.zeros_like(want)
    for i in range(t):
        for s in range(k):
            e, share = int(ids[i, s]), w[i, s].double()
            gate, rise = (x[i].double()[None] @ up_value[(2 * e + b) * f:(2 * e + b + 1) * f].T for b in range(2))
            h = gate / (1 + torch.exp(-gate)) * rise
            wd = down.value[e * d:(e + 1) * d]
            dh = h.abs() * (8 * 2.0 ** -23 + UNIT[elem] ** 2) + (2.0 ** -25 if elem == U.F16 else 0)
            want[i] += ((h @ wd.T) * share)[0]
            once[i] += ((h.to(TORCH[elem]).double() @ wd.T) * share)[0]
            bound[i] += ((dh @ wd.abs().T + dot_bound(h.abs() + dh, wd, f)) * share)[0]
            size[i] += ((h @ wd.T).abs() * share)[0]
    bound = bound + (k + 4) * 2.0 ** -23 * (size + bound)
    bound = bound + round_bound(want.abs() + bound, U.F32)
    assert bool(((y.double() - want).abs() <= bound).all())
    # the bound tells the two apart: one rounding of the inner activations is outside it
    assert bool(((once - want).abs() > bound).any())
