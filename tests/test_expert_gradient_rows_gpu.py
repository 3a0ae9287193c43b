"""Every element of the router's gradient is written: rows that end inside a lane's share of the
experts, contiguous and padded, in a buffer that held something else."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, UNIT, generator
from test_expert_route_gpu import SHARE, gradient, route, spread_logits

pytestmark = [pytest.mark.gpu, needs_gpu]


def _check(experts, stride, elem, score, renormalize, shift=0, t=37, top_k=3):
    r = U.Router(experts, top_k, score, renormalize=renormalize, scale=2.5)
    logits = spread_logits(t, experts, elem, experts)
    ids, _ = route(logits, r, elem=elem)
    dw = torch.randn(t, top_k, generator=generator(5), device="cuda")
    rows = torch.full((shift + t * stride,), 5.0, device="cuda", dtype=TORCH[elem])
    U.expert_route_backward(elem, r, logits, (t, experts), ids, (t, top_k), dw, (t, top_k), rows[shift:],
                            (t, experts, stride, 1))
    rows, before = rows[shift:].view(t, stride), rows[:shift]
    want, size = gradient(logits, r, ids, dw)
    bound = 2 * SHARE * size + (UNIT[elem] * want.abs() + (2.0 ** -25 if elem == U.F16 else 0)) * 1.01 + 1e-37
    assert bool(((rows[:, :experts].double() - want).abs() <= bound).all())
    assert bool((rows[:, experts:] == 5).all()) and bool((before == 5).all())


@pytest.mark.parametrize("experts", [66, 132, 140, 204, 244, 260, 264, 520, 1000])
@pytest.mark.parametrize("elem", [U.F32, U.BF16, U.F16])
@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
@pytest.mark.parametrize("renormalize", [False, True])
def test_rows_that_end_inside_a_lane(experts, elem, score, renormalize):
    _check(experts, experts, elem, score, renormalize)


@pytest.mark.parametrize("experts,stride,elem", [(66, 68, U.F32), (101, 104, U.F32), (129, 160, U.F32), (250, 256, U.BF16),
                                                 (250, 256, U.F16), (513, 520, U.BF16), (1023, 1024, U.F16)])
@pytest.mark.parametrize("score", [U.SOFTMAX, U.SIGMOID])
@pytest.mark.parametrize("renormalize", [False, True])
def test_padded_rows(experts, stride, elem, score, renormalize):
    """Gaps between the rows keep what they hold, also where rows begin off a vector."""
    _check(experts, stride, elem, score, renormalize)
    _check(experts, stride, elem, score, renormalize, shift=1)
