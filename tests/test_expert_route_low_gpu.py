"""Sigmoid scores at the lower end of f32: 1 / (1 + exp(-l)) between 2^-128 and 2^-126.

There a score is a denormal f32: a unit of 2^-149 absolute beside the 128 units relative that the
other scores are held to."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from test_expert_route_gpu import SHARE, back, generator, route

pytestmark = [pytest.mark.gpu, needs_gpu]
BOUND = 2.0 ** -148  # two units of a denormal


def _band(t, e):
    """Rows of logits from -87.2 down to -88.7, apart by 1.5 / e, in random order."""
    order = torch.rand(t, e, generator=generator(e), device="cuda").argsort(1)
    return -87.2 - order.float() * (1.5 / e)


@pytest.mark.parametrize("e", [8, 40, 200])
def test_scores_and_choice(e):
    """The largest scores are chosen in order, and weights without renormalisation are the scores."""
    logits, k = _band(25, e), min(e, 32)
    ids, w = route(logits, U.Router(e, k, U.SIGMOID, renormalize=False))
    assert torch.equal(ids.long(), logits.sort(1, descending=True).indices[:, :k])
    want = torch.sigmoid(logits.double()).gather(1, ids.long())
    assert bool((w > 0).all())
    # exp's argument is rounded to f32 by the input alone: only exp, the sum and the division count
    assert bool(((w.double() - want).abs() <= SHARE * want + BOUND).all())


def test_gradient():
    e, k = 24, 3
    logits = _band(9, e)
    r = U.Router(e, k, U.SIGMOID, renormalize=False)
    ids = logits.sort(1).indices[:, :k].to(torch.int32).contiguous()
    dw = 1 + torch.rand(9, k, generator=generator(1), device="cuda")
    got = back(logits, r, ids, dw).double()
    s = torch.sigmoid(logits.double())
    want = torch.zeros_like(s).scatter_(1, ids.long(), dw.double()) * s * (1 - s)
    assert bool((got.gather(1, ids.long()) > 0).all())
    assert bool(((got - want).abs() <= 2 * SHARE * want + 4 * BOUND).all())
