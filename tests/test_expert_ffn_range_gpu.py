"""Inner activations past float16's largest value: infinite in that type, as the layer's definition
rounds them to it, in their own token alone; bfloat16 holds them."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import TORCH, assert_within, ffn_reference
from test_expert_ffn_gpu import Layer, tokens

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("t", [1, 4, 30, 600])
def test_large_inner_activations(t):
    layer = Layer(5, 128, 96, 64)
    results = {}
    for elem in (U.F16, U.BF16):
        x, ids, w = tokens(t, 128, 5, 2, elem)
        clean = layer.run(x, ids, w, elem, U.F32)
        x[0] = (x[0] * 2048).to(TORCH[elem])  # inner activations some 2^22 times their size
        y = layer.run(x, ids, w, elem, U.F32)
        assert torch.equal(y[1:], clean[1:])
        results[elem] = y[0]
    assert not bool(torch.isfinite(results[U.F16]).any())
    want, bound = ffn_reference(x.double(), ids, w, layer.up.value, layer.down.value, 5, U.BF16, U.F32)
    assert_within(results[U.BF16], want[0], bound[0])
