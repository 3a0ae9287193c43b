"""The example's attention half: its graph's tokens are to the byte what eager calls give, and it runs for a
prompt and behind it at odd sizes."""
import importlib.util
import pathlib

import pytest

from gpu_util import needs_gpu, torch

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("tokens,d", [(1, 128), (37, 256), (300, 192)])
def test_prompt_then_tokens(tokens, d):
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "moe_layer.py"
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    moe = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(moe)
    layer = moe.MoELayer(d, 64, 8, 2)
    x = torch.randn(tokens, d, device="cuda").bfloat16()
    torch.cuda.synchronize()
    far, replayed, half = moe.run_attention(layer, x, report=lambda s: None)
    assert torch.isfinite(replayed.float()).all() and far == far
    assert int(half.length) == tokens
    last = replayed.shape[0]
    with torch.cuda.stream(layer.stream):
        half.length.fill_(tokens - last)
        one = half.batch(1)
        eager = torch.cat([layer.forward(half.forward(x[t:t + 1].clone(), one)) for t in range(tokens - last, tokens)])
        layer.done()
    assert torch.equal(eager, replayed)
    layer.close()
