"""The example of a mixture-of-experts layer: its parts against 64 bits, its CUDA graph against the
eager calls, and its router's descent."""
import importlib.util
import pathlib

import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import assert_within, dot_bound, ffn_reference, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.fixture(scope="module")
def moe():
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "moe_layer.py"
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("rows,cols,group", [(5, 64, 32), (7, 200, 64), (3, 33, 32), (16, 97, 96)])
def test_quantized_weights(moe, rows, cols, group):
    """Half a step of 15 over the group's range, the zero point's own rounding included: one step."""
    w = torch.randn(rows, cols, device="cuda")
    q = moe.quantize(w, group)
    step = q.arrays[1].view(rows, -1).double()[:, torch.arange(cols, device="cuda") // group]
    assert bool(((moe.dequantize(q) - w.double()).abs() <= step * (1 + 2.0 ** -20)).all())


@pytest.mark.parametrize("t,d,f,experts,k", [(1, 128, 64, 4, 2), (5, 200, 96, 8, 2), (70, 256, 128, 16, 4)])
def test_layer_against_the_formula(moe, t, d, f, experts, k):
    layer = moe.MoELayer(d, f, experts, k, seed=3)
    x = torch.randn(t, d, device="cuda").bfloat16()
    torch.cuda.synchronize()
    with torch.cuda.stream(layer.stream):
        mixed = torch.empty_like(x)
        U.q4_gemm(U.BF16, U.BF16, x, (t, d), layer.mix, mixed, (t, d), ctx=layer.ctx, asynchronous=True)
        h = layer.mixed(x)
        logits, ids, weights = layer.route(h)
        y = layer.experts_out(h, ids, weights)
        whole = layer.forward(x)
        layer.done()
    torch.cuda.synchronize()
    w = moe.dequantize(layer.mix)
    want = x.double() @ w.T
    bound = dot_bound(x.double(), w, d)
    assert_within(mixed, want, bound + round_bound(want.abs() + bound, U.BF16), "mix")
    score = torch.softmax(logits.double(), 1)
    top = torch.topk(logits, k, 1).indices
    assert torch.equal(ids.long(), top)
    want = score.gather(1, top)
    want = want / want.sum(1, keepdim=True)
    assert float((weights.double() - want).abs().max()) <= 32 * 2.0 ** -23
    want, bound = ffn_reference(h.double(), ids, weights, moe.dequantize(layer.up), moe.dequantize(layer.down), experts,
                                U.BF16, U.BF16)
    assert_within(y, want, bound, "experts")
    assert torch.equal(whole, h + y)
    layer.close()


def test_graph_replays_the_layer(moe):
    layer = moe.MoELayer(160, 64, 8, 2, seed=4)
    decoder = moe.Decoder(layer)
    for seed in range(3):
        x = torch.randn(1, 160, device="cuda").bfloat16()
        torch.cuda.synchronize()
        got = decoder.step(x)
        with torch.cuda.stream(layer.stream):
            want = layer.forward(x)
            layer.done()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del decoder
    layer.close()


def test_example_runs_and_learns(moe):
    lines = []
    found = moe.run(64, 128, 64, 8, 2, steps=10, report=lines.append)
    assert len(lines) == 3
    assert found["losses"][-1] < found["losses"][0]
