"""The same bytes on every pass, the first one over weights that were just laid out among them: their
addresses are new to the device then, and loads that wait for them come late."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import assert_within, ffn_reference, generator
from test_expert_ffn_gpu import Layer

pytestmark = [pytest.mark.gpu, needs_gpu]


def _elsewhere(q, keep):
    """The descriptor's arrays copied to memory of their own, unlike any before."""
    torch.cuda.empty_cache()
    keep.append(torch.empty(1 << 22, dtype=torch.uint8, device="cuda"))
    codes, scales, zeros = (None if a is None else a.clone() for a in q.arrays)
    return U.Q4(codes, scales, q.scale_type, q.rows, q.cols, q.group, zeros=zeros)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_experts(zeros, group):
    """Experts with 60 to 250 of the pairs each: tiles of all widths, several to a processor pair."""
    t, k, experts, d, f = 1024, 4, 32, 1024, 512
    layer = Layer(experts, d, f, group, U.BF16, zeros, seed=3)
    g = generator(9)
    x = torch.randn(t, d, generator=g, device="cuda").bfloat16()
    score = torch.randn(t, experts, generator=g, device="cuda") - 1.5 * torch.arange(experts, device="cuda") / experts
    ids = score.argsort(1, descending=True)[:, :k].to(torch.int32).contiguous()
    w = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), 1)
    first, keep = None, []
    for _ in range(25):
        up, down = _elsewhere(layer.up.q, keep), _elsewhere(layer.down.q, keep)
        for _ in range(3):
            y = torch.full((t, d), 7.0, device="cuda")
            U.expert_q4_ffn(U.BF16, U.F32, experts, x, (t, d), ids, (t, k), w, (t, k), up, down, y, (t, d))
            if first is None:
                first = y
                want, bound = ffn_reference(x.double(), ids, w, layer.up.value, layer.down.value, experts, U.BF16, U.F32)
                assert_within(y, want, bound)
            assert torch.equal(y, first)


@pytest.mark.parametrize("m", [40, 100, 700])
def test_products(m):
    n, k = 4608, 3712
    g = generator(m)
    codes = torch.randint(0, 256, (n * k // 2,), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    q = U.Q4(codes, (torch.rand(n * k // 64, generator=g, device="cuda") + 0.5).bfloat16(), U.BF16, n, k, 64)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    first, keep = None, []
    for _ in range(25):
        there = _elsewhere(q, keep)
        for _ in range(3):
            y = torch.full((m, n), 7.0, device="cuda")
            U.q4_gemm(U.BF16, U.F32, x, (m, k), there, y, (m, n))
            first = y if first is None else first
            assert torch.equal(y, first)
