"""The route that a call reports names the columns of the kernel that ran."""
import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from q4_data import Weights

pytestmark = [pytest.mark.gpu, needs_gpu]


@pytest.mark.parametrize("m,k,group,columns", [
    (1, 512, 64, 8), (8, 512, 64, 8), (9, 512, 64, 16),
    (1, 20480, 64, 8),                                   # one row whatever its length
    (4, 8192, 64, 8), (5, 8192, 64, 16),                 # 64 KB of activations for eight columns
    (1, 512, 96, 8), (8, 512, 96, 8), (3, 4096, 96, 16), (2, 4096, 96, 8), (9, 512, 96, 16)])  # 16 KB by way of rings
def test_columns_of_few_rows(m, k, group, columns):
    n = 40
    w = Weights(n, k, group)
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    y = torch.empty(m, n, device="cuda")
    route = U.Route()
    U.q4_gemm(U.BF16, U.F32, x, (m, k), w.q, y, (m, n), route=route)
    assert (route.tile_m, route.tile_n) == (16, columns)


@pytest.mark.parametrize("t,d,columns", [(1, 256, 8), (8, 256, 8), (9, 256, 16), (8, 5120, 16)])
def test_columns_of_experts(t, d, columns):
    """The up product's: 5120 positions of 8 tokens are more than eight columns have room for."""
    experts, f = 2, 32
    up, down = Weights(experts * 2 * f, d, 64), Weights(experts * d, f, 64)
    x = torch.zeros(t, d, device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(t, 1, device="cuda", dtype=torch.int32)
    w = torch.ones(t, 1, device="cuda")
    y = torch.empty(t, d, device="cuda")
    route = U.Route()
    U.expert_q4_ffn(U.BF16, U.F32, experts, x, (t, d), ids, (t, 1), w, (t, 1), up.q, down.q, y, (t, d), route=route)
    assert (route.tile_m, route.tile_n) == (16, columns)
