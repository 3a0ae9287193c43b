"""The binding looks at the types of the 4-bit family's and the router's arrays: an array that is
not of its operand's type is refused before the library reads it."""
import numpy as np
import pytest

import uor_b200 as U

try:
    import torch
except Exception:  # pragma: no cover
    torch = None

needs_torch = pytest.mark.skipif(torch is None, reason="needs torch")
T, K, E, D, F = 3, 2, 4, 64, 32


def _ffn(elem=U.F16, out=U.F16, x=None, ids=None, w=None, y=None, codes=np.uint8, scales=np.float32, zeros=None):
    up = U.Q4(np.zeros(E * 2 * F * D // 2, codes), np.ones(E * 2 * F * 2, scales), U.F32, E * 2 * F, D, 32,
              zeros=None if zeros is None else np.zeros(E * 2 * F * 2, zeros))
    down = U.Q4(np.zeros(E * D * F // 2, np.uint8), np.ones(E * D, np.float32), U.F32, E * D, F, 32)
    U.expert_q4_ffn(elem, out, E, np.zeros(T * D, np.float16) if x is None else x, (T, D),
                    np.zeros(T * K, np.int32) if ids is None else ids, (T, K),
                    np.zeros(T * K, np.float32) if w is None else w, (T, K), up, down,
                    np.zeros(T * D, np.float16) if y is None else y, (T, D))


def test_experts_operands():
    for more in ({"ids": np.zeros(T * K, np.int64)}, {"ids": np.zeros(T * K, np.int16)}, {"ids": np.zeros(T * K, np.float32)},
                 {"x": np.zeros(T * D, np.float32)}, {"w": np.zeros(T * K, np.float64)}, {"w": np.zeros(T * K, np.float16)},
                 {"y": np.zeros(T * D, np.float32)}, {"out": U.F32}, {"elem": U.BF16, "out": U.BF16}, {"codes": np.int32},
                 {"scales": np.float64}, {"scales": np.float16}, {"zeros": np.float32}, {"ids": [0] * (T * K)}):
        with pytest.raises(TypeError):
            _ffn(**more)


def test_q4_operands():
    q = U.Q4(np.zeros(3 * 32, np.uint8), np.ones(3 * 2, np.float32), U.F32, 3, 64, 32)
    for elem, out, a, c in ((U.F16, U.F16, np.float32, np.float16), (U.F16, U.F32, np.float16, np.float16),
                            (U.F16, U.F16, np.float16, np.float64), (U.BF16, U.BF16, np.float16, np.uint16),
                            (U.BF16, U.F32, np.uint16, np.uint16), (U.F16, U.F16, np.int8, np.float16)):
        with pytest.raises(TypeError):
            U.q4_gemm(elem, out, np.zeros(2 * 64, a), (2, 64), q, np.zeros(2 * 3, c), (2, 3))


def test_router_operands():
    r = U.Router(E, K)

    def forward(elem=U.F32, logits=np.float32, bias=None, ids=np.int32, w=np.float32):
        U.expert_route(elem, r, np.zeros(T * E, logits), (T, E), None if bias is None else np.zeros(E, bias),
                       np.zeros(T * K, ids), (T, K), np.zeros(T * K, w), (T, K))

    def backward(elem=U.F32, logits=np.float32, ids=np.int32, g=np.float32, d=np.float32):
        U.expert_route_backward(elem, r, np.zeros(T * E, logits), (T, E), np.zeros(T * K, ids), (T, K),
                                np.zeros(T * K, g), (T, K), np.zeros(T * E, d), (T, E))

    for more in ({"logits": np.float16}, {"logits": np.float64}, {"elem": U.F16}, {"ids": np.int64}, {"ids": np.float32},
                 {"w": np.float64}, {"bias": np.float64}, {"bias": np.float16}, {"elem": U.BF16, "logits": np.float16}):
        with pytest.raises(TypeError):
            forward(**more)
    for more in ({"logits": np.float16}, {"ids": np.int64}, {"g": np.float64}, {"d": np.float16}, {"d": np.float64}):
        with pytest.raises(TypeError):
            backward(**more)


@needs_torch
def test_torch_operands():
    """torch's own defaults: topk's int64, bfloat16 beside float16."""
    ids = torch.zeros(T, K, dtype=torch.int64)
    with pytest.raises(TypeError):
        _ffn(ids=ids)
    with pytest.raises(TypeError):
        _ffn(x=torch.zeros(T, D, dtype=torch.bfloat16))
    r = U.Router(E, K)
    with pytest.raises(TypeError):
        U.expert_route(U.F32, r, torch.zeros(T, E, dtype=torch.bfloat16), (T, E), None, torch.zeros(T, K, dtype=torch.int32),
                       (T, K), torch.zeros(T, K), (T, K))


def test_what_is_taken():
    """16-bit floats' bits as integers, and types that the library itself refuses, pass the look."""
    none = (0, D)
    for elem, x, y in ((U.BF16, np.uint16, np.uint16), (U.BF16, np.int16, np.int16), (U.F16, np.float16, np.float16),
                       (U.F16, np.uint16, np.float16)):
        q = U.Q4(np.zeros(3 * 32, np.uint8), np.ones(3 * 2, np.float32), U.F32, 3, 64, 32)
        U.q4_gemm(elem, elem, np.zeros(0, x), none, q, np.zeros(0, y), (0, 3))
    U.Q4(np.zeros(96, np.int8), np.ones(6, np.uint16), U.BF16, 3, 64, 32, zeros=np.zeros(6, np.int8))
    with pytest.raises(U.UorError):
        _ffn(elem=U.F64)
