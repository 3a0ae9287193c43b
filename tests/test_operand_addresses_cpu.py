"""A device pointer that is no multiple of its element's size is refused on the host: a kernel that
read through it would fault. No device is needed, and none is touched."""
import ctypes

import pytest

import uor_b200 as U

T, K, E, D, F = 3, 2, 4, 64, 32
BASE = 1 << 20  # addresses that nothing reads


def _view(rows, cols, at=0):
    return U.View(BASE + at, rows * cols, rows, cols, cols, 1)


def _q4(rows, cols, scales=0, scale_type=U.F32):
    q = U.Q4.__new__(U.Q4)
    ctypes.Structure.__init__(q, BASE, rows * cols // 2, rows, cols, cols // 2, BASE + scales, rows * cols // 32, scale_type, 32,
                              cols // 32, None, 0)
    return q


def _call():
    return U.make_call(U.NEAREST, device=True)


@pytest.mark.parametrize("at", [1, 3])
def test_q4_gemm(at):
    fn = U.lib().uor_b200_q4_gemm
    for elem, out, a, scales, scale_type, c in ((U.BF16, U.BF16, at, 0, U.F32, 0), (U.F16, U.F16, 0, 0, U.F32, at),
                                                (U.BF16, U.F32, 0, 0, U.F32, 2), (U.BF16, U.F32, 0, at, U.BF16, 0),
                                                (U.BF16, U.F32, 0, 2, U.F32, 0), (U.F16, U.F32, 0, at, U.F32, 0)):
        assert fn(elem, out, _view(T, D, a), _q4(F, D, scales, scale_type), _view(T, F, c), _call()) == U.INVALID_ARGUMENT


@pytest.mark.parametrize("at", [1, 2, 3])
def test_router(at):
    r = U.Router(E, K)
    forward, backward = U.lib().uor_b200_expert_route, U.lib().uor_b200_expert_route_backward
    none = ctypes.c_void_p(None)
    for logits, bias, ids, w in ((at, none, 0, 0), (0, BASE + at, 0, 0), (0, none, at, 0), (0, none, 0, at)):
        assert forward(U.F32, r, _view(T, E, logits), bias, E, _view(T, K, ids), _view(T, K, w), _call()) == U.INVALID_ARGUMENT
    for logits, ids, g, d in ((at, 0, 0, 0), (0, at, 0, 0), (0, 0, at, 0), (0, 0, 0, at)):
        assert backward(U.F32, r, _view(T, E, logits), _view(T, K, ids), _view(T, K, g), _view(T, E, d),
                        _call()) == U.INVALID_ARGUMENT
    assert forward(U.BF16, r, _view(T, E, 1), none, 0, _view(T, K), _view(T, K), _call()) == U.INVALID_ARGUMENT


@pytest.mark.parametrize("at", [1, 3])
def test_experts(at):
    fn = U.lib().uor_b200_expert_q4_ffn
    for x, ids, w, up, down, y in ((at, 0, 0, 0, 0, 0), (0, at, 0, 0, 0, 0), (0, 0, at, 0, 0, 0), (0, 0, 0, at, 0, 0),
                                   (0, 0, 0, 0, at, 0), (0, 0, 0, 0, 0, at), (0, 2, 0, 0, 0, 0), (0, 0, 0, 0, 2, 0)):
        assert fn(U.BF16, U.BF16, E, _view(T, D, x), _view(T, K, ids), _view(T, K, w), _q4(E * 2 * F, D, up), _q4(E * D, F, down),
                  _view(T, D, y), _call()) == U.INVALID_ARGUMENT


def test_empty_operands_have_no_address():
    assert U.lib().uor_b200_q4_gemm(U.BF16, U.F32, _view(0, D, 1), _q4(F, D), _view(0, F, 1), _call()) == U.OK
