"""The 4-bit family's and the router's refusals, all from the host before any device work."""
import ctypes

import numpy as np

import uor_b200 as U


def _status(fn, *args, **kw):
    try:
        fn(*args, **kw)
    except U.UorError as e:
        return e.status
    return U.OK


def _q4(n=3, k=70, group=32, codes=None, scales=None, zeros=None, scale_type=U.F32, **more):
    codes = np.zeros(n * 35, np.uint8) if codes is None else codes
    scales = np.ones(n * 3, np.float32) if scales is None else scales
    return U.Q4(codes, scales, scale_type, n, k, group, zeros=zeros, **more)


def test_q4_gemm_refuses():
    a, c = np.zeros(2 * 70, np.float16), np.zeros(2 * 3, np.float16)
    av, cv = (2, 70), (2, 3)
    g = U.q4_gemm
    assert _status(g, U.F32, U.F32, a, av, _q4(), c, cv) == U.UNSUPPORTED
    assert _status(g, U.F16, U.BF16, a, av, _q4(), c, cv) == U.UNSUPPORTED
    assert _status(g, U.F16, U.F16, a, av, _q4(scale_type=U.I8), c, cv) == U.UNSUPPORTED
    for group in (0, 1, 16, 33, 48):
        assert _status(g, U.F16, U.F16, a, av, _q4(group=group, groups_rs=3), c, cv) == U.INVALID_ARGUMENT
    assert _status(g, U.F16, U.F16, a, (2, 69), _q4(), c, cv) == U.NONCONFORMANT
    assert _status(g, U.F16, U.F16, a, av, _q4(), c, (2, 2)) == U.NONCONFORMANT
    assert _status(g, U.F16, U.F16, a, av, _q4(), c, (2, 3, 0, 1)) == U.OUTPUT_ALIASES
    assert _status(g, U.F16, U.F16, a[:-1], av, _q4(), c, cv) == U.DOES_NOT_FIT
    assert _status(g, U.F16, U.F16, a, av, _q4(), c[:-1], cv) == U.DOES_NOT_FIT
    assert _status(g, U.F16, U.F16, a, av, _q4(codes=np.zeros(104, np.uint8)), c, cv) == U.DOES_NOT_FIT
    assert _status(g, U.F16, U.F16, a, av, _q4(scales=np.ones(8, np.float32)), c, cv) == U.DOES_NOT_FIT
    assert _status(g, U.F16, U.F16, a, av, _q4(zeros=np.ones(8, np.uint8)), c, cv) == U.DOES_NOT_FIT
    assert _status(g, U.F16, U.F16, a, av, _q4(row_bytes=2**63), c, cv) == U.DOES_NOT_FIT
    assert _status(g, U.F16, U.F16, a, (0, 70), _q4(), c, (0, 3)) == U.OK
    # encodings other than round to nearest, and a null descriptor, straight at the C entry
    A, C, w = U.view(a, *av), U.view(c, *cv), _q4()
    for encode, status in ((U.WRAPPING, U.UNSUPPORTED), (9, U.INVALID_ARGUMENT)):
        call = U.make_call(encode)
        assert U.lib().uor_b200_q4_gemm(U.F16, U.F16, ctypes.byref(A), ctypes.byref(w), ctypes.byref(C),
                                        ctypes.byref(call)) == status
    assert U.lib().uor_b200_q4_gemm(U.F16, U.F16, ctypes.byref(A), None, ctypes.byref(C), None) == U.INVALID_ARGUMENT


def test_other_families_refuse_16_bit_floats():
    a = np.zeros(4, np.uint16)
    v = U.view(a, 2, 2)
    call = U.make_call()
    for t in (U.BF16, U.F16):
        for fn in (U.lib().uor_b200_gemm, U.lib().uor_b200_gemm_float, U.lib().uor_b200_gemm_complex):
            for pair in ((t, t), (U.I8, t), (U.F32, t), (t, U.F32), (t, U.I32)):
                assert fn(*pair, ctypes.byref(v), ctypes.byref(v), ctypes.byref(v), 1, 0, ctypes.byref(call)) == U.UNSUPPORTED


def _route(router, e=8, k=2, t=3, elem=U.F32, lv=None, iv=None, wv=None, bias=None, short=0):
    logits, ids, w = np.zeros(t * e, np.float32), np.zeros(t * k, np.int32), np.zeros(t * k - short, np.float32)
    return _status(U.expert_route, elem, router, logits, lv or (t, e), bias, ids, iv or (t, k), w, wv or (t, k))


def test_expert_route_refuses():
    R = U.Router
    for bad in (R(0, 2), R(8, 0), R(8, 2, score=2), R(8, 2, groups=3, top_groups=1), R(8, 2, groups=0), R(8, 2, top_groups=0),
                R(8, 2, groups=2, top_groups=3), R(8, 5, groups=2, top_groups=1), R(8, 9)):
        assert _route(bad) == U.INVALID_ARGUMENT
    for big in (R(1025, 2), R(64, 33), R(66, 1, groups=33, top_groups=1)):
        assert _route(big) == U.UNSUPPORTED
    good = R(8, 2)
    assert _route(good, elem=U.I8) == U.UNSUPPORTED
    assert _route(good, e=7) == U.NONCONFORMANT
    assert _route(good, iv=(3, 1)) == U.NONCONFORMANT
    assert _route(good, wv=(2, 2)) == U.NONCONFORMANT
    assert _route(good, iv=(3, 2, 0, 1)) == U.OUTPUT_ALIASES
    assert _route(good, lv=(3, 8, 9, 1)) == U.DOES_NOT_FIT
    assert _route(good, short=1) == U.DOES_NOT_FIT
    assert _route(good, bias=np.zeros(7, np.float32)) == U.DOES_NOT_FIT
    assert _route(good, lv=(0, 8), iv=(0, 2), wv=(0, 2)) == U.OK


def test_expert_route_backward_refuses():
    t, e, k = 3, 8, 2
    good = U.Router(e, k)
    x, ids, g = np.zeros(t * e, np.float32), np.zeros(t * k, np.int32), np.zeros(t * k, np.float32)
    d = np.zeros(t * e, np.float32)
    b = U.expert_route_backward
    assert _status(b, U.F64, good, x, (t, e), ids, (t, k), g, (t, k), d, (t, e)) == U.UNSUPPORTED
    assert _status(b, U.F32, U.Router(8, 9), x, (t, e), ids, (t, k), g, (t, k), d, (t, e)) == U.INVALID_ARGUMENT
    assert _status(b, U.F32, good, x, (t, e), ids, (t, k), g, (2, k), d, (t, e)) == U.NONCONFORMANT
    assert _status(b, U.F32, good, x, (t, e), ids, (t, k), g, (t, k), d, (t, 7)) == U.NONCONFORMANT
    assert _status(b, U.F32, good, x, (t, e), ids, (t, k), g, (t, k), d, (t, e, 0, 1)) == U.OUTPUT_ALIASES
    assert _status(b, U.F32, good, x, (t, e), ids, (t, k), g, (t, k), d[:-1], (t, e)) == U.DOES_NOT_FIT
    assert _status(b, U.F32, good, x, (0, e), ids, (0, k), g, (0, k), d, (0, e)) == U.OK


def test_expert_q4_ffn_refuses():
    t, k, experts, d, f = 3, 2, 4, 64, 32
    x, ids, w = np.zeros(t * d, np.float16), np.zeros(t * k, np.int32), np.zeros(t * k, np.float32)
    y = np.zeros(t * d, np.float16)
    up = U.Q4(np.zeros(experts * 2 * f * d // 2, np.uint8), np.ones(experts * 2 * f * 2, np.float32), U.F32, experts * 2 * f, d, 32)
    down = U.Q4(np.zeros(experts * d * f // 2, np.uint8), np.ones(experts * d, np.float32), U.F32, experts * d, f, 32)

    def run(elem=U.F16, out=U.F16, experts=experts, xv=(t, d), iv=(t, k), wv=(t, k), up=up, down=down, yv=(t, d), x=x):
        return _status(U.expert_q4_ffn, elem, out, experts, x, xv, ids, iv, w, wv, up, down, y, yv)

    assert run(elem=U.F32) == U.UNSUPPORTED
    assert run(out=U.BF16) == U.UNSUPPORTED
    assert run(experts=0) == U.INVALID_ARGUMENT
    assert run(experts=3) == U.NONCONFORMANT
    assert run(xv=(t, 32)) == U.NONCONFORMANT
    assert run(iv=(t, 1)) == U.NONCONFORMANT
    assert run(wv=(2, k)) == U.NONCONFORMANT
    assert run(up=down) == U.NONCONFORMANT
    assert run(down=up) == U.NONCONFORMANT
    assert run(yv=(2, d)) == U.NONCONFORMANT
    assert run(yv=(t, d, 0, 1)) == U.OUTPUT_ALIASES
    assert run(x=x[:-1]) == U.DOES_NOT_FIT
    bad = U.Q4(down.arrays[0], down.arrays[1], U.F32, experts * d, f, 40)
    assert run(down=bad) == U.INVALID_ARGUMENT
    assert run(xv=(0, d), iv=(0, k), wv=(0, k), yv=(0, d)) == U.OK
