"""What the entries of the 4-bit cache and the product with an epilogue refuse on the host. No device is
needed, and none is touched: every call here is refused or has nothing to do."""
import ctypes

import numpy as np
import pytest

import uor_b200 as U

BASE = 1 << 20  # addresses that nothing reads
R, H, D, PAGE, SEQS, COLS = 6, 2, 64, 16, 3, 4


def _view(rows, cols, at=0, rs=None, cs=1, length=None):
    return U.View(BASE + at, rows * (rs or cols) if length is None else length, rows, cols, cols if rs is None else rs, cs)


def _raw(cls, *values):
    c = cls.__new__(cls)
    ctypes.Structure.__init__(c, *values)
    return c


def _cache(pool=BASE, pages=8, page=PAGE, heads=H, dim=D, group=32, elem=U.BF16, size=None):
    if size is None:
        size = pages * U.kv4_page_bytes(page, heads, dim, group, elem)
    return _raw(U.KV4, pool, size, pages, page, heads, dim, group, elem)


def _batch(seqs=SEQS, starts=BASE, starts_len=None, lengths=BASE, lengths_len=None, table=BASE, table_len=None, cols=COLS, rs=None):
    rs = cols if rs is None else rs
    return _raw(U.Batch, seqs, starts, seqs + 1 if starts_len is None else starts_len, lengths,
                seqs if lengths_len is None else lengths_len, table, seqs * rs if table_len is None else table_len, cols, rs)


def _turn(cos=BASE, sin=BASE, n=None, positions=COLS * PAGE, rs=None, dims=D, interleaved=0):
    rs = dims // 2 if rs is None else rs
    return _raw(U.Rotation, cos, sin, positions * rs if n is None else n, positions, rs, dims, interleaved)


DEVICE = lambda: U.make_call(U.NEAREST, device=True)  # noqa: E731


def _append(elem=U.BF16, cache=None, batch=None, k=None, v=None, q=None, q_out=None, turn=None, call=None):
    view = lambda x: _view(R, H * D) if x is None else x  # noqa: E731
    return U.lib().uor_b200_kv4_append(elem, _cache() if cache is None else cache, _batch() if batch is None else batch, view(k),
                                       view(v), q, q_out, turn, DEVICE() if call is None else call)


def _read(out=U.F32, cache=None, batch=None, k=None, v=None, call=None):
    view = lambda x: _view(R, H * D) if x is None else x  # noqa: E731
    return U.lib().uor_b200_kv4_read(out, _cache() if cache is None else cache, _batch() if batch is None else batch, view(k),
                                     view(v), DEVICE() if call is None else call)


def _attend(elem=U.BF16, out=U.BF16, cache=None, batch=None, q=None, y=None, lse=None, scale=0.125, call=None):
    view = lambda x: _view(R, 2 * H * D) if x is None else x  # noqa: E731
    return U.lib().uor_b200_kv4_attention(elem, out, _cache() if cache is None else cache, _batch() if batch is None else batch,
                                          view(q), scale, 0, 0, view(y), lse, DEVICE() if call is None else call)


ALL = [_append, _read, _attend]


@pytest.mark.parametrize("page,heads,dim,group,elem,size", [
    (16, 1, 64, 32, U.BF16, 16 * 64 + 128 * 2), (64, 8, 128, 32, U.BF16, 4 * 8 * (16 * 128 + 128 * 4)),
    (32, 3, 96, 32, U.F16, 2 * 3 * (16 * 96 + 128 * 3)), (16, 1, 256, 256, U.F16, 16 * 256 + 128), (4096, 1024, 192, 64, U.F16, 256 * 1024 * (16 * 192 + 128 * 3)),
    (8, 1, 64, 32, U.BF16, 0), (48, 1, 64, 32, U.BF16, 0), (8192, 1, 64, 32, U.BF16, 0), (16, 0, 64, 32, U.BF16, 0), (16, 1025, 64, 32, U.BF16, 0),
    (16, 1, 80, 16, U.BF16, 0), (16, 1, 64, 128, U.BF16, 0), (16, 1, 96, 96, U.BF16, 0), (16, 1, 64, 16, U.BF16, 0), (16, 1, 64, 0, U.BF16, 0),
    (16, 1, 64, 32, U.F32, 0)])
def test_page_bytes(page, heads, dim, group, elem, size):
    assert U.kv4_page_bytes(page, heads, dim, group, elem) == size
    if not size:
        for fn in ALL:
            assert fn(cache=_cache(page=page, heads=heads, dim=dim, group=group, elem=elem, size=1 << 30)) == U.UNSUPPORTED


@pytest.mark.parametrize("fn", ALL)
def test_caches_and_batches_refused(fn):
    assert fn(cache=ctypes.POINTER(U.KV4)()) == U.INVALID_ARGUMENT
    assert fn(batch=ctypes.POINTER(U.Batch)()) == U.INVALID_ARGUMENT
    whole = 8 * U.kv4_page_bytes(PAGE, H, D, 32, U.BF16)
    assert fn(cache=_cache(size=whole - 1)) == U.DOES_NOT_FIT
    assert fn(cache=_cache(pages=1 << 40, size=1 << 62)) == U.UNSUPPORTED
    assert fn(cache=_cache(pages=(1 << 31) - 1, size=whole)) == U.DOES_NOT_FIT
    assert fn(cache=_cache(pool=None)) == U.INVALID_ARGUMENT
    assert fn(cache=_cache(pool=BASE + 8)) == U.INVALID_ARGUMENT
    assert fn(batch=_batch(starts_len=SEQS)) == U.DOES_NOT_FIT
    assert fn(batch=_batch(lengths_len=SEQS - 1)) == U.DOES_NOT_FIT
    assert fn(batch=_batch(table_len=SEQS * COLS - 1)) == U.DOES_NOT_FIT
    assert fn(batch=_batch(rs=COLS + 1, table_len=(SEQS - 1) * (COLS + 1) + COLS - 1)) == U.DOES_NOT_FIT
    assert fn(batch=_batch(seqs=4097)) == U.UNSUPPORTED
    assert fn(batch=_batch(cols=1 << 27, table_len=1 << 40)) == U.UNSUPPORTED
    assert fn(batch=_batch(cols=1 << 60, rs=1, table_len=1 << 62)) == U.UNSUPPORTED
    assert fn(batch=_batch(rs=1 << 60, table_len=(1 << 63) - 1)) == U.UNSUPPORTED
    for name in ("starts", "lengths", "table"):
        assert fn(batch=_batch(**{name: None})) == U.INVALID_ARGUMENT
        assert fn(batch=_batch(**{name: BASE + 2})) == U.INVALID_ARGUMENT


@pytest.mark.parametrize("fn", ALL)
def test_calls_refused(fn):
    assert fn(call=U.make_call(U.NEAREST, device=False)) == U.INVALID_ARGUMENT
    assert fn(call=ctypes.POINTER(U.Call)()) == U.INVALID_ARGUMENT
    assert fn(call=U.make_call(U.SATURATING, device=True)) == U.UNSUPPORTED
    assert fn(call=U.make_call(9, device=True)) == U.INVALID_ARGUMENT


def test_append_refused():
    none = ctypes.POINTER(U.View)()
    assert U.lib().uor_b200_kv4_append(U.BF16, _cache(), _batch(), none, _view(R, H * D), None, None, None, DEVICE()) == U.INVALID_ARGUMENT
    assert U.lib().uor_b200_kv4_append(U.BF16, _cache(), _batch(), _view(R, H * D), none, None, None, None, DEVICE()) == U.INVALID_ARGUMENT
    assert _append(elem=U.F32) == U.UNSUPPORTED
    assert _append(elem=U.F16) == U.UNSUPPORTED  # of a bfloat16 cache
    wide = _view(R, 2 * H * D)
    assert _append(q=wide) == U.INVALID_ARGUMENT
    assert _append(q_out=wide) == U.INVALID_ARGUMENT
    assert _append(k=_view(R, H * D + 1)) == U.NONCONFORMANT
    assert _append(v=_view(R + 1, H * D)) == U.NONCONFORMANT
    assert _append(q=_view(R, D + 1), q_out=_view(R, D + 1)) == U.NONCONFORMANT
    assert _append(q=_view(R, D), q_out=_view(R, 2 * D)) == U.NONCONFORMANT
    assert _append(k=_view(R, H * D, length=R * H * D - 1)) == U.DOES_NOT_FIT
    assert _append(k=_view(R, H * D, at=1)) == U.INVALID_ARGUMENT
    assert _append(v=_view(R, H * D, rs=1, cs=R, length=1 << 20)) == U.UNSUPPORTED
    assert _append(q=wide, q_out=_view(R, 2 * H * D, rs=2, length=1 << 20)) == U.OUTPUT_ALIASES
    assert _append(q=wide, q_out=_view(R, 2 * H * D, rs=2 * H * D + 8)) == U.INVALID_ARGUMENT  # from one address, by other strides


@pytest.mark.parametrize("turn,status", [
    (dict(dims=63), U.INVALID_ARGUMENT), (dict(dims=66), U.INVALID_ARGUMENT), (dict(interleaved=2), U.INVALID_ARGUMENT),
    (dict(positions=COLS * PAGE - 1), U.DOES_NOT_FIT), (dict(n=COLS * PAGE * D // 2 - 1), U.DOES_NOT_FIT),
    (dict(rs=1 << 62, n=1 << 63), U.DOES_NOT_FIT), (dict(cos=None), U.INVALID_ARGUMENT), (dict(sin=None), U.INVALID_ARGUMENT),
    (dict(cos=BASE + 2), U.INVALID_ARGUMENT), (dict(sin=BASE + 1), U.INVALID_ARGUMENT)])
def test_rotations_refused(turn, status):
    assert _append(turn=_turn(**turn)) == status


def test_read_refused():
    assert _read(out=U.F16) == U.UNSUPPORTED
    assert _read(out=U.I32) == U.UNSUPPORTED
    assert _read(k=_view(R, H * D - 1)) == U.NONCONFORMANT
    assert _read(v=_view(R - 1, H * D)) == U.NONCONFORMANT
    assert _read(k=_view(R, H * D, rs=1, length=1 << 20)) == U.OUTPUT_ALIASES
    assert _read(k=_view(R, H * D, at=2)) == U.INVALID_ARGUMENT


def test_attention_refused():
    assert _attend(elem=U.F32) == U.UNSUPPORTED
    assert _attend(out=U.F16) == U.UNSUPPORTED
    assert _attend(elem=U.F16, out=U.F16) == U.UNSUPPORTED
    assert _attend(q=_view(R, 0)) == U.NONCONFORMANT
    assert _attend(q=_view(R, 3 * D), y=_view(R, 3 * D)) == U.NONCONFORMANT  # heads that two do not share
    assert _attend(y=_view(R, H * D)) == U.NONCONFORMANT
    assert _attend(y=_view(R - 1, 2 * H * D)) == U.NONCONFORMANT
    assert _attend(lse=_view(R, H)) == U.NONCONFORMANT
    assert _attend(lse=_view(R, 2 * H, rs=0, length=1 << 20)) == U.OUTPUT_ALIASES
    assert _attend(lse=_view(R, 2 * H, at=2)) == U.INVALID_ARGUMENT
    assert _attend(q=_view(R, 2 * H * D, rs=1, cs=R, length=1 << 20)) == U.UNSUPPORTED
    for scale in (float("nan"), float("inf"), -float("inf")):
        assert _attend(scale=scale) == U.INVALID_ARGUMENT


def test_nothing_to_do():
    empty = _batch(seqs=0, starts=None, lengths=None, table=None)
    for fn in ALL:
        assert fn(batch=empty) == U.OK
    assert _append(k=_view(0, H * D), v=_view(0, H * D)) == U.OK
    assert _attend(q=_view(0, 2 * H * D), y=_view(0, 2 * H * D)) == U.OK


def test_binding_takes_no_host_arrays():
    ints, floats = np.zeros(8, np.int32), np.zeros(64, np.float32)
    with pytest.raises(U.UorError):
        U.KV4(np.zeros(64, np.uint8), 1, 16, 1, 64, 32, U.BF16)
    with pytest.raises(U.UorError):
        U.Batch(ints, ints, ints, 1, 1)
    with pytest.raises(U.UorError):
        U.Rotation(floats, floats, 1, 64)
    with pytest.raises(U.UorError):
        U.kv4_attention(U.F16, U.F16, _cache(elem=U.F16), _batch(), np.zeros((R, H * D), np.float16), (R, H * D),
                        np.zeros((R, H * D), np.float16), (R, H * D))


def test_linear_refused():
    m, n, k = 3, 32, 64
    q = _raw(U.Q4, BASE, n * k // 2, n, k, k // 2, BASE, n * 2, U.F32, 32, 2, None, 0)
    fn = U.lib().uor_b200_q4_linear

    def call(out=U.F32, bias=None, bias_len=n, bias_type=U.F32, act=U.IDENTITY, residual=None):
        return fn(U.BF16, out, _view(m, k), q, bias, bias_len, bias_type, act, residual, _view(m, n), DEVICE())

    assert call(act=5) == U.INVALID_ARGUMENT
    assert call(bias=BASE, bias_type=U.F16) == U.UNSUPPORTED
    assert call(bias=BASE, bias_type=U.I32) == U.UNSUPPORTED
    assert call(bias=BASE, bias_len=n - 1) == U.DOES_NOT_FIT
    assert call(bias=BASE + 2) == U.INVALID_ARGUMENT
    assert call(bias=BASE + 1, bias_type=U.BF16) == U.INVALID_ARGUMENT
    assert call(residual=_view(m, n - 1)) == U.NONCONFORMANT
    assert call(residual=_view(m + 1, n)) == U.NONCONFORMANT
    assert call(residual=_view(m, n, at=2)) == U.INVALID_ARGUMENT
    assert call(residual=_view(m, n, length=m * n - 1)) == U.DOES_NOT_FIT
    assert call(residual=_view(m, n, rs=n + 1, length=m * n + m)) == U.INVALID_ARGUMENT  # C's address, other strides
    assert fn(U.BF16, U.F32, _view(0, k), q, BASE, n, U.F32, U.RELU, _view(0, n), _view(0, n), DEVICE()) == U.OK


def test_linear_binding_refuses_other_types():
    a, w = np.zeros((2, 64), np.uint16), U.Q4(np.zeros(32 * 32, np.uint8), np.ones(64, np.float32), U.F32, 32, 64, 32)
    c = np.zeros((2, 32), np.float32)
    for bias in (np.zeros(32, np.float64), np.zeros(32, np.int64)):
        with pytest.raises(TypeError):
            U.q4_linear(U.BF16, U.F32, a, (2, 64), w, c, (2, 32), bias=bias)
    with pytest.raises(TypeError):
        U.q4_linear(U.BF16, U.F32, a, (2, 64), w, c, (2, 32), residual=np.zeros((2, 32), np.float64))
