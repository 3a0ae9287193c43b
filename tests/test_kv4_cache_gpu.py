"""Tokens into the 4-bit cache and back: the definition's values to the bit, whatever the layout of the
rows, the rotation, the pages' order and the memory that was there before."""
import math

import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from kv4_data import MOST, Cache, held, rotated
from q4_data import TORCH

pytestmark = [pytest.mark.gpu, needs_gpu]


def _tables(positions, dims, seed=0, base=10000.0):
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, dims, 2, device="cuda", dtype=torch.float64) / max(dims, 1))
    return torch.cos(angle).float(), torch.sin(angle).float()


def _positions(cache):
    return torch.cat([torch.arange(n - new, n, device="cuda") for n, new in zip(cache.lengths, cache.news)])


def _read(cache, out, batch=None, rows=None, fill=0.0):
    rows = cache.rows if rows is None else rows
    k, v = (torch.full((rows, cache.heads * cache.dim), fill, device="cuda", dtype=TORCH[out]) for _ in range(2))
    U.kv4_read(out, cache.kv, cache.batch if batch is None else batch, k, k.shape, v, v.shape)
    return k.view(rows, cache.heads, cache.dim), v.view(rows, cache.heads, cache.dim)


SHAPES = [
    # lengths, news, page, heads, dim, group, share, dims, interleaved, elem
    ([1], [1], 16, 1, 64, 32, 1, 64, False, U.BF16),
    ([4097], [1], 16, 8, 128, 32, 4, 128, False, U.BF16),
    ([17, 16, 33], [17, 1, 3], 16, 2, 96, 32, 3, 48, True, U.F16),
    ([100, 250, 31, 1], [37, 250, 5, 1], 32, 3, 128, 64, 2, 64, False, U.F16),
    ([70, 5], [70, 2], 64, 5, 256, 256, 1, 256, True, U.BF16),
    ([129, 300], [100, 40], 128, 1, 192, 64, 5, 190, False, U.BF16),  # 95 pairs: channels one by one
    ([50], [50], 16, 3, 96, 32, 1, 36, True, U.F16),
    ([40], [40], 16, 2, 64, 64, 2, 0, False, U.F16),
    ([2000, 1500], [2000, 700], 256, 4, 128, 128, 4, 128, False, U.BF16),
]


@pytest.mark.parametrize("lengths,news,page,heads,dim,group,share,dims,interleaved,elem", SHAPES)
@pytest.mark.parametrize("fused", [True, False])
def test_append_and_read(lengths, news, page, heads, dim, group, share, dims, interleaved, elem, fused):
    c = Cache(lengths, news, page, heads, dim, group, elem, pad=2, seed=dim + len(lengths))
    rows, live, wide = c.rows, sum(news), heads * dim
    if fused:  # queries, keys and values side by side, rows at multiples of 16 bytes
        x = c.normal(rows, (share + 2) * wide).to(c.kind)
        q, k, v = x, x.view(-1)[share * wide:], x.view(-1)[(share + 1) * wide:]
        rs = (share + 2) * wide
    else:  # rows at any address
        rs = share * wide + 3
        q, k, v = (c.normal(rows * rs + 1).to(c.kind)[1:] for _ in range(3))
    as_rows = lambda b, w: b.as_strided((rows, w), (rs, 1), b.storage_offset()).clone()  # noqa: E731
    q0, k0, v0 = as_rows(q, share * wide), as_rows(k, wide), as_rows(v, wide)
    q_out = torch.full((rows, share * wide), 7.0, device="cuda", dtype=c.kind)
    positions = c.cols * page
    turn = None
    at = _positions(c)
    cos, sin = _tables(positions, dims)
    if dims:
        turn = U.Rotation(cos, sin, positions, dims, interleaved)
    U.kv4_append(elem, c.kv, c.batch, k, (rows, wide, rs), v, (rows, wide, rs), q=q, qv=(rows, share * wide, rs), q_out=q_out,
                 ov=q_out.shape, rotation=turn)
    want_q = rotated(q0[:live].view(live, -1, dim), cos[at], sin[at], dims, interleaved)
    assert torch.equal(q_out[:live].view(live, -1, dim), want_q)
    assert bool((q_out[live:] == 7.0).all())  # rows behind the last sequence
    want_k = held(rotated(k0[:live].view(live, -1, dim), cos[at], sin[at], dims, interleaved), group)
    want_v = held(v0[:live].view(live, -1, dim), group)
    for out in (U.F32, elem):
        got_k, got_v = _read(c, out, fill=3.0)
        for got, want in ((got_k, want_k), (got_v, want_v)):
            assert torch.equal(got[:live], want.float().to(TORCH[out]))
            assert bool((got[live:] == 3.0).all())
    if fused:  # queries in place
        U.kv4_append(elem, c.kv, c.batch, k, (rows, wide, rs), v, (rows, wide, rs), q=q, qv=(rows, share * wide, rs), q_out=q,
                     ov=(rows, share * wide, rs), rotation=turn)
        assert torch.equal(x[:live, :share * wide].view(live, -1, dim), want_q)
        assert torch.equal(x[live:, :share * wide], q0[live:])
        assert torch.equal(x[:, share * wide:(share + 1) * wide], k0)


def test_other_tokens_stay():
    """A token's codes and scales are its own: tokens beside it, in its words and blocks, keep theirs."""
    c = Cache([40, 61], [1, 1], 16, 3, 128, 32, U.BF16, seed=5).fill()
    both = c.batch_of([40, 61])
    before = _read(c, U.F32, both, 101)
    wide = 3 * 128
    k, v = (c.normal(2, wide).bfloat16() for _ in range(2))
    U.kv4_append(U.BF16, c.kv, c.batch_of([1, 1], [24, 54]), k, (2, wide), v, (2, wide))  # positions 23 and 53
    after = _read(c, U.F32, both, 101)
    for was, now, x in zip(before, after, (k, v)):
        want = was.clone()
        want[[23, 40 + 53]] = held(x.view(2, 3, 128), 32).float()
        assert torch.equal(now, want)


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
def test_extremes(elem):
    """Groups of one value, of zeros, of the type's ends, of its least and of what is not finite."""
    kind, group = TORCH[elem], 32
    x = torch.randn(16, 64, device="cuda").to(kind)
    tiny = torch.finfo(kind).smallest_normal
    x[0] = 0.0
    x[1] = 3.25
    x[2, :32] = MOST[elem]
    x[2, 32:] = -MOST[elem]
    x[3, ::2], x[3, 1::2] = MOST[elem], -MOST[elem]
    x[4] = torch.linspace(-tiny, tiny, 64, device="cuda").to(kind)
    x[5] = tiny
    x[6, 5] = math.inf
    x[7, 7], x[7, 40] = -math.inf, math.inf
    x[8, ::3] = math.nan
    x[9] = math.nan
    x[10, 0] = MOST[elem]
    x[11] = torch.arange(64, device="cuda").to(kind) / 64 + 1000
    x[12] = -x[12].abs()
    c = Cache([16], [16], 16, 1, 64, group, elem)
    U.kv4_append(elem, c.kv, c.batch, x, x.shape, x.flip(0).contiguous(), x.shape)
    k, v = _read(c, U.F32)
    assert torch.equal(k, held(x.view(16, 1, 64), group).float())
    assert torch.equal(v, held(x.flip(0).view(16, 1, 64), group).float())
    assert bool(torch.isfinite(k).all())


def test_rotation_of_what_is_not_finite_and_of_large_values():
    """Queries turn as the formula has them, infinities and NaN included; tables need not be cosines."""
    rows, dim = 64, 64
    c = Cache([rows], [rows], 16, 1, dim, 32, U.BF16, seed=2)
    x = c.normal(rows, 3 * dim)
    x[::5] *= 1e38
    x[1::7, ::9] = math.inf
    x[2::11, ::13] = math.nan
    x = x.bfloat16()
    cos, sin = (torch.randn(c.cols * 16, dim // 2, device="cuda") * 2 for _ in range(2))
    cos[3], sin[4], cos[9], sin[9] = 0.0, 0.0, 1e-38, 1e-44
    out = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    flat = x.view(-1)
    U.kv4_append(U.BF16, c.kv, c.batch, flat[dim:], (rows, dim, 3 * dim), flat[2 * dim:], (rows, dim, 3 * dim), q=x,
                 qv=(rows, dim, 3 * dim), q_out=out, ov=(rows, dim), rotation=U.Rotation(cos, sin, c.cols * 16, dim))
    at = torch.arange(rows, device="cuda")
    want_q, want_k = (rotated(x[:, i * dim:(i + 1) * dim].view(rows, 1, dim), cos[at], sin[at], dim, False) for i in range(2))
    assert torch.equal(torch.isnan(out), torch.isnan(want_q[:, 0]))
    assert torch.equal(out.nan_to_num(0, 1, 2), want_q[:, 0].nan_to_num(0, 1, 2))
    assert torch.equal(_read(c, U.F32)[0], held(want_k, 32).float())


def test_values_near_a_half():
    """Rotated values and quotients that land beside, or on, where they round: many rows of a few values."""
    rows, dim = 4096, 128
    c = Cache([rows], [rows], 64, 2, dim, 32, U.BF16, seed=8)
    x = (torch.randint(-8, 9, (rows, 2 * dim), generator=c.g, device="cuda").float() / 4).bfloat16()
    cos = torch.randint(-4, 5, (rows, dim // 2), generator=c.g, device="cuda").float() / 256 + 0.5
    sin = torch.randint(-4, 5, (rows, dim // 2), generator=c.g, device="cuda").float() * 2.0 ** -9
    y = (torch.randint(0, 31, (rows, 2 * dim), generator=c.g, device="cuda").float() / 2).bfloat16()  # steps and halves
    U.kv4_append(U.BF16, c.kv, c.batch, x, x.shape, y, y.shape, rotation=U.Rotation(cos, sin, rows, dim))
    k, v = _read(c, U.F32)
    assert torch.equal(k, held(rotated(x.view(rows, 2, dim), cos, sin, dim, False), 32).float())
    assert torch.equal(v, held(y.view(rows, 2, dim), 32).float())


def test_places_that_do_not_exist():
    """Tokens below 0, past the table and on pages outside the pool are not appended, their rows left."""
    heads, dim, page = 2, 64, 16
    c = Cache([60, 20, 48], [4, 4, 4], page, heads, dim, 32, U.F16, pad=1, seed=3).fill()
    wide = heads * dim
    whole = c.batch_of([60, 20, 48])
    before = _read(c, U.F32, whole, 128)
    c.table[2, 2] = c.pages  # the page with positions 32 .. 47
    k, v, q = (c.normal(13, wide).half() for _ in range(3))
    out = torch.full((13, wide), 5.0, device="cuda", dtype=torch.float16)
    read = [torch.full((13, wide), 6.0, device="cuda", dtype=torch.float16) for _ in range(2)]
    # sequence 0 has its rows at 62 .. 65 of a table of 64 positions, 1 at -2 .. 1, 2 at 30 .. 33
    batch = c.batch_of([4, 4, 4], [66, 2, 34])
    U.kv4_append(U.F16, c.kv, batch, k, (13, wide), v, (13, wide), q=q, qv=(13, wide), q_out=out, ov=(13, wide))
    U.kv4_read(U.F16, c.kv, batch, read[0], (13, wide), read[1], (13, wide))
    there = torch.tensor([1, 1, 0, 0, 0, 0, 1, 1, 1, 1, 0, 0, 0], device="cuda").bool()
    assert torch.equal(out[there], q[there]) and bool((out[~there] == 5.0).all())
    for got, x in zip(read, (k, v)):
        assert torch.equal(got[there], held(x[there].view(-1, heads, dim), 32).float().half().view(-1, wide))
        assert bool((got[~there] == 6.0).all())
    c.table[2, 2] = -5
    U.kv4_append(U.F16, c.kv, batch, k, (13, wide), v, (13, wide))
    after = _read(c, U.F32, whole, 128)  # positions 62, 63 lie on the last page behind the 60 tokens
    for was, now, x in zip(before, after, (k, v)):
        want = was.clone()
        want[60:62] = held(x[6:8].view(2, heads, dim), 32).float()
        want[80 + 30:80 + 32] = held(x[8:10].view(2, heads, dim), 32).float()
        valid = torch.ones(128, dtype=torch.bool, device="cuda")
        valid[80 + 32:] = False  # on the page that is gone; left as they were
        assert torch.equal(now[valid], want[valid])
        assert bool((now[~valid] == 0.0).all())


@pytest.mark.parametrize("starts,lengths", [([0, 9, 4, 12], [12, 3, 9]), ([5, 0, 3, 40], [10, 3, 11]), ([-7, 2, 2, 10], [4, 0, 8]),
                                            ([3, 3, 3, 3], [5, 5, 5]), ([2 ** 31 - 1, -2 ** 31, 0, 3], [2 ** 31 - 1, -2 ** 31, 7])])
def test_starts_that_do_not_rise(starts, lengths):
    """Whatever the arrays hold, nothing outside the rows and pages is touched: every write lands within a
    sequence's own positions or nowhere."""
    wide = 64
    c = Cache([16, 16, 16], [1, 1, 1], 16, 1, 64, 32, U.BF16, seed=1).fill()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = U.Batch(ints(starts), ints(lengths), c.table, 3, c.cols)
    guard = torch.full((14, wide), 9.0, device="cuda", dtype=torch.bfloat16)
    rows = 10
    x = c.normal(rows, wide).bfloat16()
    U.kv4_append(U.BF16, c.kv, batch, x, (rows, wide), x, (rows, wide), q=x, qv=(rows, wide), q_out=guard[2:], ov=(rows, wide))
    U.kv4_read(U.BF16, c.kv, batch, guard[2:], (rows, wide), guard[2:].clone(), (rows, wide))
    assert bool((guard[:2] == 9.0).all()) and bool((guard[12:] == 9.0).all())


def test_many_sequences():
    """4096 sequences of a token each."""
    c = Cache([1 + i % 20 for i in range(4096)], [1] * 4096, 16, 1, 64, 64, U.F16, seed=4)
    x, y = (c.normal(4096, 64).half() for _ in range(2))
    U.kv4_append(U.F16, c.kv, c.batch, x, x.shape, y, y.shape)
    k, v = _read(c, U.F32)
    assert torch.equal(k[:, 0], held(x, 64).float()) and torch.equal(v[:, 0], held(y, 64).float())


def test_pool_past_4_gb():
    """Pages whose bytes lie past 2^32."""
    page, heads, dim, group = 4096, 8, 128, 32
    size = U.kv4_page_bytes(page, heads, dim, group, U.BF16)
    pages = (1 << 32) // size + 3
    pool = torch.zeros(pages * size, dtype=torch.uint8, device="cuda")
    kv = U.KV4(pool, pages, page, heads, dim, group, U.BF16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = U.Batch(ints([0, 5]), ints([2 * page]), ints([0, pages - 1]), 1, 2)
    x, y = (torch.randn(5, heads * dim, device="cuda").bfloat16() for _ in range(2))
    U.kv4_append(U.BF16, kv, batch, x, x.shape, y, y.shape)
    k, v = (torch.zeros(5, heads * dim, device="cuda") for _ in range(2))
    U.kv4_read(U.F32, kv, batch, k, k.shape, v, v.shape)
    assert torch.equal(k, held(x.view(5, heads, dim), group).float().view(5, -1))
    assert torch.equal(v, held(y.view(5, heads, dim), group).float().view(5, -1))
    # attention over the first page and this one: the keys of the last five positions alone are not zero
    q = torch.randn(1, heads * dim, device="cuda").bfloat16()
    out = torch.zeros(1, heads * dim, device="cuda")
    U.kv4_attention(U.BF16, U.F32, kv, U.Batch(ints([0, 1]), ints([2 * page]), ints([0, pages - 1]), 1, 2), q, q.shape, out, out.shape,
                    window=5)
    p = torch.softmax((q.double().view(heads, dim) * k.double().view(5, heads, dim)).sum(2) * dim ** -0.5, 0)
    want = (p[:, :, None] * v.double().view(5, heads, dim)).sum(0)
    assert float((out.double().view(heads, dim) - want).abs().max()) <= 2.0 ** -14 * float(v.abs().max())
