"""Attention over the 4-bit cache against 64 bits: lengths from none to thousands, heads that share keys,
windows and first tokens, drafts and prompts, batches with padded rows and pages that are not there."""
import math

import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from kv4_data import Cache, attention, held
from q4_data import TORCH, assert_within

pytestmark = [pytest.mark.gpu, needs_gpu]


def _run(c, q, share, out, scale=None, window=0, sinks=0, lse=True, batch=None, y=None, ctx=None):
    rows, wide = q.shape
    y = torch.full((rows, wide), 7.0, device="cuda", dtype=TORCH[out]) if y is None else y
    s = torch.full((rows, c.heads * share), 7.0, device="cuda") if lse else None
    route = U.Route()
    U.kv4_attention(c.elem, out, c.kv, c.batch if batch is None else batch, q, q.shape, y, y.shape, scale=scale, window=window,
                    sinks=sinks, lse=s, lv=(rows, c.heads * share), route=route, ctx=ctx)
    assert route.kernel == 10
    c.rounded = route.tile_m > 16  # many rows: keys, values and weights in 16 bits
    return y, s


def _check(c, q, share, out, got, window=0, sinks=0, scale=None, keys_of=None):
    y, s = got
    want, off, want_s, off_s = attention(c, q, share, c.dim ** -0.5 if scale is None else scale, out, window, sinks, c.rounded, keys_of)
    live = sum(c.news)
    assert_within(y[:live], want[:live], off[:live], "y")
    if s is not None:
        assert_within(s[:live], want_s[:live], off_s[:live], "lse")
        assert bool((s[live:] == 7.0).all())
    assert bool((y[live:] == 7.0).all()), "rows behind the last sequence"


CASES = [
    # lengths, news, page, heads, dim, group, share, elem, out, window, sinks
    ([1], [1], 16, 1, 64, 32, 1, U.BF16, U.BF16, 0, 0),
    ([16], [1], 16, 2, 128, 32, 4, U.BF16, U.F32, 0, 0),
    ([17, 1, 64, 65], [1, 1, 1, 1], 16, 3, 128, 128, 1, U.F16, U.F16, 0, 0),
    ([4096], [1], 16, 8, 128, 32, 4, U.BF16, U.BF16, 0, 0),
    ([700, 33, 5000, 1, 129], [1, 1, 1, 1, 1], 64, 2, 128, 64, 8, U.F16, U.F32, 0, 0),
    ([300, 31, 90], [5, 3, 1], 32, 2, 96, 32, 3, U.BF16, U.F32, 0, 0),
    ([1000, 40], [4, 4], 128, 1, 192, 64, 16, U.F16, U.F32, 0, 0),
    ([513, 2, 77], [2, 2, 2], 16, 2, 256, 32, 5, U.BF16, U.BF16, 0, 0),
    ([513, 2, 77], [1, 2, 1], 16, 2, 256, 256, 2, U.F16, U.F32, 0, 0),
    ([2000, 100, 9], [1, 3, 2], 16, 2, 64, 64, 3, U.F16, U.F32, 100, 4),
    ([2000, 100, 9], [1, 3, 2], 16, 2, 64, 64, 3, U.BF16, U.F32, 1, 0),
    ([700], [20], 16, 1, 128, 32, 2, U.F16, U.F32, 17, 33),
    ([500, 300], [1, 9], 32, 2, 128, 32, 1, U.BF16, U.F32, 64, 400),
    ([90, 200, 33], [90, 150, 1], 16, 2, 64, 32, 2, U.F16, U.F16, 0, 0),
    ([260], [260], 64, 2, 128, 32, 4, U.BF16, U.BF16, 0, 0),
    ([400, 37], [300, 37], 32, 1, 128, 64, 3, U.BF16, U.F32, 50, 8),
]


@pytest.mark.parametrize("lengths,news,page,heads,dim,group,share,elem,out,window,sinks", CASES)
def test_against_64_bits(lengths, news, page, heads, dim, group, share, elem, out, window, sinks):
    c = Cache(lengths, news, page, heads, dim, group, elem, pad=2, seed=len(CASES) + dim + share).fill(shift=0.3)
    q = c.queries(share)
    got = _run(c, q, share, out, window=window, sinks=sinks)
    _check(c, q, share, out, got, window, sinks)
    again = _run(c, q, share, out, window=window, sinks=sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # the same bytes


@pytest.mark.parametrize("new", [1, 200])
def test_rows_that_see_nothing(new):
    """Sequences without tokens, with fewer tokens than rows, without pages."""
    c = Cache([0, 50, 3, 20], [1, 1, 5, new if new > 1 else 20], 16, 2, 64, 32, U.BF16, pad=1, extra_pages=8)
    c.fill()
    q = c.queries(2)
    got = _run(c, q, 2, U.F32)
    y, s = got
    start = 0
    for n, length in zip(c.news, c.lengths):
        for i in range(n):
            if length - n + i < 0:
                assert bool((y[start + i] == 0.0).all()) and bool((s[start + i] == -math.inf).all())
        start += n
    _check(c, q, 2, U.F32, got)


def test_no_table():
    """A table without columns has no tokens: zeros."""
    c = Cache([16], [3], 16, 1, 64, 32, U.F16, pad=1).fill()
    c.cols = 0
    q = c.queries(1)
    y, s = _run(c, q, 1, U.F16, batch=c.batch_of([3]))
    assert bool((y[:3] == 0).all()) and bool((s[:3] == -math.inf).all()) and bool((y[3:] == 7).all())


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 20)])
@pytest.mark.parametrize("new", [2, 150])
def test_pages_that_are_not_there(new, window, sinks):
    c = Cache([200, 300], [new, 2], 32, 2, 64, 32, U.BF16, seed=6).fill()
    c.table[0, 1], c.table[0, 5], c.table[1, 0] = -1, c.pages, 2 ** 31 - 1
    there = [torch.ones(n, dtype=torch.bool, device="cuda") for n in c.lengths]
    there[0][32:64] = there[0][160:192] = there[1][:32] = False
    q = c.queries(3)
    got = _run(c, q, 3, U.F32, window=window, sinks=sinks)
    _check(c, q, 3, U.F32, got, window, sinks, keys_of=there)


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("new", [1, 130])
def test_what_lies_behind_the_last_token(elem, new):
    """Slots behind a sequence's last token hold anything: here scales and middles of NaN and infinity."""
    c = Cache([150, 165], [new, 1], 16, 2, 128, 32, elem, seed=7)
    bits = 0x7FC0 if elem == U.BF16 else 0x7E00
    c.pool.view(torch.int16).fill_(bits)
    c.fill()
    q = c.queries(2)
    got = _run(c, q, 2, U.F32)
    _check(c, q, 2, U.F32, got)


@pytest.mark.parametrize("new", [3, 140])
def test_queries_that_are_not_finite(new):
    """A row's NaN and infinities are its own."""
    c = Cache([180], [new], 16, 1, 64, 32, U.BF16, seed=9).fill()
    q = c.queries(2)
    q2 = q.clone()
    q2[1, 5], q2[2, 64 + 9] = math.nan, math.inf
    y, s = _run(c, q2, 2, U.F32)
    assert bool(torch.isnan(y[1, :64]).all()) and bool(torch.isnan(s[1, 0]))
    assert bool(torch.isnan(y[2, 64:]).any())
    want, off, _, _ = attention(c, q, 2, 64 ** -0.5, U.F32, rounded=c.rounded)
    y[1, :64], y[2, 64:] = want[1, :64].float(), want[2, 64:].float()
    assert_within(y, want, off + 2.0 ** -24 * want.abs(), "the others")


@pytest.mark.parametrize("new", [1, 160])
@pytest.mark.parametrize("scale", [0.0, -0.2, 30.0])
def test_scales(new, scale):
    """Even weights, the least score first, and one token that takes all."""
    c = Cache([333], [new], 32, 2, 64, 32, U.F16, seed=10).fill(size=0.2)
    q = c.queries(1, size=0.5)
    got = _run(c, q, 1, U.F32, scale=scale)
    _check(c, q, 1, U.F32, got, scale=scale)


@pytest.mark.parametrize("new", [1, 300])
def test_scores_that_rise_and_fall(new):
    """Keys whose scores climb by hundreds along the sequence: maxima move at every block."""
    c = Cache([600], [new], 16, 1, 64, 32, U.BF16, seed=11)
    ramp = torch.linspace(-4, 4, 600, device="cuda")[:, None].expand(600, 64)
    q = torch.ones(new, 128, device="cuda").bfloat16()
    q[:, 64:] = -1.0
    k, v = ramp.bfloat16().contiguous(), c.normal(600, 64).bfloat16()
    U.kv4_append(U.BF16, c.kv, c.batch_of([600]), k, k.shape, v, v.shape)
    c.k, c.v = [held(k.view(600, 1, 64), 32)], [held(v.view(600, 1, 64), 32)]
    got = _run(c, q, 2, U.F32, scale=1.0)
    _check(c, q, 2, U.F32, got, scale=1.0)


@pytest.mark.parametrize("elem,value_size", [(U.F16, 1e-6), (U.F16, 3000.0), (U.BF16, 1e30), (U.BF16, 1e-30)])
@pytest.mark.parametrize("new", [1, 150])
def test_values_of_any_size(elem, value_size, new):
    c = Cache([700], [new], 16, 1, 64, 32, elem, seed=12)
    k, v = c.normal(700, 64).to(c.kind), (c.normal(700, 64) * value_size).to(c.kind)
    U.kv4_append(elem, c.kv, c.batch_of([700]), k, k.shape, v, v.shape)
    c.k, c.v = [held(k.view(700, 1, 64), 32)], [held(v.view(700, 1, 64), 32)]
    q = c.queries(2)
    got = _run(c, q, 2, U.F32)
    _check(c, q, 2, U.F32, got)


@pytest.mark.parametrize("new", [2, 140])
def test_strided_rows(new):
    """Queries and outputs of rows at any address and distance; what lies between rows stays."""
    c = Cache([300, 150], [new, 1], 16, 2, 64, 32, U.F16, seed=13).fill()
    rows, wide, share = c.rows, 2 * 3 * 64, 3
    store = (c.normal(rows * (wide + 5) + 1) * 1.5).half()[1:]
    q = store.as_strided((rows, wide), (wide + 5, 1), 1).contiguous()
    out = torch.full((rows * (wide + 3) + 1,), 7.0, device="cuda", dtype=torch.float16)
    s = torch.full((rows * (6 + 2),), 7.0, device="cuda")
    route = U.Route()
    U.kv4_attention(U.F16, U.F16, c.kv, c.batch, store, (rows, wide, wide + 5), out[1:], (rows, wide, wide + 3), lse=s,
                    lv=(rows, 6, 8), route=route)
    c.rounded = route.tile_m > 16
    y = out[1:].as_strided((rows, wide), (wide + 3, 1), 1)
    _check(c, q, share, U.F16, (y, s.view(rows, 8)[:, :6]))
    assert bool((s.view(rows, 8)[:, 6:] == 7.0).all())
    gaps = out[1:1 + rows * (wide + 3)].view(rows, wide + 3)[:, wide:]
    assert bool((gaps == 7.0).all()) and float(out[0]) == 7.0


def test_long_and_short_together():
    """A long context among short ones: its share is cut over many blocks."""
    lengths = [20000, 5, 17, 1000]
    c = Cache(lengths, [1, 1, 1, 1], 64, 2, 128, 32, U.BF16, seed=14).fill()
    q = c.queries(4)
    _check(c, q, 4, U.F32, _run(c, q, 4, U.F32))


def test_many_sequences():
    c = Cache([1 + 37 * i % 100 for i in range(1500)], [1] * 1500, 16, 1, 64, 32, U.F16, seed=15).fill()
    q = c.queries(2)
    _check(c, q, 2, U.F16, _run(c, q, 2, U.F16))


@pytest.mark.parametrize("starts,lengths", [([0, 9, 4, 12], [12, 3, 9]), ([5, 0, 3, 40], [10, 3, 11]), ([-7, 2, 2, 10], [4, 0, 8]),
                                            ([2 ** 31 - 1, -2 ** 31, 0, 3], [2 ** 31 - 1, -2 ** 31, 7])])
def test_starts_that_do_not_rise(starts, lengths):
    """Whatever the arrays hold, nothing outside the rows is written."""
    c = Cache([16, 16, 16], [1, 1, 1], 16, 1, 64, 32, U.BF16, seed=1).fill()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = U.Batch(ints(starts), ints(lengths), c.table, 3, c.cols)
    q = c.normal(10, 64).bfloat16()
    guard = torch.full((14, 64), 9.0, device="cuda")
    U.kv4_attention(U.BF16, U.F32, c.kv, batch, q, q.shape, guard[2:12], (10, 64))
    assert bool((guard[:2] == 9.0).all()) and bool((guard[12:] == 9.0).all())


def test_pieces_join_by_their_lse():
    """A window's part and the rest, joined by their sums' logarithms, are the whole."""
    c = Cache([500], [1], 16, 2, 64, 32, U.BF16, seed=16).fill()
    q = c.queries(2)
    whole, s = _run(c, q, 2, U.F32)
    near, s1 = _run(c, q, 2, U.F32, window=180)
    far = c.batch_of([1], [320])  # as a row at position 319
    old, s2 = _run(c, q, 2, U.F32, batch=far)
    top = torch.maximum(s1, s2)
    w1, w2 = torch.exp(s1 - top), torch.exp(s2 - top)
    joined = (w1[..., None] * near.view(1, 4, 64) + w2[..., None] * old.view(1, 4, 64)) / (w1 + w2)[..., None]
    assert float((joined.view(1, -1) - whole).abs().max()) <= 2.0 ** -13 * float(whole.abs().max())
    assert float((top + torch.log(w1 + w2) - s).abs().max()) <= 2.0 ** -14
