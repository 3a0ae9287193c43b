"""Attention of prompts over the 4-bit cache, 16-bit results: the kernel for many rows against 64 bits, in
every head size and group, over windows, pages that are not there, batches that mix lengths, and sequences
whose rows see nothing between others."""
import math

import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from kv4_data import Cache, attention, held
from q4_data import TORCH, assert_within

pytestmark = [pytest.mark.gpu, needs_gpu]


def _run(c, q, share, batch=None, window=0, sinks=0, scale=None, ctx=None, fill=7.0, asynchronous=False):
    """Rows behind the last sequence's make the call as large as those that this kernel is for."""
    rows, wide = q.shape
    all_rows = max(rows, 6500 // (c.heads * share))
    padded = torch.cat((q, torch.full((all_rows - rows, wide), math.nan, device="cuda", dtype=q.dtype)))
    y = torch.full((all_rows, wide), fill, device="cuda", dtype=c.kind)
    s = torch.full((all_rows, c.heads * share), fill, device="cuda")
    route = U.Route()
    U.kv4_attention(c.elem, c.elem, c.kv, c.batch if batch is None else batch, padded, padded.shape, y, y.shape, scale=scale, window=window,
                    sinks=sinks, lse=s, lv=s.shape, route=route, ctx=ctx, asynchronous=asynchronous)
    assert route.tile_m >= 128
    if not asynchronous:
        assert bool((y[rows:] == fill).all()) and bool((s[rows:] == fill).all())
    return y[:rows], s[:rows]


def _check(c, q, share, got, window=0, sinks=0, scale=None, keys_of=None):
    want, off, want_s, off_s = attention(c, q, share, c.dim ** -0.5 if scale is None else scale, c.elem, window, sinks, True, keys_of)
    live = sum(c.news)
    assert_within(got[0][:live], want[:live], off[:live], "y")
    assert_within(got[1][:live], want_s[:live], off_s[:live], "lse")
    assert bool((got[0][live:] == 7.0).all()) and bool((got[1][live:] == 7.0).all())


CASES = [
    # lengths, news, page, heads, dim, group, share, elem, window, sinks
    ([70], [70], 16, 1, 64, 32, 1, U.BF16, 0, 0),
    ([130, 257, 64], [130, 257, 64], 16, 2, 64, 64, 2, U.F16, 0, 0),
    ([300, 500], [40, 300], 32, 2, 96, 32, 4, U.BF16, 0, 0),
    ([1000, 90, 333], [130, 90, 100], 64, 2, 128, 32, 3, U.F16, 0, 0),
    ([1000], [513], 128, 3, 128, 64, 1, U.BF16, 0, 0),
    ([700, 65], [64, 65], 16, 1, 128, 128, 8, U.F16, 0, 0),
    ([400, 200], [300, 129], 32, 2, 192, 64, 2, U.BF16, 0, 0),
    ([400, 200], [100, 129], 16, 2, 192, 32, 1, U.F16, 0, 0),
    ([300, 129], [300, 17], 16, 1, 256, 32, 3, U.F16, 0, 0),
    ([260], [200], 64, 2, 256, 256, 1, U.BF16, 0, 0),
    ([900, 300], [500, 300], 16, 2, 64, 32, 2, U.F16, 100, 0),
    ([900, 300], [500, 300], 16, 2, 128, 32, 2, U.BF16, 65, 70),
    ([900], [300], 32, 1, 256, 128, 2, U.F16, 130, 5),
    ([2000], [600], 16, 1, 96, 32, 1, U.BF16, 17, 1000),
    ([600], [600], 16, 1, 64, 32, 4, U.BF16, 1, 0),
    ([5000, 129, 1, 64, 3000], [1, 129, 1, 64, 700], 64, 2, 128, 32, 4, U.BF16, 0, 0),
]


@pytest.mark.parametrize("lengths,news,page,heads,dim,group,share,elem,window,sinks", CASES)
def test_against_64_bits(lengths, news, page, heads, dim, group, share, elem, window, sinks):
    c = Cache(lengths, news, page, heads, dim, group, elem, pad=3, seed=dim + share).fill(shift=0.2)
    q = c.queries(share)
    got = _run(c, q, share, window=window, sinks=sinks)
    _check(c, q, share, got, window, sinks)
    again = _run(c, q, share, window=window, sinks=sinks)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dim", [64, 256])
def test_many_items(dim):
    """More items than processors, most of them of few steps, some of none."""
    lengths = [(37 * i) % 300 for i in range(90)]
    news = [max(1, n * (i % 3 + 1) // 3) + (5 if i % 7 == 0 else 0) for i, n in enumerate(lengths)]
    c = Cache(lengths, news, 16, 2, dim, 32, U.BF16, pad=1, seed=1).fill()
    q = c.queries(2)
    got = _run(c, q, 2)
    _check(c, q, 2, got)


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 40)])
@pytest.mark.parametrize("dim", [128, 192])
def test_pages_that_are_not_there(dim, window, sinks):
    c = Cache([400, 300], [200, 100], 32, 2, dim, 32, U.F16, seed=2).fill()
    c.table[0, 0], c.table[0, 3], c.table[0, 11], c.table[1, 9] = -1, c.pages, -2 ** 31, 2 ** 31 - 1
    there = [torch.ones(n, dtype=torch.bool, device="cuda") for n in c.lengths]
    there[0][:32] = there[0][96:128] = there[0][352:384] = there[1][288:] = False
    q = c.queries(2)
    _check(c, q, 2, _run(c, q, 2, window=window, sinks=sinks), window, sinks, keys_of=there)


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
@pytest.mark.parametrize("dim", [64, 256])
def test_what_lies_behind_the_last_token(elem, dim):
    c = Cache([150, 165, 17], [150, 90, 17], 64, 2, dim, 32, elem, seed=3)
    c.pool.view(torch.int16).fill_(0x7FC0 if elem == U.BF16 else 0x7E00)
    c.fill()
    q = c.queries(1)
    _check(c, q, 1, _run(c, q, 1))


@pytest.mark.parametrize("elem", [U.BF16, U.F16])
def test_extreme_keys_and_values(elem):
    """Keys and values at the type's ends, infinities among them, in tokens that most rows do not see yet:
    what a row does not see is not in its result."""
    n, dim = 320, 64
    c = Cache([n], [n], 16, 1, dim, 32, elem, seed=4)
    k, v = c.normal(n, dim).to(c.kind), c.normal(n, dim).to(c.kind)
    k[300, ::2], k[301, 3], v[302] = math.inf, -math.inf, math.inf
    v[303, ::2], v[304, 5], v[305] = -math.inf, math.nan, math.nan
    k[306, 7] = math.nan
    U.kv4_append(elem, c.kv, c.batch, k, k.shape, v, v.shape)
    c.k, c.v = [held(k.view(n, 1, dim), 32)], [held(v.view(n, 1, dim), 32)]
    q = c.queries(2)
    y, s = _run(c, q, 2)
    c.news, c.lengths = [300], [300]
    c.k, c.v = [c.k[0][:300]], [c.v[0][:300]]
    want, off, want_s, off_s = attention(c, q[:300], 2, dim ** -0.5, elem, rounded=True)
    assert_within(y[:300], want, off, "rows before them")
    assert_within(s[:300], want_s, off_s, "lse of rows before them")


def test_queries_that_are_not_finite():
    c = Cache([300], [200], 16, 1, 128, 32, U.F16, seed=5).fill()
    q = c.queries(2)
    bad = q.clone()
    bad[1, 5], bad[70, 128 + 9] = math.nan, math.inf
    y, s = _run(c, bad, 2)
    assert bool(torch.isnan(y[1, :128]).all()) and bool(torch.isnan(s[1, 0])) and bool(torch.isnan(y[70, 128:]).any())
    want, off, _, _ = attention(c, q, 2, 128 ** -0.5, U.F16, rounded=True)
    y[1, :128], y[70, 128:] = want[1, :128].half(), want[70, 128:].half()
    assert_within(y, want, off + 2.0 ** -11 * want.abs() + 2.0 ** -25, "the others")


@pytest.mark.parametrize("scale", [0.0, -0.3, 8.0])
def test_scales(scale):
    c = Cache([333], [222], 32, 2, 64, 32, U.BF16, seed=6).fill(size=0.3)
    q = c.queries(1, size=0.7)
    _check(c, q, 1, _run(c, q, 1, scale=scale), scale=scale)


def test_scores_that_climb():
    """Maxima that move at every step, by far and by little: sums in tensor memory are multiplied again and again."""
    n = 900
    c = Cache([n], [n], 16, 1, 64, 32, U.BF16, seed=7)
    ramp = torch.linspace(-6, 6, n, device="cuda")[:, None].expand(n, 64)
    q = torch.ones(n, 128, device="cuda").bfloat16()
    q[:, 64:] = 0.25
    k, v = ramp.bfloat16().contiguous(), c.normal(n, 64).bfloat16()
    U.kv4_append(U.BF16, c.kv, c.batch, k, k.shape, v, v.shape)
    c.k, c.v = [held(k.view(n, 1, 64), 32)], [held(v.view(n, 1, 64), 32)]
    _check(c, q, 2, _run(c, q, 2, scale=0.5), scale=0.5)


@pytest.mark.parametrize("starts,lengths", [([0, 90, 40, 120], [120, 30, 90]), ([50, 0, 30, 400], [100, 30, 110]),
                                            ([2 ** 31 - 1, -2 ** 31, 0, 300], [2 ** 31 - 1, -2 ** 31, 70])])
def test_starts_that_do_not_rise(starts, lengths):
    """Whatever the arrays hold, nothing outside the rows is written."""
    c = Cache([128, 128, 128], [1, 1, 1], 16, 1, 64, 32, U.BF16, seed=8).fill()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = U.Batch(ints(starts), ints(lengths), c.table, 3, c.cols)
    q = c.normal(200, 40 * 64).bfloat16()
    guard = torch.full((204, 40 * 64), 9.0, device="cuda", dtype=torch.bfloat16)
    route = U.Route()
    U.kv4_attention(U.BF16, U.BF16, c.kv, batch, q, q.shape, guard[2:202], (200, 40 * 64), route=route)
    assert route.tile_m >= 128
    assert bool((guard[:2] == 9.0).all()) and bool((guard[202:] == 9.0).all())


def test_strided_rows():
    c = Cache([300, 150], [200, 70], 16, 2, 64, 32, U.F16, pad=900, seed=9).fill()
    rows, wide, live = c.rows, 2 * 3 * 64, 270
    store = (c.normal(rows * (wide + 5) + 1) * 1.5).half()[1:]
    q = store.as_strided((rows, wide), (wide + 5, 1), 1).contiguous()
    out = torch.full((rows * (wide + 3) + 1,), 7.0, device="cuda", dtype=torch.float16)
    route = U.Route()
    U.kv4_attention(U.F16, U.F16, c.kv, c.batch, store, (rows, wide, wide + 5), out[1:], (rows, wide, wide + 3), route=route)
    assert route.tile_m >= 128
    want, off, _, _ = attention(c, q, 3, 64 ** -0.5, U.F16, rounded=True)
    assert_within(out[1:].as_strided((rows, wide), (wide + 3, 1), 1)[:live], want[:live], off[:live])
    assert bool((out[1:1 + rows * (wide + 3)].view(rows, wide + 3)[:, wide:] == 7.0).all()) and float(out[0]) == 7.0


def test_two_streams_and_a_graph():
    """Two contexts on two streams at once, and a captured call that follows what the arrays hold at its replay."""
    caches = [Cache([300 + 50 * i], [200], 16, 2, 128, 32, U.BF16, seed=10 + i).fill() for i in range(2)]
    qs = [c.queries(2) for c in caches]
    want = [_run(c, q, 2) for c, q in zip(caches, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [U.Context(0) for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for c, q, s, ctx in zip(caches, qs, streams, ctxs):
            ctx.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                got.append(_run(c, q, 2, ctx=ctx, asynchronous=True))
    assert all(ctx.sync() == 0 for ctx in ctxs)
    for i, g in enumerate(got):
        assert torch.equal(g[0], want[i % 2][0]) and torch.equal(g[1], want[i % 2][1])
    c, q, s, ctx = caches[0], qs[0], streams[0], ctxs[0]
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y, lse = _run(c, q, 2, ctx=ctx, asynchronous=True)
    lengths = c.batch.arrays[1]
    lengths.fill_(250)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    again = _run(c, q, 2)
    assert torch.equal(y, again[0]) and torch.equal(lse, again[1]) and not torch.equal(y, want[0][0])
    del graph
    for ctx in ctxs:
        ctx.close()


def test_pages_past_4_gb():
    """The same pages at the end of a pool of more than 2^32 bytes: the same bytes."""
    c = Cache([300, 40], [200, 40], 16, 2, 64, 32, U.BF16, seed=11).fill()
    q = c.queries(2)
    here = _run(c, q, 2)
    size = U.kv4_page_bytes(16, 2, 64, 32, U.BF16)
    behind = (1 << 32) // size + 1
    pool = torch.empty((behind + c.pages) * size, dtype=torch.uint8, device="cuda")
    pool[behind * size:] = c.pool
    c.kv = U.KV4(pool, behind + c.pages, 16, 2, 64, 32, U.BF16)
    c.table[c.table >= 0] += behind
    there = _run(c, q, 2)
    assert all(torch.equal(a, b) for a, b in zip(here, there))
