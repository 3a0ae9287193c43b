"""A decoder layer's attention half as a program runs it: the projection to queries, keys and values with its
bias, tokens into the cache with their rotation, attention, and the projection back onto the stream. Each
stage against 64 bits from what the one before it gave; prompts, then steps, eager and captured."""
import math

import pytest

import uor_b200 as U
from gpu_util import needs_gpu, torch
from kv4_data import Cache, attention, held, rotated
from q4_data import TORCH, Weights, assert_within, dot_bound, generator, round_bound

pytestmark = [pytest.mark.gpu, needs_gpu]


class Layer:
    def __init__(self, elem, heads, share, dim, group, window=0, sinks=0, width=320, positions=512):
        self.elem, self.heads, self.share, self.dim, self.group = elem, heads, share, dim, group
        self.window, self.sinks, self.width, self.kind = window, sinks, width, TORCH[elem]
        self.parts = [heads * share * dim, heads * dim, heads * dim]
        g = generator(5)
        self.into = Weights(sum(self.parts), width, 64, seed=1, zeros=True, spread=width ** -0.5 / 8)
        self.back = Weights(width, self.parts[0], 32, seed=2, zeros=False, spread=self.parts[0] ** -0.5 / 4)
        self.bias = (torch.randn(sum(self.parts), generator=g, device="cuda") * 0.2).to(self.kind)
        angle = torch.arange(positions, device="cuda").double()[:, None] * 10000.0 ** (
            -torch.arange(dim // 2, device="cuda").double() / (dim // 2))
        self.cos, self.sin = torch.cos(angle).float(), torch.sin(angle).float()
        self.turn = U.Rotation(self.cos, self.sin, positions, dim, False)

    def buffers(self, rows):
        empty = lambda n, kind=self.kind: torch.empty(rows, n, device="cuda", dtype=kind)  # noqa: E731
        return empty(sum(self.parts)), empty(self.parts[0]), empty(self.parts[0]), empty(self.heads * self.share, torch.float32)

    def run(self, kv, batch, x, buffers, ctx=None, asynchronous=False):
        """x (rows, width) becomes x plus the attention's part."""
        rows, (qkv, q, y, lse), how = x.shape[0], buffers, dict(ctx=ctx, asynchronous=asynchronous)
        n, wide = sum(self.parts), self.parts
        U.q4_linear(self.elem, self.elem, x, (rows, self.width), self.into.q, qkv, (rows, n), bias=self.bias, **how)
        flat = qkv.view(-1)
        U.kv4_append(self.elem, kv, batch, flat[wide[0]:], (rows, wide[1], n), flat[wide[0] + wide[1]:], (rows, wide[2], n),
                     q=qkv, qv=(rows, wide[0], n), q_out=q, ov=(rows, wide[0]), rotation=self.turn, **how)
        self.route = U.Route()
        U.kv4_attention(self.elem, self.elem, kv, batch, q, (rows, wide[0]), y, (rows, wide[0]), window=self.window, sinks=self.sinks,
                        lse=lse, lv=tuple(lse.shape), route=self.route, **how)
        U.q4_linear(self.elem, self.elem, y, (rows, wide[0]), self.back.q, x, (rows, self.width), residual=x, **how)


def _check(layer, cache, x0, x1, buffers, seen):
    """Every stage's output against 64 bits of its input. seen: per sequence the (keys, values) that the
    cache held before; grows by what it holds now."""
    qkv, q, y, lse = buffers
    rows, n = sum(cache.news), sum(layer.parts)
    want = x0[:rows].double() @ layer.into.value.T + layer.bias.double()
    off = dot_bound(x0[:rows].double(), layer.into.value, layer.width) + 2.0 ** -23 * want.abs()
    assert_within(qkv[:rows], want, off + round_bound(want.abs() + off, layer.elem))
    at = torch.cat([torch.arange(length - new, length, device="cuda") for new, length in zip(cache.news, cache.lengths)])
    heads = qkv[:rows].view(rows, -1, layer.dim)
    turned = rotated(heads[:, :layer.heads * (layer.share + 1)], layer.cos[at], layer.sin[at], layer.dim, False)
    assert torch.equal(q[:rows].view(rows, -1, layer.dim), turned[:, :layer.heads * layer.share])
    k = held(turned[:, layer.heads * layer.share:], layer.group)
    v = held(heads[:, layer.heads * (layer.share + 1):], layer.group)
    first = 0
    for i, new in enumerate(cache.news):
        seen[i] = tuple(torch.cat((old, now[first:first + new])) for old, now in zip(seen[i], (k, v)))
        first += new
    cache.k, cache.v = [s[0] for s in seen], [s[1] for s in seen]
    a, a_off, l, l_off = attention(cache, q[:rows], layer.share, layer.dim ** -0.5, layer.elem, layer.window, layer.sinks,
                                   rounded=layer.route.tile_m > 16)
    assert_within(y[:rows], a, a_off)
    assert_within(lse[:rows], l, l_off)
    want = y[:rows].double() @ layer.back.value.T
    off = dot_bound(y[:rows].double(), layer.back.value, layer.parts[0])
    want = want + x0[:rows].double()
    off = off + 2.0 ** -23 * (want.abs() + off)
    assert_within(x1[:rows], want, off + round_bound(want.abs() + off, layer.elem))


@pytest.mark.parametrize("many", [False, True])  # a large batch, most of it padding
@pytest.mark.parametrize("elem,heads,share,dim,group,window,sinks",
                         [(U.BF16, 2, 2, 64, 32, 0, 0), (U.F16, 1, 4, 128, 64, 0, 0), (U.BF16, 2, 3, 96, 32, 50, 4)])
def test_prompt_and_steps(elem, heads, share, dim, group, window, sinks, many):
    layer = Layer(elem, heads, share, dim, group, window, sinks)
    cache = Cache([144, 144, 16], [90, 133, 1], 16, heads, dim, group, elem, pad=6500 // (heads * share) if many else 2)
    cache.lengths = [90, 133, 1]
    cache.batch = cache.batch_of(cache.news)
    seen = [tuple(torch.empty(0, heads, dim, dtype=torch.float64, device="cuda") for _ in range(2)) for _ in cache.news]
    x0 = cache.normal(cache.rows, layer.width).to(layer.kind)
    x1, buffers = x0.clone(), layer.buffers(cache.rows)
    layer.run(cache.kv, cache.batch, x1, buffers)
    assert (layer.route.tile_m > 16) == many
    _check(layer, cache, x0, x1, buffers, seen)
    for _ in range(4):
        cache.news, cache.lengths, cache.rows = [1, 1, 1], [n + 1 for n in cache.lengths], 3
        x0 = cache.normal(3, layer.width).to(layer.kind)
        x1, buffers = x0.clone(), layer.buffers(3)
        layer.run(cache.kv, cache.batch_of([1, 1, 1]), x1, buffers)
        _check(layer, cache, x0, x1, buffers, seen)


def _decoding(layer):
    """A cache of two sequences with room to grow, in order, filled to 70 and 41 tokens."""
    cache = Cache([256, 256], [1, 1], 16, layer.heads, layer.dim, layer.group, layer.elem)
    cache.lengths = [70, 41]
    cache.batch = cache.batch_of([1, 1])
    cache.fill()
    return cache


@pytest.mark.parametrize("news,pad", [([1, 1], 0), ([3, 2], 1), ([60, 41], 0), ([60, 41], 1600)])
def test_a_captured_step_follows_the_device(news, pad):
    """One graph of the whole half, replayed over lengths and inputs that the device holds, is to the byte
    what eager calls give; a second graph of the same context between its replays changes nothing."""
    layer = Layer(U.BF16, 2, 2, 64, 32)
    eager, replayed = _decoding(layer), _decoding(layer)
    rows, live = sum(news) + pad, sum(news)
    inputs = [eager.normal(rows, layer.width).to(layer.kind) for _ in range(3)]
    ctx, stream = U.Context(0), torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    x, buffers = inputs[0].clone(), layer.buffers(rows)
    replayed.lengths = [n + new for n, new in zip(replayed.lengths, news)]
    batch = replayed.batch_of(news)
    lengths, grow = batch.arrays[1], torch.tensor(news, dtype=torch.int32, device="cuda")
    other, other_x, other_buffers = _decoding(layer), inputs[1].clone(), layer.buffers(rows)
    other_batch = other.batch_of(news)
    torch.cuda.synchronize()
    pool0 = replayed.pool.clone()
    with torch.cuda.stream(stream):
        layer.run(replayed.kv, batch, x, buffers, ctx, True)  # workspaces
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        with torch.cuda.graph(graphs[0], stream=stream):
            layer.run(replayed.kv, batch, x, buffers, ctx, True)
            lengths.add_(grow)
        with torch.cuda.graph(graphs[1], stream=stream):
            layer.run(other.kv, other_batch, other_x, other_buffers, ctx, True)
        replayed.pool.copy_(pool0)
        got = []
        for v in inputs:
            x.copy_(v)
            graphs[0].replay()
            got.append([x.clone(), buffers[2].clone(), buffers[3].clone()])
            graphs[1].replay()
    torch.cuda.synchronize()
    assert ctx.sync() == 0
    for v, g in zip(inputs, got):
        eager.lengths = [n + new for n, new in zip(eager.lengths, news)]
        mine, own = v.clone(), layer.buffers(rows)
        layer.run(eager.kv, eager.batch_of(news), mine, own)
        for a, b in zip(g, (mine, own[2], own[3])):
            assert torch.equal(a[:live], b[:live])
    assert torch.equal(eager.pool, replayed.pool)
    del graphs
    ctx.close()


def test_two_contexts_at_once():
    """Steps of two layers' halves queued on two streams by turns."""
    layers = [Layer(U.BF16, 2, 2, 64, 32), Layer(U.F16, 1, 4, 128, 64)]
    ctxs, streams = [U.Context(0) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    xs = [generator_rows(layer, i) for i, layer in enumerate(layers)]
    want = []
    for layer, x in zip(layers, xs):
        cache, mine, own = _decoding(layer), x.clone(), layer.buffers(2)
        layer.run(cache.kv, cache.batch, mine, own)
        want.append((mine, own[3]))
    caches, outs = [_decoding(layer) for layer in layers], [[(x.clone(), layer.buffers(2)) for _ in range(4)] for x, layer in zip(xs, layers)]
    torch.cuda.synchronize()
    for ctx, s in zip(ctxs, streams):
        ctx.set_stream(s.cuda_stream)
    for turn in range(4):
        for layer, cache, ctx, out in zip(layers, caches, ctxs, outs):
            layer.run(cache.kv, cache.batch, out[turn][0], out[turn][1], ctx, True)
    assert all(ctx.sync() == 0 for ctx in ctxs)
    for out, (x, lse) in zip(outs, want):
        for mine, own in out:
            assert torch.equal(mine, x) and torch.equal(own[3], lse)
    for ctx in ctxs:
        ctx.close()


def generator_rows(layer, seed):
    return torch.randn(2, layer.width, generator=generator(seed), device="cuda").to(layer.kind)


@pytest.mark.parametrize("n", [264, 1001])
@pytest.mark.parametrize("elem,out", [(U.BF16, U.BF16), (U.F16, U.F32)])
@pytest.mark.parametrize("skip", [0, 1, 8])
def test_many_rows_and_a_residual_that_lies_elsewhere(n, elem, out, skip):
    """Rows of the residual with a stride of their own, at any alignment, and added in place."""
    m, k = 530, 520
    w = Weights(n, k, 64, seed=n, zeros=True, spread=k ** -0.5)
    g = generator(n + skip)
    x = torch.randn(m, k, generator=g, device="cuda").to(TORCH[elem])
    lies = torch.randn(m, n + 24, generator=g, device="cuda").to(TORCH[out])
    residual = lies.view(-1)[skip:]
    added = torch.as_strided(lies, (m, n), (n + 24, 1), skip).double()
    v = x.double() @ w.value.T
    off = dot_bound(x.double(), w.value, k)
    want = v / (1 + torch.exp(-v)) + added
    off = 1.13 * off + 2.0 ** -18 * v.abs() + 2.0 ** -24 + 2.0 ** -23 * (want.abs() + off)
    off = off + round_bound(want.abs() + off, out)
    y = torch.empty(m, n, device="cuda", dtype=TORCH[out])
    U.q4_linear(elem, out, x, (m, k), w.q, y, (m, n), activation=U.SILU, residual=residual, rv=(m, n, n + 24))
    assert_within(y, want, off)
    U.q4_linear(elem, out, x, (m, k), w.q, residual, (m, n, n + 24), activation=U.SILU, residual=residual, rv=(m, n, n + 24))
    assert torch.equal(torch.as_strided(lies, (m, n), (n + 24, 1), skip), y)
