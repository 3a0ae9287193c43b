"""A mixture-of-experts layer over 4-bit weights, from float weights to trained router.

    python examples/moe_layer.py [--tokens 512] [--d 1024] [--f 512] [--experts 32] [--top-k 4]

For a row x of hidden states the layer computes

    h = x + O x                         O in 4 bits (q4_gemm)
    ids, weights = route(R h)           expert_route over f32 logits
    y = h + sum_s weights[s] FFN_ids[s](h)   experts in 4 bits (expert_q4_ffn)

first for a batch, then token by token from a CUDA graph, as a decoder does, and then trains R
with the experts held fixed, through expert_route_backward. Last it puts an attention half before the
layer, over keys and values in 4 bits (q4_linear, kv4_append, kv4_attention, q4_linear), and runs the two
for a prompt and then token by token from one graph. Needs a CUDA GPU."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "uor-matmul_b200"))
import uor_b200 as U  # noqa: E402


def quantize(w, group):
    """Float weights (rows x cols) as a Q4 descriptor: per row and group the range of the weights,
    with 0 in it, in 15 steps, and the zero point that 0 falls on."""
    rows, cols = w.shape
    groups = -(-cols // group)
    padded = torch.nn.functional.pad(w.float(), (0, groups * group - cols)).view(rows, groups, group)
    low, high = padded.amin(2).clamp(max=0), padded.amax(2).clamp(min=0)
    scales = ((high - low) / 15).clamp(min=1e-8)
    zeros = (-low / scales).round().clamp(0, 15)
    codes = (padded / scales[..., None] + zeros[..., None]).round().clamp(0, 15).to(torch.uint8).view(rows, -1)
    codes = codes[:, :cols + cols % 2]  # groups are even: the last byte's other half is there
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous()
    return U.Q4(packed.view(-1), scales.view(-1), U.F32, rows, cols, group, zeros=zeros.to(torch.uint8).view(-1))


def dequantize(q):
    """The descriptor's weights in float64, for comparison."""
    codes, scales, zeros = (t.view(q.rows, -1) for t in q.arrays)
    code = torch.stack((codes & 15, codes >> 4), 2).view(q.rows, -1)[:, :q.cols]
    at = torch.arange(q.cols, device=codes.device) // q.group
    return (code.double() - zeros[:, at].double()) * scales[:, at].double()


class MoELayer:
    """The layer's weights and a library context bound to a stream."""

    def __init__(self, d, f, experts, top_k, group=64, seed=0, stream=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.d, self.f, self.experts, self.top_k = d, f, experts, top_k
        self.mix = quantize(normal(d, d) * 0.5 * d ** -0.5, group)
        self.router = normal(experts, d) * d ** -0.5
        self.up = quantize(normal(experts * 2 * f, d) * d ** -0.5, group)
        self.down = quantize(normal(experts * d, f) * f ** -0.5, group)
        self.choice = U.Router(experts, top_k, score=U.SOFTMAX, renormalize=True)
        self.stream = stream or torch.cuda.Stream()
        self.ctx = U.Context(torch.cuda.current_device())
        self.ctx.set_stream(self.stream.cuda_stream)

    def close(self):
        self.ctx.close()

    def done(self):
        """Wait for the calls so far and raise what the device reported."""
        status = self.ctx.sync()
        if status:
            raise U.UorError(status, "moe layer")

    def mixed(self, x):
        t, d = x.shape
        out = torch.empty_like(x)
        U.q4_gemm(U.BF16, U.BF16, x, (t, d), self.mix, out, (t, d), ctx=self.ctx, asynchronous=True)
        return x + out

    def route(self, h):
        t = h.shape[0]
        logits = h.float() @ self.router.T
        ids = torch.empty(t, self.top_k, dtype=torch.int32, device="cuda")
        weights = torch.empty(t, self.top_k, dtype=torch.float32, device="cuda")
        U.expert_route(U.F32, self.choice, logits, (t, self.experts), None, ids, (t, self.top_k),
                       weights, (t, self.top_k), ctx=self.ctx, asynchronous=True)
        return logits, ids, weights

    def experts_out(self, h, ids, weights, out=U.BF16):
        t, k = ids.shape
        y = torch.empty(t, self.d, dtype=torch.bfloat16 if out == U.BF16 else torch.float32, device="cuda")
        U.expert_q4_ffn(U.BF16, out, self.experts, h, (t, self.d), ids, (t, k), weights, (t, k),
                        self.up, self.down, y, (t, self.d), ctx=self.ctx, asynchronous=True)
        return y

    def forward(self, x):
        """x (tokens x d, bfloat16) -> the layer's output, on the layer's stream."""
        h = self.mixed(x)
        _, ids, weights = self.route(h)
        return h + self.experts_out(h, ids, weights)

    def router_step(self, h, target, rate):
        """One descent step of 0.5 |sum_s weights[s] FFN_s(h) - target|^2 / tokens on the router.
        The gradient of weights[t][s] is the output's along what expert s gives alone."""
        t = h.shape[0]
        logits, ids, weights = self.route(h)
        y = self.experts_out(h, ids, weights, U.F32)
        dy = (y - target) / t
        alone = torch.ones(t, 1, device="cuda")
        dweights = torch.empty_like(weights)
        for s in range(self.top_k):
            part = self.experts_out(h, ids[:, s:s + 1].contiguous(), alone, U.F32)
            dweights[:, s] = (dy * part).sum(1)
        dlogits = torch.empty_like(logits)
        U.expert_route_backward(U.F32, self.choice, logits, (t, self.experts), ids, (t, self.top_k), dweights,
                                (t, self.top_k), dlogits, (t, self.experts), ctx=self.ctx, asynchronous=True)
        self.router -= rate * (dlogits.T @ h.float())
        return 0.5 * (y - target).square().sum() / t


class Attention:
    """The attention half before a layer, for one sequence: x + O attention(rotated heads of W x + b) over a
    paged cache of 4-bit keys and values, whose length the device holds."""

    def __init__(self, layer, heads=8, shared_by=4, dim=64, positions=512, group=64, seed=2):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.layer, self.heads, self.wide = layer, heads, heads * dim
        self.keys = heads // shared_by * dim  # channels of a token's keys, and of its values
        rows = self.wide + 2 * self.keys
        self.into = quantize(torch.randn(rows, layer.d, generator=g, device="cuda") * layer.d ** -0.5, group)
        self.bias = (torch.randn(rows, generator=g, device="cuda") * 0.1).bfloat16()
        self.back = quantize(torch.randn(layer.d, self.wide, generator=g, device="cuda") * 0.5 * self.wide ** -0.5, group)
        page = 64
        pages = -(-positions // page)
        self.pool = torch.zeros(pages * U.kv4_page_bytes(page, heads // shared_by, dim, 32, U.BF16), dtype=torch.uint8, device="cuda")
        self.cache = U.KV4(self.pool, pages, page, heads // shared_by, dim, 32, U.BF16)
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, pages)
        self.length = torch.zeros(1, dtype=torch.int32, device="cuda")
        angle = torch.arange(pages * page, device="cuda").double()[:, None] * 10000.0 ** (
            -torch.arange(dim // 2, device="cuda").double() / (dim // 2))
        self.turn = U.Rotation(torch.cos(angle).float(), torch.sin(angle).float(), pages * page, dim, False)

    def batch(self, rows):
        """The sequence's newest `rows` tokens."""
        return U.Batch(torch.tensor([0, rows], dtype=torch.int32, device="cuda"), self.length, self.table, 1, self.table.shape[1])

    def forward(self, x, batch):
        """x (rows x d): the sequence's next tokens, on the layer's stream; its length grows by them."""
        t, d = x.shape
        self.length += t
        how = dict(ctx=self.layer.ctx, asynchronous=True)
        rows = self.wide + 2 * self.keys
        heads = torch.empty(t, rows, dtype=torch.bfloat16, device="cuda")
        U.q4_linear(U.BF16, U.BF16, x, (t, d), self.into, heads, (t, rows), bias=self.bias, **how)
        q, k, v = heads, heads.view(-1)[self.wide:], heads.view(-1)[self.wide + self.keys:]
        U.kv4_append(U.BF16, self.cache, batch, k, (t, self.keys, rows), v, (t, self.keys, rows), q=q, qv=(t, self.wide, rows),
                     q_out=q, ov=(t, self.wide, rows), rotation=self.turn, **how)
        y = torch.empty(t, self.wide, dtype=torch.bfloat16, device="cuda")
        U.kv4_attention(U.BF16, U.BF16, self.cache, batch, q, (t, self.wide, rows), y, (t, self.wide), **how)
        out = torch.empty_like(x)
        U.q4_linear(U.BF16, U.BF16, y, (t, self.wide), self.back, out, (t, d), residual=x, **how)
        return out


def run_attention(layer, x, report=print):
    """A prompt through an attention half and the layer, then its last tokens once more, one by one from a
    graph; how far the two are apart in units of the largest output."""
    half, last = Attention(layer, positions=x.shape[0] + 64), min(8, x.shape[0])
    torch.cuda.synchronize()
    with torch.cuda.stream(layer.stream):
        batch = half.batch(x.shape[0])
        y = layer.forward(half.forward(x, batch))
        one, token = half.batch(1), x[:1].clone()
        layer.forward(half.forward(token, one))  # the context's buffers grow to this shape before the capture
        layer.done()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=layer.stream):
            out = layer.forward(half.forward(token, one))
        half.length.fill_(x.shape[0] - last)
        found = []
        for t in range(x.shape[0] - last, x.shape[0]):
            token.copy_(x[t:t + 1])
            graph.replay()
            found.append(out.clone())
        layer.done()
    far = float((torch.cat(found).float() - y[-last:].float()).abs().max() / y.float().abs().max())
    report(f"attention over 4-bit keys and values and the layer, {x.shape[0]} tokens, the last {last} again from a graph: "
           f"{far:.4f} of the largest output apart")
    del graph
    return far, torch.cat(found), half


class Decoder:
    """One token at a time: the layer's forward captured once in a CUDA graph and replayed."""

    def __init__(self, layer):
        self.layer = layer
        self.x = torch.zeros(1, layer.d, dtype=torch.bfloat16, device="cuda")
        with torch.cuda.stream(layer.stream):
            layer.forward(self.x)  # the context's buffers grow to this shape before the capture
            layer.done()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=layer.stream):
                self.y = layer.forward(self.x)

    def step(self, x):
        with torch.cuda.stream(self.layer.stream):
            self.x.copy_(x)
            self.graph.replay()
            return self.y.clone()


def timed(stream, fn, repeats=20):
    """Microseconds of one fn(), by events on the stream after three warm-up runs."""
    with torch.cuda.stream(stream):
        for _ in range(3):
            fn()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(repeats):
            fn()
        b.record()
    b.synchronize()
    return a.elapsed_time(b) * 1e3 / repeats


def run(tokens, d, f, experts, top_k, steps=10, report=print):
    """The example; returns what it found."""
    layer = MoELayer(d, f, experts, top_k)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(tokens, d, generator=g, device="cuda").bfloat16()
    torch.cuda.synchronize()
    with torch.cuda.stream(layer.stream):
        y = layer.forward(x)
        layer.done()
    report(f"{tokens} tokens, {top_k} of {experts} experts of {d}x{f}: "
           f"{timed(layer.stream, lambda: layer.forward(x)):.1f} us a layer")

    decoder = Decoder(layer)
    one = torch.cat([decoder.step(x[t:t + 1]) for t in range(min(tokens, 8))])
    torch.cuda.synchronize()
    far = float((one.float() - y[:one.shape[0]].float()).abs().max() / y.float().abs().max())
    report(f"token by token from a CUDA graph: {timed(layer.stream, decoder.graph.replay):.1f} us a layer, "
           f"{far:.4f} of the largest output from the batch's")

    # a router that was knocked off its place finds back to the outputs it gave
    with torch.cuda.stream(layer.stream):
        h = layer.mixed(x)
        _, ids, weights = layer.route(h)
        target = layer.experts_out(h, ids, weights, U.F32)
        layer.router += 0.2 * d ** -0.5 * torch.randn(experts, d, generator=g, device="cuda")
        rate = 2.0 * tokens / d ** 2  # a token's logits see |h|^2 / tokens ~ d / tokens, its outputs ~ d
        losses = [float(layer.router_step(h, target, rate)) for _ in range(steps)]
        layer.done()
    report(f"router: loss {losses[0]:.3f} -> {losses[-1]:.3f} in {steps} steps")
    del decoder
    layer.close()
    return {"far": far, "losses": losses}


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tokens", 512), ("d", 1024), ("f", 512), ("experts", 32), ("top-k", 4), ("steps", 10)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args()
    run(a.tokens, a.d, a.f, a.experts, a.top_k, a.steps)
    whole = MoELayer(a.d, a.f, a.experts, a.top_k)
    run_attention(whole, torch.randn(a.tokens, a.d, device="cuda").bfloat16())
    whole.close()
