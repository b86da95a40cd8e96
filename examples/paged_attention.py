"""A decoder layer's attention block over a paged cache: prompts in chunks, then decoding.

The q|k|v and o projections are 4-bit ``QuantizedLinear`` handles; between them one launch
norms and rotates the heads and appends keys and values to the cache, and one call attends.
Prompts of several requests go in together, a chunk at a time; then every request decodes
one token a step, the whole block captured in a graph whose replays follow the batch's
device arrays.

    python examples/paged_attention.py [--layer sliding|full] [--requests 8] [--prompt 2000] [--e4m3 [--block 64]]

Weights are random, in the shapes of the decoder that bench.py runs.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from helios_amd import HeadNorm, KVBatch, PagedKVCache, QuantizedLinear, Rope, quantize  # noqa: E402

HIDDEN = 3840
# query heads, KV heads, head_dim, window, rotation base, rotated pairs
LAYERS = {"sliding": (16, 8, 256, 1024, 1e4, 128), "full": (16, 1, 512, 0, 1e6, 64)}


class AttentionBlock:
    """x -> o(attention(q, k, v of x)) for the new tokens of a batch."""

    def __init__(self, hidden, q_heads, kv_heads, head_dim, window, base, pairs, generator):
        randn = lambda *s: torch.randn(s, device="cuda", generator=generator)  # noqa: E731
        self.q_heads, self.kv_heads, self.head_dim, self.window = q_heads, kv_heads, head_dim, window
        # a layer of one KV head takes its values from the keys' columns
        self.shared_kv = kv_heads == 1
        columns = (q_heads + kv_heads * (1 if self.shared_kv else 2)) * head_dim
        self.qkv = QuantizedLinear(*quantize(randn(columns, hidden) * hidden ** -0.5))
        self.o = QuantizedLinear(*quantize(randn(hidden, q_heads * head_dim) * (q_heads * head_dim) ** -0.5))
        inv_freq = base ** (-2.0 * torch.arange(pairs, device="cuda", dtype=torch.float32) / head_dim)
        self.rope = Rope(inv_freq, head_dim // 2)
        self.q_norm = HeadNorm((1 + 0.1 * randn(head_dim)).bfloat16())
        self.k_norm = HeadNorm((1 + 0.1 * randn(head_dim)).bfloat16())
        self.v_norm = HeadNorm()

    def attend(self, rows, cache, batch):
        """Attention of fused q|k|v rows [tokens, columns]; their keys and values join the cache."""
        d, q_end, k_end = self.head_dim, self.q_heads * self.head_dim, (self.q_heads + self.kv_heads) * self.head_dim
        q, k = rows[:, :q_end].unflatten(1, (-1, d)), rows[:, q_end:k_end].unflatten(1, (-1, d))
        v = k if self.shared_kv else rows[:, k_end:].unflatten(1, (-1, d))
        q = cache.append(k, v, batch, rope=self.rope, k_norm=self.k_norm, v_norm=self.v_norm, q=q, q_norm=self.q_norm)
        return cache.attend(q, batch, scale=1.0, window=self.window)

    def __call__(self, x, cache, batch):
        return self.o(self.attend(self.qkv(x), cache, batch).flatten(1))


def make_batch(q_lens, kv_lens, tables):
    """The device arrays of requests with q_lens new tokens each, kv_lens tokens with them."""
    starts = torch.zeros(len(q_lens) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(q_lens).cumsum(0)
    return KVBatch(starts.cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda(), tables)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--layer", choices=sorted(LAYERS), default="sliding")
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--prompt", type=int, default=2000, help="tokens of the longest prompt")
    p.add_argument("--chunk", type=int, default=512, help="tokens of a prompt that go in at once")
    p.add_argument("--steps", type=int, default=64, help="tokens decoded per request")
    p.add_argument("--page", type=int, default=64)
    p.add_argument("--e4m3", action="store_true", help="keep the cache in 8-bit floats")
    p.add_argument("--block", type=int, default=0, help="with --e4m3: a scale for each so many tokens, found from the values")
    a = p.parse_args()
    g = torch.Generator(device="cuda").manual_seed(1)
    q_heads, kv_heads, head_dim, window, base, pairs = LAYERS[a.layer]
    block = AttentionBlock(HIDDEN, q_heads, kv_heads, head_dim, window, base, pairs, g)

    prompts = [max(1, a.prompt * (a.requests - i) // a.requests) for i in range(a.requests)]
    width = -(-(a.prompt + a.steps) // a.page)
    tables = torch.randperm(a.requests * width, device="cuda", generator=g).to(torch.int32).view(a.requests, width)
    kind, scale = (torch.float8_e4m3fn, 1.0 if a.block else 1 / 16) if a.e4m3 else (torch.bfloat16, 1.0)
    cache = PagedKVCache.allocate(a.requests * width, a.page, kv_heads, head_dim, kind, scale, scale, scale_block=a.block)

    def timed(what, tokens, call):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        call()
        end.record()
        torch.cuda.synchronize()
        ms = begin.elapsed_time(end)
        print(f"{what}: {tokens} tokens, {ms:.2f} ms, {tokens / ms * 1e3:.0f} tokens/s", flush=True)

    def prefill():
        for at in range(0, max(prompts), a.chunk):
            ends = [min(n, at + a.chunk) for n in prompts]
            new = [max(0, e - at) for e in ends]
            x = torch.randn(sum(new), HIDDEN, device="cuda", generator=g).bfloat16()
            block(x, cache, make_batch(new, ends, tables))

    prefill()  # the first calls take scratch memory; the second pass stores the same slots again
    timed("prompts", sum(prompts), prefill)

    batch = make_batch([1] * a.requests, [n + 1 for n in prompts], tables)
    x = torch.randn(a.requests, HIDDEN, device="cuda", generator=g).bfloat16()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(x, cache, batch)  # takes the stream's scratch memory before the capture
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = block(x, cache, batch)

    def decode():
        for _ in range(a.steps - 1):
            graph.replay()
            x.copy_(y)  # a model's next layer would go here
            batch.kv_lens += 1

    timed("decoding", a.requests * (a.steps - 1), decode)


if __name__ == "__main__":
    main()
