"""The attention block of examples/paged_attention.py on the GPU: prompts in chunks and
single tokens leave the same cache as the whole prompts at once and attend as its 64-bit
values do; a captured step replays as the eager one runs."""

import numpy as np
import pytest

import attention_oracle as O

pytestmark = pytest.mark.gpu

SMALL = {"sliding": (4, 2, 256, 40, 1e4, 128), "full": (8, 1, 512, 0, 1e6, 64)}


def block_and_tables(layer, prompts, page, generator):
    import torch

    from examples import paged_attention as E

    block = E.AttentionBlock(256, *SMALL[layer], generator)
    width = -(-max(prompts) // page)
    tables = torch.randperm(len(prompts) * width, device="cuda", generator=generator).to(torch.int32).view(len(prompts), width)
    return E, block, tables, width


@pytest.mark.parametrize("layer", sorted(SMALL))
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_chunks_and_tokens_leave_the_cache_of_whole_prompts(gpu_lib, layer, kind):
    import torch

    g = torch.Generator(device="cuda").manual_seed(3)
    prompts, page = [130, 57, 7], 32
    E, block, tables, width = block_and_tables(layer, prompts, page, g)
    x = [torch.randn(n, 256, device="cuda", generator=g).bfloat16() for n in prompts]
    rows = block.qkv(torch.cat(x)).split(prompts)
    dtype, scale = (torch.bfloat16, 1.0) if kind == "bf16" else (torch.float8_e4m3fn, 0.0625)
    caches = [E.PagedKVCache.allocate(len(prompts) * width, page, block.kv_heads, block.head_dim, dtype, scale, scale) for _ in range(2)]
    for c in caches:
        c.k.zero_()
        c.v.zero_()
    whole = block.attend(torch.cat(rows), caches[0], E.make_batch(prompts, prompts, tables)).split(prompts)
    parts = [[] for _ in prompts]
    steps = [0, 50, 51, 52, 100, 129, 130]
    for a, b in zip(steps, steps[1:]):
        ends = [min(n, b) for n in prompts]
        new = [max(0, e - a) for e in ends]
        out = block.attend(torch.cat([r[a:a + n] for r, n in zip(rows, new)]), caches[1], E.make_batch(new, ends, tables))
        for part, o in zip(parts, out.split(new)):
            part.append(o)
    for name in ("k", "v"):
        one, two = (getattr(c, name).view(torch.uint8) for c in caches)
        assert torch.equal(one, two), name
    b = {"starts": np.concatenate([[0], np.cumsum(prompts)]), "kv_lens": np.array(prompts), "tables": tables.cpu().numpy(),
         "page": page, "num_pages": len(prompts) * width, "rows": sum(prompts)}
    at = torch.cat([torch.arange(n) for n in prompts]).int().cuda()
    q_cols = block.q_heads * block.head_dim
    q = torch.cat(rows)[:, :q_cols].unflatten(1, (-1, block.head_dim))
    q, _ = normed_q(q, at, block)
    k64, v64 = O.f64(caches[0].k) * scale, O.f64(caches[0].v) * scale
    want, bound, _, _ = O.attend(O.f64(q), k64, v64, b, 1.0, block.window)
    O.assert_within(O.f64(torch.cat(whole)), want, bound, "whole prompts")
    O.assert_within(O.f64(torch.cat([torch.cat(p) for p in parts])), want, bound, "chunks and tokens")


def normed_q(q, positions, block):
    from helios_amd import qk_norm_rope

    return qk_norm_rope(q, None, positions, block.rope, q_norm=block.q_norm)


@pytest.mark.parametrize("layer", sorted(SMALL))
def test_a_captured_step_follows_the_batch(gpu_lib, layer):
    """qkv, append, attention and o in one graph, replayed as the requests grow, against the
    eager block, with eager work between the replays."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(5)
    lens, steps, page = [1, 40, 700], 4, 16
    E, block, tables, width = block_and_tables(layer, [n + steps + 1 for n in lens], page, g)
    caches = [E.PagedKVCache.allocate(len(lens) * width, page, block.kv_heads, block.head_dim) for _ in range(2)]
    for c in caches:
        c.k.normal_(generator=torch.Generator(device="cuda").manual_seed(7))
        c.v.normal_(generator=torch.Generator(device="cuda").manual_seed(8))
    batches = [E.make_batch([1] * len(lens), [n + 1 for n in lens], tables) for _ in range(2)]
    x = torch.randn(len(lens), 256, device="cuda", generator=g).bfloat16()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(x, caches[0], batches[0])
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        replayed = block(x, caches[0], batches[0])
    for i in range(steps):
        x.normal_(generator=g)
        graph.replay()
        eager = block(x, caches[1], batches[1])
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager), f"step {i}"
        for b in batches:
            b.kv_lens += 1
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
