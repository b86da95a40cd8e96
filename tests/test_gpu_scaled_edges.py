"""The append to block-scaled pages at the ends of what it takes, on the GPU."""

import numpy as np
import pytest

from test_gpu_attention import dev, randn

pytestmark = pytest.mark.gpu


def ints(*values):
    return dev(np.array(values, np.int32))


def filled(cache, code=0x38, byte=127):
    import torch

    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(code)
    for t in (cache.k_scale, cache.v_scale):
        t.view(torch.uint8).fill_(byte)
    return cache


@pytest.mark.parametrize("past,rows", [(1, 1), (3, 5), (100, 7), (2 ** 30 - 1, 3), (5, 6)])
def test_tokens_past_a_table_of_2_30(gpu_lib, past, rows):
    """Lengths behind a full table of 2^30 tokens (a request that got no pages counts them): each
    token goes to its own place, or nowhere."""
    import torch

    from helios_amd import KVBatch, PagedKVCache

    rng = np.random.default_rng(past + rows)
    page, width, d = 65536, 16384, 64
    tables = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    tables[0, -1] = 1
    x, y = randn(rng, rows, 1, d), randn(rng, rows, 1, d)
    got = filled(PagedKVCache.allocate(2, page, 1, d, torch.float8_e4m3fn, scale_block=16))
    got.append(x, y, KVBatch(ints(0, rows), ints(2 ** 30 + past), tables))
    want = filled(PagedKVCache.allocate(2, page, 1, d, torch.float8_e4m3fn, scale_block=16))
    inside = max(0, rows - past)
    if inside:
        want.append(x[:inside], y[:inside], KVBatch(ints(0, inside), ints(2 ** 30), tables))
    for a, b in ((got.k, want.k), (got.v, want.v), (got.k_scale, want.k_scale), (got.v_scale, want.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
