"""The append to block-scaled pages at the ends of what it takes, on the GPU."""

import numpy as np
import pytest

from test_gpu_attention import dev, randn
from test_gpu_scaled_cache import codes64, e4m3, exponents, least

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


def test_arrays_of_one_allocation(gpu_lib):
    """K and V between each other, scales likewise, q normed in place within a fused projection's rows: as
    from arrays apart; what shares bytes is refused and nothing is written."""
    import torch

    from helios_amd import Gemma4Error, HeadNorm, KVBatch, PagedKVCache

    rng = np.random.default_rng(8)
    pages, hk, page, d, rows = 6, 2, 32, 128, 40
    batch = KVBatch(ints(0, 33, rows), ints(50, 7), ints(0, 1, 2, 3).view(2, 2))
    x = randn(rng, rows, 8 * d)
    norm = HeadNorm(None, 1e-6)
    of = lambda t, a, b: t[:, a * d:b * d].unflatten(1, (b - a, d))  # noqa: E731
    apart = filled(PagedKVCache.allocate(pages, page, hk, d, torch.float8_e4m3fn, scale_block=16))
    want = apart.append(of(x, 4, 6), of(x, 6, 8), batch, k_norm=norm, v_norm=norm, q=of(x, 0, 4), q_norm=norm)
    for axis in (0, 1, 2, 3):  # where K and V take turns
        shape, small = [pages, hk, page, d], [pages, hk, page // 16]
        both = torch.zeros(shape[:axis] + [2] + shape[axis:], device="cuda").to(torch.float8_e4m3fn)
        scale = torch.zeros(small[:min(axis, 2)] + [2] + small[min(axis, 2):], dtype=torch.uint8, device="cuda")
        cache = filled(PagedKVCache(both.select(axis, 0), both.select(axis, 1), scale.select(min(axis, 2), 0), scale.select(min(axis, 2), 1)))
        y = x.clone()
        got = cache.append(of(y, 4, 6), of(y, 6, 8), batch, k_norm=norm, v_norm=norm, q=of(y, 0, 4), q_norm=norm, out_q=of(y, 0, 4))
        assert torch.equal(got, want) and torch.equal(y[:, :4 * d], want.flatten(1)) and torch.equal(y[:, 4 * d:], x[:, 4 * d:])
        for a, b in ((cache.k, apart.k), (cache.v, apart.v), (cache.k_scale, apart.k_scale), (cache.v_scale, apart.v_scale)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), axis
    before = [t.view(torch.uint8).clone() for t in (apart.k, apart.v, apart.k_scale, apart.v_scale, x)]
    k, v, s, t = apart.k, apart.v, apart.k_scale, apart.v_scale
    args = (of(x, 4, 6), of(x, 6, 8), batch)
    for cache in (PagedKVCache(k, k, s, t), PagedKVCache(k, v, s, s), PagedKVCache(k[:-1], k[1:], s[:-1], t[:-1])):
        with pytest.raises(Gemma4Error, match="must not overlap"):
            cache.append(*args, k_norm=norm)
        cache.attend(of(x, 0, 4), batch)  # reads alone
    for out in (of(x, 2, 6), of(x, 4, 8)):
        with pytest.raises(Gemma4Error, match="k's or v's rows"):
            apart.append(*args, k_norm=norm, v_norm=norm, q=of(x, 0, 4), q_norm=norm, out_q=out)
    with pytest.raises(Gemma4Error, match="be its x"):
        apart.append(*args, q=of(x, 0, 3), q_norm=norm, out_q=of(x, 1, 4))
    for was, t in zip(before, (apart.k, apart.v, apart.k_scale, apart.v_scale, x)):
        assert torch.equal(was, t.view(torch.uint8))


@pytest.mark.parametrize("d,block,kept,loud", [(64, 16, 5, 3), (256, 32, 20, 8), (512, 64, 1, 40), (128, 16, 15, 1)])
def test_dropped_drafts_leave_their_scale(gpu_lib, d, block, kept, loud):
    """Drafts 64 times as large as the tokens before them raise the block's scale for good: the
    tokens before them are rounded twice, the second time to a step of the raised scale, and no
    more than that; the block begun anew has a scale of its own again."""
    import torch

    from helios_amd import KVBatch, PagedKVCache

    rng = np.random.default_rng(d)
    page, hk = 64, 2
    cache = filled(PagedKVCache.allocate(1, page, hk, d, torch.float8_e4m3fn, scale_block=block))
    table = ints(0).view(1, 1)
    batch = lambda n, length: KVBatch(ints(0, n), ints(length), table)  # noqa: E731
    first, drafts, last = (randn(rng, n, hk, d) for n in (kept, loud, 1))
    cache.append(first, first, batch(kept, kept))
    before, low = codes64(cache.k), exponents(cache.k_scale)
    cache.append(drafts * 64, drafts * 64, batch(loud, kept + loud))
    cache.append(last, last, batch(1, kept + 1))  # in the first draft's place
    after, high = codes64(cache.k), exponents(cache.k_scale)
    in_block = min(loud, block - kept)
    for h in range(hk):
        y = first[:, h].double().cpu().numpy()
        e0, e1 = int(low[0, h, 0]), int(high[0, h, 0])
        assert e0 == least(np.abs(y).max())
        assert e1 == least(np.abs(drafts[:in_block, h].double().cpu().numpy() * 64).max()) > e0
        assert np.array_equal(after[0, h, :kept], e4m3(before[0, h, :kept] * 2.0 ** (e0 - e1)))
        # half a step of each scale: 2^-4 of the value, 2^-10 of the scale under its least normal code
        one = np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** (e0 - 10))
        both = one + np.maximum(2.0 ** -4 * (np.abs(y) + one), 2.0 ** (e1 - 10))
        assert (np.abs(after[0, h, :kept] * 2.0 ** e1 - y) <= both).all()
        z = last[0, h].double().cpu().numpy()
        assert (np.abs(after[0, h, kept] * 2.0 ** e1 - z) <= np.maximum(2.0 ** -4 * np.abs(z), 2.0 ** (e1 - 10))).all()
    assert torch.equal(cache.k.view(torch.uint8), cache.v.view(torch.uint8)) and torch.equal(cache.k_scale, cache.v_scale)
    cache.append(first, first, batch(kept, kept))
    assert np.array_equal(codes64(cache.k)[0, :, :kept], before[0, :, :kept]) and np.array_equal(exponents(cache.k_scale)[0, :, 0], low[0, :, 0])


def test_requests_without_pages_left_out_of_a_step(gpu_lib):
    """A second reserve of new_tokens * granted is the same step without the requests that got no
    pages: the others keep what they were given, and nothing is stored for those."""
    import torch

    from helios_amd import PagedKVCache, PagePool

    rng = np.random.default_rng(12)
    for new, held, pages in (([5, 40, 3], [3, 10, 0], 3), ([9, 17, 17, 0, 30], [16, 16, 15, 4, 2], 6)):
        n = len(new)
        pool = PagePool.allocate(pages, 16, n, 6)
        pool.reserve(ints(*held))
        assert pool.granted.tolist() == [1] * n
        pool.release(ints(*held))
        first = ints(*new)
        pool.reserve(first)
        granted = pool.granted.tolist()
        assert 0 in granted and 1 in granted
        tables, count = pool.block_tables.clone(), int(pool.free_count)
        _, slots = pool.reserve(first * pool.granted, sum(new))
        assert pool.granted.tolist() == [1] * n and torch.equal(pool.block_tables, tables) and int(pool.free_count) == count
        left = [a * g for a, g in zip(new, granted)]
        assert pool.batch.query_starts.tolist() == [0] + np.cumsum(left).tolist()
        assert pool.batch.kv_lens.tolist() == [a + b for a, b in zip(held, left)]
        cache = filled(PagedKVCache.allocate(pages, 16, 1, 64, torch.float8_e4m3fn, scale_block=16))
        x = randn(rng, sum(new), 1, 64)
        cache.append(x, x, pool.batch)
        stored = {int(s) for s in slots.tolist() if s >= 0}
        assert len(stored) == sum(left)
        # the places of the tokens held before, whose codes may have been lowered, and those of the new ones
        pages_of = pool.block_tables.tolist()
        before = {16 * pages_of[r][i // 16] + i % 16 for r in range(n) if granted[r] for i in range(held[r])}
        changed = (cache.k.view(torch.uint8) != 0x38).any(-1).flatten().nonzero().flatten().tolist()
        assert set(changed) <= stored | before and stored <= set(changed) | before
