"""Pages given out and taken back on the GPU, against the same done one by one on the host."""

import numpy as np
import pytest

from pooled_streams import streams  # noqa: F401

pytestmark = pytest.mark.gpu


class Host:
    """A pool's state on the host, and its two calls as they are defined."""

    def __init__(self, num_pages, page, requests, width, rng=None):
        order = np.arange(num_pages)[::-1].copy() if rng is None else rng.permutation(num_pages)
        self.page, self.num_pages, self.width = page, num_pages, width
        self.free = [int(p) for p in order]
        self.lens = np.zeros(requests, np.int64)
        self.tables = np.full((requests, width), -1, np.int64)

    def there(self, entry):
        return 0 <= entry < self.num_pages

    def reserve(self, new, rows):
        starts, kv, granted, needs = [0], [], [], 0
        positions, slots = np.zeros(rows, np.int64), np.full(rows, -1, np.int64)
        count = len(self.free)
        taken = 0
        for r, n in enumerate(np.clip(new, 0, 1 << 24)):
            held = int(np.clip(self.lens[r], 0, self.width * self.page))
            first, end = -(-held // self.page), -(-(held + int(n)) // self.page)
            fits = end <= self.width
            absent = [j for j in range(first, end) if fits and not self.there(self.tables[r, j])]
            needs += len(absent)
            ok = fits and (not absent or needs <= count)
            if ok:
                for j in absent:
                    self.tables[r, j] = self.free[count - 1 - taken]
                    taken += 1
            granted.append(int(ok))
            kv.append(held + int(n))
            for i in range(int(n)):
                row, p = starts[-1] + i, held + i
                if row < rows:
                    positions[row] = p
                    entry = self.tables[r, p // self.page] if p // self.page < self.width else -1
                    slots[row] = entry * self.page + p % self.page if self.there(entry) else -1
            starts.append(starts[-1] + int(n))
        del self.free[count - taken:]
        return starts, kv, granted, positions, slots

    def release(self, lens, window=0):
        freed = []
        for r, n in enumerate(lens):
            n = int(np.clip(n, 0, self.width * self.page))
            lo = max(0, n - window + 1) // self.page if window else 0
            for j in range(self.width):
                if self.there(self.tables[r, j]) and (j < lo or j >= -(-n // self.page)):
                    freed.append(int(self.tables[r, j]))
                    self.tables[r, j] = -1
            self.lens[r] = n
        self.free += freed[::-1]


def device(host, stride=None):
    import torch

    from helios_amd import PagePool

    free = torch.full((host.num_pages,), -99, dtype=torch.int32)
    free[:len(host.free)] = torch.tensor(host.free, dtype=torch.int32)
    wide = torch.full((len(host.lens), stride or host.width), -5, dtype=torch.int32)
    wide[:, :host.width] = torch.from_numpy(host.tables)
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    return PagePool(free.cuda(), ints([len(host.free)]), ints(host.lens.tolist()), wide.cuda()[:, :host.width], host.page)


def same(pool, host):
    assert pool.free_count.tolist() == [len(host.free)]
    assert pool.free_pages[:len(host.free)].tolist() == host.free
    assert np.array_equal(pool.block_tables.cpu().numpy(), host.tables)
    assert pool.lens.tolist() == host.lens.tolist()


def reserve_both(pool, host, new, rows):
    import torch

    got = pool.reserve(torch.tensor(new, dtype=torch.int32).cuda(), rows)
    starts, kv, granted, positions, slots = host.reserve(np.array(new), rows)
    assert pool.batch.query_starts.tolist() == starts and pool.batch.kv_lens.tolist() == kv
    assert pool.granted.tolist() == granted
    assert np.array_equal(got[0].cpu().numpy(), positions) and np.array_equal(got[1].cpu().numpy(), slots)
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.int64
    same(pool, host)
    return granted


def release_both(pool, host, lens, window=0):
    import torch

    pool.release(torch.tensor(lens, dtype=torch.int32).cuda(), window=window)
    host.release(lens, window)
    same(pool, host)


# requests, page, width, pages: one to several workgroups' worth of requests, rows and entries
POOLS = [(1, 16, 1, 3), (3, 16, 5, 11), (8, 64, 130, 400), (70, 32, 40, 1500), (96, 16, 300, 9000), (1030, 16, 6, 3500), (2100, 16, 9, 9000)]


@pytest.mark.parametrize("requests,page,width,num_pages", POOLS)
@pytest.mark.parametrize("window", [0, 1, 50])
def test_steps_of_a_server(gpu_lib, requests, page, width, num_pages, window):
    """Prompts, drafts, refusals, requests that end and begin, a window that moves on."""
    rng = np.random.default_rng(requests + window)
    host = Host(num_pages, page, requests, width, rng)
    pool = device(host, stride=width + 3)
    most = page * width
    for step in range(8):
        new = np.where(rng.random(requests) < 0.6, rng.choice([0, 1, 5], requests), rng.integers(0, most // 3 + 2, requests))
        if step == 5:
            new = rng.integers(-3, most + 40, requests)  # negative ones, and more than a table holds
        rows = int(np.clip(new, 0, None).sum()) + 3
        granted = np.array(reserve_both(pool, host, new.tolist(), rows))
        kept = host.lens + np.where(granted == 1, (np.clip(new, 0, None) * rng.random(requests)).astype(np.int64), 0)
        kept = np.where(rng.random(requests) < 0.2, 0, kept)
        release_both(pool, host, kept.tolist(), window)


def test_release_after_reserve_restores_the_order(gpu_lib):
    rng = np.random.default_rng(2)
    for requests, width in ((5, 20), (200, 100)):
        host = Host(requests * 10, 16, requests, width, rng)
        pool = device(host)
        reserve_both(pool, host, rng.integers(0, 40, requests).tolist(), 10)
        release_both(pool, host, host.lens.tolist())
        first = list(host.free)
        reserve_both(pool, host, rng.integers(0, 70, requests).tolist(), 10)
        release_both(pool, host, [0] * requests)
        assert host.free == first


def test_pages_run_out(gpu_lib):
    """The first that does not fit gets nothing, nor do those behind it that need pages; a request
    too long for its table takes none from the others; a second reserve finds what is there."""
    host = Host(6, 16, 5, 4)
    pool = device(host)
    assert reserve_both(pool, host, [40, 100, 16, 0, 30], 190) == [1, 0, 1, 1, 1]
    assert reserve_both(pool, host, [40, 100, 16, 0, 30], 190) == [1, 0, 1, 1, 1]  # the same tokens again: no page is lost
    # 3 + 1 + 2 pages are given out, none is left: only what needs no further one is granted
    assert reserve_both(pool, host, [64, 1, 17, 1, 30], 0) == [0, 0, 0, 0, 1]
    release_both(pool, host, [0, 0, 16, 0, 0])
    assert reserve_both(pool, host, [0, 0, 0, 0, 0], 2) == [1] * 5


def test_rows_without_the_map(gpu_lib):
    import torch

    from helios_amd import PagePool

    pool = PagePool.allocate(20, 16, 3, 8)
    assert pool.reserve(torch.tensor([5, 0, 33], dtype=torch.int32).cuda()) == (None, None)
    assert pool.block_tables.tolist() == [[0] + [-1] * 7, [-1] * 8, [1, 2, 3] + [-1] * 5]
    assert pool.free_count.tolist() == [16] and pool.batch.query_starts.tolist() == [0, 5, 5, 38]
    # a longer map than there are rows, a shorter one, none
    p, s = pool.reserve(torch.tensor([5, 0, 33], dtype=torch.int32).cuda(), 40)
    assert p.tolist() == list(range(5)) + list(range(33)) + [0, 0] and s.tolist()[5:8] == [16, 17, 18] and s.tolist()[38:] == [-1, -1]
    p, s = pool.reserve(torch.tensor([5, 0, 33], dtype=torch.int32).cuda(), 6)
    assert p.tolist() == [0, 1, 2, 3, 4, 0] and s.tolist() == [0, 1, 2, 3, 4, 16]
    p, s = pool.reserve(torch.tensor([5, 0, 33], dtype=torch.int32).cuda(), 0)
    assert p.shape == (0,) and s.shape == (0,)


def test_lengths_and_counts_past_their_ends(gpu_lib):
    """Device arrays that hold nonsense are clamped: nothing is read or written out of place."""
    import torch

    host = Host(8, 16, 3, 4)
    pool = device(host)
    reserve_both(pool, host, [16, 16, 16], 48)
    pool.lens.copy_(torch.tensor([-5, 2 ** 31 - 1, 1000]))
    host.lens[:] = [-5, 2 ** 31 - 1, 1000]
    reserve_both(pool, host, [3, 3, 2 ** 31 - 1], 100)
    release_both(pool, host, [-7, 2 ** 31 - 1, 0])
    pool.free_count.fill_(2 ** 31 - 1)  # more free pages than there are
    pool.reserve(torch.tensor([0, 0, 0], dtype=torch.int32).cuda())
    assert pool.free_count.tolist() == [8]
    pool.free_count.fill_(-3)
    pool.reserve(torch.tensor([16, 0, 0], dtype=torch.int32).cuda())
    assert pool.granted.tolist() == [0, 1, 1] and pool.free_count.tolist() == [0]


@pytest.mark.parametrize("requests,width", [(6, 40), (90, 200)])
def test_captured_steps(gpu_lib, requests, width, streams):
    """Replays of a captured reserve and release follow what the device arrays hold."""
    import torch

    rng = np.random.default_rng(requests)
    host = Host(requests * width // 2, 16, requests, width, rng)
    pool = device(host)
    new, kept = (torch.zeros(requests, dtype=torch.int32, device="cuda") for _ in range(2))
    rows = 6000
    stream = streams()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool.reserve(new, rows)
        pool.release(kept, window=100)  # takes the stream's scratch memory before the capture
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        positions, slots = pool.reserve(new, rows)
        pool.release(kept, window=100)
    for step in range(5):
        n = rng.integers(0, 60, requests)
        k = host.lens + n // 2
        new.copy_(torch.from_numpy(n).int())
        kept.copy_(torch.from_numpy(k).int())
        graph.replay()
        torch.cuda.synchronize()
        starts, kv, granted, want, want_slots = host.reserve(n, rows)
        host.release(k, 100)
        assert np.array_equal(positions.cpu().numpy(), want) and np.array_equal(slots.cpu().numpy(), want_slots)
        assert pool.batch.query_starts.tolist() == starts and pool.granted.tolist() == granted
        same(pool, host)
        torch.zeros(1000, device="cuda").sum().item()  # work of the program's own between replays


@pytest.mark.parametrize("requests,width", [(5, 40), (90, 200)])
def test_release_of_the_lens_held(gpu_lib, requests, width, streams):
    """pool.release(pool.lens) gives back what a reserve took, and with a window what is behind it."""
    import torch

    rng = np.random.default_rng(width)
    host = Host(requests * width, 16, requests, width, rng)
    pool = device(host)
    stream = streams()
    for window in (0, 40, 0):
        n = rng.integers(1, 16 * width // 4, requests)
        reserve_both(pool, host, n, 50)
        release_both(pool, host, (host.lens + n).tolist())
        reserve_both(pool, host, np.full(requests, 33), 50)
        stream.wait_stream(torch.cuda.current_stream())
        pool.release(pool.lens, window=window, stream=stream)
        stream.synchronize()
        host.release(host.lens.tolist(), window)
        same(pool, host)


def test_arrays_that_overlap(gpu_lib):
    """A pool's own arrays as arguments: read where that is sound, else refused."""
    import torch

    from helios_amd import Gemma4Error, PagePool

    pool = PagePool.allocate(9, 16, 2, 3)
    pool.release(torch.tensor([5, 17], dtype=torch.int32, device="cuda"))
    for bad in (pool.batch.kv_lens, pool.batch.query_starts[:2], pool.batch.query_starts[1:], pool.granted, pool.block_tables.view(-1)[2:4]):
        with pytest.raises(Gemma4Error, match="overlap"):
            pool.reserve(bad)
    for bad in (pool.free_pages[3:5], pool.block_tables[1, :2]):
        with pytest.raises(Gemma4Error, match="overlap"):
            pool.release(bad)
    pool.reserve(pool.lens, 4)  # as many again
    assert pool.batch.kv_lens.tolist() == [10, 34] and pool.batch.query_starts.tolist() == [0, 5, 22]


def test_refusals(gpu_lib):
    import torch

    from helios_amd import Gemma4Error, PagePool

    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for args in ((ints(4).long(), ints(1), ints(2), ints(2, 3), 16), (ints(4), ints(2), ints(2), ints(2, 3), 16), (ints(4), ints(1), ints(2), ints(3, 3), 16),
                 (ints(4), ints(1), ints(2), ints(2, 3, 1), 16), (ints(4), ints(1), ints(2), ints(2, 6)[:, ::2], 16), (ints(4), ints(1), ints(2), ints(2, 3), 0),
                 (ints(4), ints(1).cpu(), ints(2), ints(2, 3), 16), (ints(8)[::2], ints(1), ints(2), ints(2, 3), 16)):
        with pytest.raises(Gemma4Error):
            PagePool(*args)
    pool = PagePool.allocate(4, 16, 2, 3)
    for bad in (ints(3), ints(2).long(), ints(2).cpu(), ints(2, 1)):
        with pytest.raises(Gemma4Error):
            pool.reserve(bad)
        with pytest.raises(Gemma4Error):
            pool.release(bad)
    for rows in (-1, 1 << 24):
        with pytest.raises(Gemma4Error):
            pool.reserve(ints(2), rows)
    for window in (-1, (1 << 30) + 1):
        with pytest.raises(Gemma4Error):
            pool.release(ints(2), window=window)
    with pytest.raises(Gemma4Error, match="page_size"):
        PagePool.allocate(4, 24, 2, 3).release(ints(2))
