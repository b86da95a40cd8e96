"""The e4m3 cache with a scale for each block of tokens and KV head, on the GPU through the
Python API: the append against what its definition gives in 64 bits, the attention against
attention_oracle.py over the values that codes and scales stand for."""

import math

import numpy as np
import pytest

import attention_oracle as O
from test_gpu_attention import dev, inv_freq, kernel, randn

pytestmark = pytest.mark.gpu

LOW, HIGH = -100, 80


def exponents(t):
    import torch

    return t.view(torch.uint8).cpu().numpy().astype(np.int64) - 127


def least(top):
    """The least exponent with top <= 448 * 2^e, held to its range."""
    m, e = math.frexp(top)
    return min(HIGH, max(LOW, e - 9 + (m > 0.875))) if top > 0 else LOW


def codes64(t):
    """Codes of e4m3 pages as float64."""
    return t.float().cpu().numpy().astype(np.float64)


def e4m3(z):
    """float64 -> e4m3 -> float64, to nearest even (the values here are exact in float32)."""
    import torch

    return torch.from_numpy(z.astype(np.float32)).to(torch.float8_e4m3fn).float().numpy().astype(np.float64)


def phsd(t, layout):
    return t.permute(0, 2, 1, 3) if layout == "pshd" else t


def check_append(y, slack, before, after, old, new, b, block, what):
    """y [rows, heads, D] and its fp32 slack; codes and exponents before and after."""
    new_at = {}  # (page, block of the page) -> its request's first position there, rows by slot
    for i, r, p in O.rows_of(b):
        at = O.slot_of(b, r, p) if r is not None else None
        if at is not None:
            new_at.setdefault((at[0], at[1] // block), []).append((at[1] % block, i))
    want, bound, scale = before.copy(), np.zeros_like(before), old.copy()
    for (page, unit), rows in new_at.items():
        first = min(s for s, _ in rows)
        index = [i for _, i in rows]
        here = slice(unit * block, unit * block + first)
        for h in range(y.shape[1]):
            top, off = np.abs(y[index, h]).max(), slack[index, h].max()
            held = min(HIGH, max(LOW, old[page, h, unit])) if first else LOW
            fit = {max(held, least(max(0.0, top + d))) for d in (-off, 0.0, off)}  # fp32 may fall on the other side of a border
            assert new[page, h, unit] in fit, f"{what}: exponent {new[page, h, unit]} of page {page} head {h} block {unit}, not {fit}"
            e = int(new[page, h, unit])
            scale[page, h, unit] = e
            if e > held:  # kept codes: exactly one more rounding
                want[page, h, here] = e4m3(before[page, h, here] * 2.0 ** max(held - e, -200))
            for s, i in rows:
                z = np.clip(y[i, h] * 2.0 ** -e, -448, 448)
                want[page, h, unit * block + s] = z
                bound[page, h, unit * block + s] = np.maximum(O.E4M3 * np.abs(z), 2.0 ** -10) + slack[i, h] * 2.0 ** -e + 1e-6 * np.abs(z)
    assert np.array_equal(new, scale), f"{what}: scales of blocks without new tokens have changed"
    O.assert_within(after, want, bound, what)
    return new_at


CASES = [  # head_dim, KV heads, page, block, layout
    (64, 3, 16, 16, "phsd"), (64, 3, 64, 32, "pshd"), (128, 2, 32, 16, "pshd"), (128, 2, 128, 128, "phsd"), (256, 8, 64, 16, "phsd"),
    (256, 4, 256, 256, "pshd"), (512, 1, 64, 64, "phsd"), (512, 2, 16, 16, "pshd"),
]


@pytest.mark.parametrize("d,hk,page,block,layout", CASES)
def test_append(gpu_lib, d, hk, page, block, layout):
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(d + page + block)
    # a prompt, one token, none, several up to a page's end, more tokens than positions, blocks begun anew, 70 runs
    q_lens = [37, 1, 0, 5, 4, 300, 2] + [1] * 70
    kv_lens = [37, 1000, 20, 2 * page, 2, 411, page + 1] + [int(v) for v in rng.integers(1, 300, 70)]
    b = O.make_batch(rng, q_lens, kv_lens, page, padding=3)
    b["tables"][8, -(-kv_lens[8] // page) - 1] = b["num_pages"]  # absent: the first page number past the cache
    b["tables"][9, -(-kv_lens[9] // page) - 1] = -7
    shape = (b["num_pages"], hk, page, d) if layout == "phsd" else (b["num_pages"], page, hk, d)
    before = [(randn(rng, *shape).float() * 96).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    # some scales that stay, some that rise, and bytes past both ends
    held = [dev(rng.choice([0, 20, 60, 119, 120, 121, 122, 140, 250, 255], (b["num_pages"], hk, page // block)).astype(np.uint8)) for _ in range(2)]
    nq, rows = 2 * hk, b["rows"]
    x = randn(rng, rows, (nq + 2 * hk) * d) * 3
    q, k, v = (x[:, a * d:e * d].unflatten(1, (e - a, d)) for a, e in ((0, nq), (nq, nq + hk), (nq + hk, nq + 2 * hk)))
    w = (1 + 0.3 * randn(rng, d).float()).bfloat16()
    freq = inv_freq(d // 4)
    rope, kn, vn = A.Rope(dev(freq), d // 2), A.HeadNorm(w, 1e-5), A.HeadNorm(None, 1e-6)
    batch = O.device_batch(b)
    results = []
    for source, qq in ((v, q), (v, None), (k, q)):  # with q, without, values from the keys' columns
        pages, by = [t.clone() for t in before], [t.clone() for t in held]
        cache = A.PagedKVCache(*pages, *by, layout=layout)
        gq = cache.append(k, source, batch, rope=rope, k_norm=kn, v_norm=vn, q=qq, q_norm=kn if qq is not None else None)
        results.append((pages, by, gq))
    assert results[1][2] is None
    for i in (0, 1):
        assert torch.equal(results[0][0][i].view(torch.uint8), results[1][0][i].view(torch.uint8)) and torch.equal(results[0][1][i], results[1][1][i])
    pos, inside = np.zeros(rows, np.int64), np.zeros(rows, bool)
    for i, r, p in O.rows_of(b):
        pos[i], inside[i] = p, r is not None
    wq, qb = O.norm_rope(O.f64(q), pos, freq, d // 2, True, O.f64(w), 1e-5)
    wq[~inside] = 0
    for got in (results[0][2], results[2][2]):
        O.assert_within(O.f64(got), wq, qb, "q")
    wk = O.norm_rope(O.f64(k), pos, freq, d // 2, True, O.f64(w), 1e-5)
    for source, (pages, by, _) in ((v, results[0]), (k, results[2])):
        wv = O.norm_rope(O.f64(source), pos, norm=True, eps=1e-6)
        for i, (name, (y, bf16_bound)) in enumerate((("k", wk), ("v", wv))):
            slack = bf16_bound - O.BF16 * np.abs(y)
            check_append(y, slack, codes64(phsd(before[i], layout)), codes64(phsd(pages[i], layout)), exponents(held[i]), exponents(by[i]), b, block, name)


@pytest.mark.parametrize("d,pairs,distance", [(64, 32, 32), (128, 64, 1), (256, 128, 128), (256, 8, 64), (512, 64, 256), (512, 256, 1)])
def test_append_rotates_as_the_norms_do(gpu_lib, d, pairs, distance):
    """The q that the append writes is the q that qk_norm_rope writes, but for a product of the
    rotation that is fused into the sum in one and rounded in the other: two fp32 values within
    3 * 2^-24 of the head's largest, whose bf16 values are the same or neighbours (2^-7 apart)."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(d + pairs)
    b = O.make_batch(rng, [5, 1, 40], [5, 900, 63], 32, padding=2)
    q, k = randn(rng, b["rows"], 6, d), randn(rng, b["rows"], 2, d)
    rope, norm = A.Rope(dev(inv_freq(pairs)), distance), A.HeadNorm((1 + 0.2 * randn(rng, d).float()).bfloat16())
    cache = A.PagedKVCache.allocate(b["num_pages"], 32, 2, d, torch.float8_e4m3fn, scale_block=16)
    got = cache.append(k, k, O.device_batch(b), rope=rope, k_norm=norm, q=q, q_norm=norm)
    pos = np.zeros(b["rows"], np.int32)
    for i, r, p in O.rows_of(b):
        pos[i] = p
    want, _ = A.qk_norm_rope(q, None, dev(pos), rope, q_norm=norm)
    live = int(b["starts"][-1])
    g, w = got[:live].float(), want[:live].float()
    most = 2 * 3 * 2.0 ** -24 * w.abs().amax(-1, keepdim=True)  # a pair's norm is within sqrt(2) of its larger one
    assert bool(((g - w).abs() <= 2.0 ** -7 * torch.maximum(g.abs(), w.abs()) + most).all())
    assert int((g != w).sum()) <= g.numel() // 200 and bool((got[live:] == 0).all())
    inplace = q.clone()
    assert cache.append(k, k, O.device_batch(b), rope=rope, k_norm=norm, q=inplace, q_norm=norm, out_q=inplace) is inplace
    assert torch.equal(inplace, got)


def test_scales_follow_the_tokens(gpu_lib):
    """One token at a time: a louder one lifts its block's scale and its neighbours' codes follow,
    a block's first slot begins anew, and what lies behind the new tokens stays."""
    import torch

    from helios_amd import attention as A

    b = O.make_batch(np.random.default_rng(0), [1], [1], 32, width=2)
    cache = A.PagedKVCache.allocate(b["num_pages"], 32, 1, 64, torch.float8_e4m3fn, scale_block=16)
    cache.k.view(torch.uint8).fill_(0x35)
    cache.k_scale.view(torch.uint8).fill_(200)
    loud = [1.0, 448.0, 449.0, 3.0, 2.0 ** 20, 0.0] + [1.0] * 10 + [0.0, 2.0 ** -95, 2.0 ** -110, 1e38]
    values = []
    for n, v in enumerate(loud):
        b["kv_lens"][0] = n + 1
        x = torch.full((1, 1, 64), v, dtype=torch.bfloat16, device="cuda")
        values.append(float(x[0, 0, 0]))
        cache.append(x, x, O.device_batch(b))
        unit = n // 16
        page = int(b["tables"][0, 0])
        here = values[16 * unit:]
        e = exponents(cache.k_scale)[page, 0, unit]
        assert e == least(max(here)), (n, e)
        got = cache.k[page, 0, 16 * unit:n + 1, 5].float().cpu().numpy().astype(np.float64) * 2.0 ** float(e)
        # what the largest scale holds; half a step of each value, and under the least step of the
        # scale nothing is told apart
        here = np.minimum(here, 448 * 2.0 ** float(e))
        assert np.all(np.abs(got - here) <= np.maximum(O.E4M3 * np.abs(here), 2.0 ** -9 * 2.0 ** float(e))), (n, got, here)
        assert bool((cache.k.view(torch.uint8)[page, 0, n + 1:] == 0x35).all())


def test_append_of_infinities_and_nan(gpu_lib):
    """They have no say in the scale; infinities are stored as the largest code, NaN as NaN."""
    import torch

    from helios_amd import attention as A

    b = O.make_batch(np.random.default_rng(0), [3], [3], 16)
    k = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2] = float("inf"), float("-inf"), float("nan")
    cache = A.PagedKVCache.allocate(b["num_pages"], 16, 1, 64, torch.float8_e4m3fn, scale_block=16)
    cache.append(k, k, O.device_batch(b))
    page = int(b["tables"][0, 0])
    e = least(1.0)
    for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        got = t[page, 0, :3].float()
        assert exponents(s)[page, 0, 0] == e
        assert got[0, 0] == 448 and got[1, 1] == -448 and bool(got[2, 2].isnan()) and got[0, 5] == 2.0 ** -e


# ------------------------------------------------------------------ attention

def attend_case(rng, d, hq, hk, q_lens, kv_lens, page, block, window=0, padding=0, layout="phsd", spread=1.0, change=None, width=None,
                scale=None, span=3):
    import torch

    from helios_amd import attention as A

    b = O.make_batch(rng, q_lens, kv_lens, page, padding=padding, width=width)
    if change is not None:
        change(b)
    per = page // block
    shape = (b["num_pages"], hk, page, d)
    used = np.zeros((b["num_pages"], page), bool)
    for r, kv in enumerate(kv_lens):
        for p in range(kv):
            at = O.slot_of(b, r, p)
            if at is not None:
                used[at] = True
    hide = dev(~used)[:, None, :, None].expand(shape)
    nan = torch.full((), float("nan"), device="cuda")
    # scales of the blocks in use differ; everything outside the requests' tokens is NaN, and its scales anything
    free = ~used.reshape(b["num_pages"], per, block).any(-1)[:, None, :]
    codes, bytes_ = [], []
    for _ in range(2):
        e = rng.integers(127 - 6 - span, 127 - 6 + span, (b["num_pages"], hk, per))
        e = np.where(free, rng.integers(0, 256, e.shape), e).astype(np.uint8)
        bytes_.append(dev(e).view(torch.float8_e8m0fnu))
        by = torch.exp2(dev(np.clip(e, 27, 207).astype(np.float32) - 127)).repeat_interleave(block, 2)[..., None]
        x = (randn(rng, *shape).float() / by).clamp(-448, 448)
        codes.append(torch.where(hide, nan, x).to(torch.float8_e4m3fn))
    if layout == "pshd":
        pages = [t.permute(0, 2, 1, 3).contiguous() for t in codes]
        # scales in an order of their own too: heads before pages
        bytes_ = [t.view(torch.uint8).permute(1, 0, 2).contiguous().permute(1, 0, 2).view(torch.float8_e8m0fnu) for t in bytes_]
    else:
        pages = codes
    cache = A.PagedKVCache(*pages, *bytes_, layout=layout)
    batch = O.device_batch(b)
    q = (randn(rng, b["rows"], hq + 1, d) * spread)[:, :hq]  # a row stride of its own
    scale = d ** -0.5 if scale is None else scale
    out, lse = cache.attend(q, batch, scale=scale, window=window, return_lse=True)
    again, lse2 = cache.attend(q, batch, scale=scale, window=window, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "two runs differ"
    wide = [O.f64(t) * 2.0 ** np.repeat(np.clip(exponents(s), LOW, HIGH), block, 2)[..., None] for t, s in zip(codes, bytes_)]
    want, bound, wl, lb = O.attend(O.f64(q), *wide, b, scale, window)
    O.assert_within(O.f64(out), want, bound, "out")
    O.assert_within(O.f64(lse), wl, lb, "lse")
    for k in (1, 2):  # each kernel, whatever the call's size
        with kernel(k):
            pinned, pinned_lse = cache.attend(q, batch, scale=scale, window=window, return_lse=True)
        O.assert_within(O.f64(pinned), want, bound, f"out, kernel {k}")
        O.assert_within(O.f64(pinned_lse), wl, lb, f"lse, kernel {k}")
    return out, lse, b, cache, batch, q, wide


SHAPES = [(64, 8, 2), (64, 40, 1), (128, 12, 4), (128, 8, 8), (256, 16, 8), (256, 20, 1), (512, 16, 1), (512, 4, 2)]


@pytest.mark.parametrize("d,hq,hk", SHAPES)
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32)])
def test_decode_lengths(gpu_lib, d, hq, hk, page, block):
    """One new token each, contexts around every boundary of groups, tiles, blocks and pages."""
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 0, 300]
    attend_case(np.random.default_rng(d + hq), d, hq, hk, [1] * len(kv), kv, page, block)


@pytest.mark.parametrize("d,hq,hk", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 37])
def test_chunks(gpu_lib, d, hq, hk, window):
    attend_case(np.random.default_rng(7 * d + hq + window), d, hq, hk, [33, 1, 0, 8, 70, 2], [33, 90, 50, 41, 130, 2], 32, 16, window=window, padding=2)


@pytest.mark.parametrize("d,hq,hk", [(64, 8, 2), (128, 12, 4), (256, 16, 8), (512, 16, 1)])
def test_long_contexts(gpu_lib, d, hq, hk):
    """Contexts of many windows of groups: cut ranges and their join, wide ranges of scores and scales."""
    rng = np.random.default_rng(d)
    attend_case(rng, d, hq, hk, [1, 3], [5003, 777], 64, 16, spread=4.0, span=4)
    attend_case(rng, d, hq, hk, [2], [4000], 128, 128, window=1024, layout="pshd")
    attend_case(rng, d, hq, hk, [70, 1, 0, 9, 1], [3100, 2500, 7, 2049, 1], 16, 16, padding=1)
    attend_case(rng, d, hq, hk, [67], [4500], 64, 32, window=1500, spread=2.0)


@pytest.mark.parametrize("d,hq,hk", [(64, 6, 2), (128, 4, 4), (256, 16, 8), (512, 16, 1)])
@pytest.mark.parametrize("q_len,kv_len,window", [(257, 257, 0), (200, 901, 0), (300, 700, 64), (129, 640, 100)])
def test_prefill_tiles(gpu_lib, d, hq, hk, q_len, kv_len, window):
    attend_case(np.random.default_rng(q_len), d, hq, hk, [q_len], [kv_len], 64, 16, window=window)


def test_pages_past_four_gigabytes(gpu_lib):
    """The same tokens in near pages and in pages whose bytes lie past 32 bits, the same page twice in a
    table: the same codes, scales and outputs."""
    import torch

    from helios_amd import attention as A

    d, page, block, pages = 512, 64, 32, 140000
    far = A.PagedKVCache.allocate(pages, page, 1, d, torch.float8_e4m3fn, scale_block=block)
    near = A.PagedKVCache.allocate(8, page, 1, d, torch.float8_e4m3fn, scale_block=block)
    assert far.k.numel() > 1 << 32
    rng = np.random.default_rng(3)
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    lens, results = [150, 300], []
    x = randn(rng, sum(lens), 3, d) * 2
    for cache, first in ((near, 0), (far, pages - 8)):
        tables = np.array([[5, 1, 7, 7, 7], [0, 2, 3, 4, 6]]) + first
        batch = A.KVBatch(ints([0, 150, 450]), ints(lens), ints(tables.tolist()))
        cache.append(x[:, 1:2], x[:, 2:], batch)
        outs = []
        for starts, kv, window in (([0, 1, 2], lens, 0), ([0, 1, 2], lens, 100), ([0, 150, 450], lens, 0), ([0, 1, 2], [320, 300], 0)):
            q = randn(np.random.default_rng(4), starts[-1], 16, d)
            # the last: the first request reads its last page three times over
            outs.append(cache.attend(q, A.KVBatch(ints(starts), ints(kv), ints(tables.tolist())), window=window))
        at = slice(first, first + 8)
        results.append(outs + [t[at].view(torch.uint8) for t in (cache.k_scale, cache.v_scale)] +
                       [cache.k[at][tables[r, p // page] - first, 0, p % page].view(torch.uint8) for r in (0, 1) for p in (0, 63, 64, lens[r] - 1)])
    unused = [5, 1, 0, 2, 3, 4]  # whose blocks are all written
    for i, (a, b) in enumerate(zip(*results)):
        a, b = (t[unused] if t.shape[:2] == (8, 1) and t.dtype == torch.uint8 else t for t in (a, b))
        if i == 3:  # slots past the 150 tokens are whatever the pages held
            a, b = a[1], b[1]
        assert torch.equal(a, b), i


def test_many_requests_and_absent_pages(gpu_lib):
    import torch

    rng = np.random.default_rng(5)
    q_lens = [int(v) for v in rng.choice([0, 1, 1, 1, 2, 5, 20], 150)] + [130, 1]
    kv_lens = [a + int(rng.integers(0, 60)) for a in q_lens[:-1]] + [3001]
    attend_case(rng, 256, 4, 2, q_lens, kv_lens, 16, 16, padding=4)

    def change(b):
        b["tables"][2, :] = -1
        b["tables"][3, 0] = b["num_pages"]

    for d, hq, hk in ((256, 16, 8), (512, 16, 1)):
        out, lse, *_ = attend_case(rng, d, hq, hk, [1, 9, 5, 20], [0, 4, 60, 60], 16, 16, padding=3, change=change)
        for row in [0] + list(range(1, 6)) + list(range(10, 15)) + list(range(35, 38)):
            assert bool((out[row] == 0).all()) and bool((lse[row] == float("-inf")).all()), row
        assert bool(torch.isfinite(lse[6:10]).all()) and bool(torch.isfinite(lse[15:35]).all())


@pytest.mark.parametrize("d,hq,hk,q_len,kv_len,window", [(256, 4, 2, 40, 40, 0), (512, 16, 1, 8, 300, 0), (64, 4, 4, 150, 400, 50), (128, 4, 2, 300, 300, 0)])
def test_nan_in_hidden_places(gpu_lib, d, hq, hk, q_len, kv_len, window):
    """A token's NaN value reaches the rows that see it and no other."""
    import torch

    *_, b, cache, batch, q, (k64, v64) = attend_case(np.random.default_rng(q_len), d, hq, hk, [q_len], [kv_len], 32, 16, window=window)
    first = kv_len - q_len
    for p, h, e in [(first + q_len // 2, 0, 1), (kv_len - 1, hk - 1, d - 1), (max(0, first - max(0, window - 5)), 0, 2)]:
        page, slot = O.slot_of(b, 0, p)
        cache.v.view(torch.uint8)[page, h, slot, e] = 0x7F
        v64[page, h, slot, e] = float("nan")
    want, bound, wl, lb = O.attend(O.f64(q), k64, v64, b, d ** -0.5, window)
    for k in (0, 1, 2):
        with kernel(k):
            out, lse = cache.attend(q, batch, window=window, return_lse=True)
        O.assert_within(O.f64(out), want, bound, f"out, kernel {k}")
        O.assert_within(O.f64(lse), wl, lb, f"lse, kernel {k}")


def test_extreme_scales(gpu_lib):
    """Blocks at both ends of the scales' range: the softmax and the sums stay finite."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(3)
    for d, rows in ((64, 1), (256, 70), (512, 12)):
        b = O.make_batch(rng, [rows], [rows + 40], 32)
        cache = A.PagedKVCache.allocate(b["num_pages"], 32, 1, d, torch.float8_e4m3fn, scale_block=16)
        for t in (cache.k, cache.v):
            t.copy_((randn(rng, *t.shape).float() * 96).clamp(-448, 448).to(torch.float8_e4m3fn))
        cache.k_scale.view(torch.uint8).copy_(dev(rng.choice([0, 27, 117, 118], tuple(cache.k_scale.shape)).astype(np.uint8)))
        cache.v_scale.view(torch.uint8).copy_(dev(rng.choice([0, 5, 27, 100, 245, 255], tuple(cache.v_scale.shape)).astype(np.uint8)))
        q = randn(rng, rows, 2, d)
        wide = [O.f64(t) * 2.0 ** np.repeat(np.clip(exponents(s), LOW, HIGH), 16, 2)[..., None] for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
        want, bound, _, _ = O.attend(O.f64(q), *wide, b, d ** -0.5)
        for k in (1, 2):
            with kernel(k):
                out = cache.attend(q, O.device_batch(b))
            O.assert_within(O.f64(out), want, bound, f"kernel {k}")


def test_refusals_of_the_cache(gpu_lib):
    import torch

    from helios_amd import attention as A

    k = torch.zeros(4, 2, 64, 128, device="cuda").to(torch.float8_e4m3fn)
    s = torch.zeros(4, 2, 4, dtype=torch.uint8, device="cuda")
    A.PagedKVCache(k, k, s, s)
    for scales in ((s, 1.0), (s, s[:, :, :2]), (s[:3], s[:3]), (s[:, :1], s[:, :1]), (s.float(), s.float()), (s[:, :, :3], s[:, :, :3]), (s.cpu(), s.cpu()),
                   (s.new_zeros(4, 2, 8)[:, :, ::2],) * 2, (s, s.new_zeros(4, 4, 2).transpose(1, 2))):
        with pytest.raises(A.Gemma4Error):
            A.PagedKVCache(k, k, *scales)
    with pytest.raises(A.Gemma4Error):
        A.PagedKVCache(k.bfloat16(), k.bfloat16(), s, s)
    for kw in (dict(scale_block=48), dict(scale_block=-16), dict(scale_block=16, k_scale=0.5)):
        with pytest.raises(A.Gemma4Error):
            A.PagedKVCache.allocate(4, 64, 2, 128, torch.float8_e4m3fn, **kw)
    with pytest.raises(A.Gemma4Error):
        A.PagedKVCache.allocate(4, 64, 2, 128, torch.bfloat16, scale_block=16)
    # a block that the library does not take is refused by the call
    cache = A.PagedKVCache.allocate(4, 64, 2, 128, torch.float8_e4m3fn, scale_block=8)
    b = O.device_batch(O.make_batch(np.random.default_rng(0), [1], [1], 64))
    with pytest.raises(A.Gemma4Error, match="block"):
        cache.attend(torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda"), b)
