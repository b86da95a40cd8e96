"""Head norms with rotation, the append to a paged cache and the attention over it, on the
GPU through the Python API, against the 64-bit implementations and bounds of
attention_oracle.py."""

import contextlib
import math

import numpy as np
import pytest

import attention_oracle as O

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def randn(rng, *shape):
    import torch

    return dev(rng.standard_normal(shape).astype(np.float32), torch.bfloat16)


def inv_freq(pairs, base=1e4):
    return (base ** (-np.arange(pairs) / pairs)).astype(np.float32)


@contextlib.contextmanager
def kernel(k):
    from helios_amd import attention as A

    before = A.set_attention_kernel(k)
    try:
        yield
    finally:
        A.set_attention_kernel(before)


# ------------------------------------------------------------------ norm and rotation

ROPES = [  # head_dim, pairs, distance
    (64, 32, 32), (64, 16, 16), (64, 32, 1), (128, 64, 64), (128, 32, 32), (128, 8, 1), (256, 128, 128), (256, 64, 64),
    (256, 128, 1), (512, 64, 256), (512, 256, 256), (512, 8, 8), (512, 24, 120),
]


@pytest.mark.parametrize("d,pairs,distance", ROPES)
@pytest.mark.parametrize("rows", [1, 3, 600])
def test_norm_rope(gpu_lib, d, pairs, distance, rows):
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(d + pairs + rows)
    nq, nk = (5, 2) if rows < 600 else (3, 1)
    x = randn(rng, rows, (nq + nk + 1) * d) * 3  # heads of a fused row, with columns left over
    q, k = x[:, :nq * d].unflatten(1, (nq, d)), x[:, nq * d:(nq + nk) * d].unflatten(1, (nk, d))
    pos = rng.integers(-5, 1 << 17, rows).astype(np.int32)
    pos[-1] = 2 ** 31 - 1
    freq = inv_freq(pairs)
    w = (1 + 0.3 * randn(rng, d).float()).bfloat16()
    rope = A.Rope(dev(freq), distance)
    gq, gk = A.qk_norm_rope(q, k, dev(pos), rope, q_norm=A.HeadNorm(w, 1e-5), k_norm=A.HeadNorm(None, 1e-6))
    want, bound = O.norm_rope(O.f64(q), pos, freq, distance, True, O.f64(w), 1e-5)
    O.assert_within(O.f64(gq), want, bound, "q")
    want, bound = O.norm_rope(O.f64(k), pos, freq, distance, True, None, 1e-6)
    O.assert_within(O.f64(gk), want, bound, "k")
    # rotation alone, norm alone, neither
    g, none = A.qk_norm_rope(q, None, dev(pos), rope)
    assert none is None
    want, bound = O.norm_rope(O.f64(q), pos, freq, distance)
    O.assert_within(O.f64(g), want, bound, "rotation")
    g, _ = A.qk_norm_rope(q, None, None, None, q_norm=A.HeadNorm(w))
    want, bound = O.norm_rope(O.f64(q), pos, norm=True, weight=O.f64(w))
    O.assert_within(O.f64(g), want, bound, "norm")
    g, _ = A.qk_norm_rope(q, None, None)
    assert torch.equal(g, q)
    # in place, the columns of no head untouched
    y = x.clone()
    yq, yk = y[:, :nq * d].unflatten(1, (nq, d)), y[:, nq * d:(nq + nk) * d].unflatten(1, (nk, d))
    A.qk_norm_rope(yq, yk, dev(pos), rope, q_norm=A.HeadNorm(w, 1e-5), k_norm=A.HeadNorm(None, 1e-6), out_q=yq, out_k=yk)
    assert torch.equal(yq, gq) and torch.equal(yk, gk) and torch.equal(y[:, (nq + nk) * d:], x[:, (nq + nk) * d:])


def test_norm_of_zeros_and_no_rows(gpu_lib):
    import torch

    from helios_amd import attention as A

    z = torch.zeros(2, 3, 256, dtype=torch.bfloat16, device="cuda")
    g, _ = A.qk_norm_rope(z, None, None, q_norm=A.HeadNorm(None, 1e-6))
    assert bool((g == 0).all())
    g, k = A.qk_norm_rope(z[:0], z[:0], dev(np.zeros(0, np.int32)), A.Rope(dev(inv_freq(8))))
    assert g.shape == (0, 3, 256) and k.shape == (0, 3, 256)


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("d,hk,page,layout,kind", [
    (64, 3, 16, "phsd", "bf16"), (128, 2, 32, "pshd", "bf16"), (256, 8, 64, "phsd", "bf16"), (512, 1, 128, "pshd", "bf16"),
    (64, 3, 64, "pshd", "e4m3"), (128, 2, 16, "phsd", "e4m3"), (256, 8, 32, "phsd", "e4m3"), (512, 1, 16, "phsd", "e4m3"),
])
def test_append(gpu_lib, d, hk, page, layout, kind):
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(d + page)
    # a prompt, one token, none, several up to a page's end, more tokens than positions, 70 runs
    q_lens = [37, 1, 0, 5, 4] + [1] * 70
    kv_lens = [37, 1000, 20, 2 * page, 2] + [int(v) for v in rng.integers(1, 300, 70)]
    b = O.make_batch(rng, q_lens, kv_lens, page, padding=3)
    b["tables"][6, -(-kv_lens[6] // page) - 1] = b["num_pages"]  # absent: the first page number past the cache
    b["tables"][7, -(-kv_lens[7] // page) - 1] = -7
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    shape = (b["num_pages"], hk, page, d) if layout == "phsd" else (b["num_pages"], page, hk, d)
    before = [randn(rng, *shape).to(dtype) for _ in range(2)]
    scales = (1.0, 1.0) if kind == "bf16" else (0.3, 0.01)
    nq, rows = 2 * hk, b["rows"]
    x = randn(rng, rows, (nq + 2 * hk) * d)
    q, k, v = (x[:, a * d:e * d].unflatten(1, (e - a, d)) for a, e in ((0, nq), (nq, nq + hk), (nq + hk, nq + 2 * hk)))
    w = (1 + 0.3 * randn(rng, d).float()).bfloat16()
    freq = inv_freq(d // 4)
    rope, kn, vn = A.Rope(dev(freq), d // 2), A.HeadNorm(w, 1e-5), A.HeadNorm(None, 1e-6)
    batch = O.device_batch(b)
    results = []
    for source, qq in ((v, q), (v, None), (k, q)):  # with q, without, values from the keys' columns
        pages = [t.clone() for t in before]
        cache = A.PagedKVCache(*pages, *scales, layout=layout)
        gq = cache.append(k, source, batch, rope=rope, k_norm=kn, v_norm=vn, q=qq, q_norm=kn if qq is not None else None)
        results.append((pages, gq))
    assert results[1][1] is None
    assert torch.equal(results[0][0][0].view(torch.uint8), results[1][0][0].view(torch.uint8))
    pos, inside = np.zeros(rows, np.int64), np.zeros(rows, bool)
    for i, r, p in O.rows_of(b):
        pos[i], inside[i] = p, r is not None
    wq, qb = O.norm_rope(O.f64(q), pos, freq, d // 2, True, O.f64(w), 1e-5)
    wq[~inside] = 0
    for got in (results[0][1], results[2][1]):
        O.assert_within(O.f64(got), wq, qb, "q")
    wk = O.norm_rope(O.f64(k), pos, freq, d // 2, True, O.f64(w), 1e-5)
    for source, (pages, _) in ((v, results[0]), (k, results[2])):
        wv = O.norm_rope(O.f64(source), pos, norm=True, eps=1e-6)
        for (y, slack), old, new, scale in ((wk, before[0], pages[0], scales[0]), (wv, before[1], pages[1], scales[1])):
            want, bound = O.f64(old), np.zeros(old.shape)
            z, zb = O.stored(y, slack, None if kind == "bf16" else scale)
            if layout == "pshd":
                want, bound = want.transpose(0, 2, 1, 3), bound.transpose(0, 2, 1, 3)
            stores = 0
            for i, r, p in O.rows_of(b):
                at = O.slot_of(b, r, p) if r is not None else None
                if at is not None:
                    want[at[0], :, at[1]], bound[at[0], :, at[1]] = z[i], zb[i]
                    stores += 1
            assert stores == sum(q_lens) - 2 - 2  # two absent pages, two rows before position 0
            got = O.f64(new)
            O.assert_within(got.transpose(0, 2, 1, 3) if layout == "pshd" else got, want, bound, "pages")


def test_append_saturates_and_keeps_nan(gpu_lib):
    import torch

    from helios_amd import attention as A

    b = O.make_batch(np.random.default_rng(0), [3], [3], 16)
    k = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2] = 1e30, float("-inf"), float("nan")
    cache = A.PagedKVCache.allocate(b["num_pages"], 16, 1, 64, torch.float8_e4m3fn, 0.5, 0.25)
    cache.append(k, k, O.device_batch(b))
    page = int(b["tables"][0, 0])
    for t, one in ((cache.k, 2.0), (cache.v, 4.0)):
        got = t[page, 0, :3].float()
        assert got[0, 0] == 448 and got[1, 1] == -448 and bool(got[2, 2].isnan()) and got[0, 5] == one


# ------------------------------------------------------------------ attention

def attend_case(rng, d, hq, hk, q_lens, kv_lens, page, kind="bf16", window=0, padding=0, layout="phsd", scale=None, spread=1.0,
                change=None, width=None):
    """Runs one batch and checks out and lse; returns what the call gave and its inputs."""
    import torch

    from helios_amd import attention as A

    b = O.make_batch(rng, q_lens, kv_lens, page, padding=padding, width=width)
    if change is not None:
        change(b)
    scales = (1.0, 1.0) if kind == "bf16" else (0.5, 0.125)
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    shape = (b["num_pages"], hk, page, d)
    k, v = ((randn(rng, *shape).float() / s).to(dtype) for s in scales)
    # everything outside the requests' tokens is NaN
    used = np.zeros((b["num_pages"], page), bool)
    for r, kv in enumerate(kv_lens):
        for p in range(kv):
            at = O.slot_of(b, r, p)
            if at is not None:
                used[at] = True
    hide = dev(~used)[:, None, :, None].expand(shape)
    k, v = (torch.where(hide, torch.full((), float("nan"), device="cuda"), t.float()).to(dtype) for t in (k, v))
    if layout == "pshd":
        k, v = (t.permute(0, 2, 1, 3).contiguous() for t in (k, v))
    cache = A.PagedKVCache(k, v, *scales, layout=layout)
    batch = O.device_batch(b)
    x = randn(rng, b["rows"], hq + 1, d) * spread
    q = x[:, :hq]  # a row stride of its own
    scale = d ** -0.5 if scale is None else scale
    out, lse = cache.attend(q, batch, scale=scale, window=window, return_lse=True)
    again, lse2 = cache.attend(q, batch, scale=scale, window=window, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "two runs differ"
    assert torch.equal(cache.attend(q, batch, scale=scale, window=window), out)
    k64, v64 = O.f64(k) * scales[0], O.f64(v) * scales[1]
    if layout == "pshd":
        k64, v64 = k64.transpose(0, 2, 1, 3), v64.transpose(0, 2, 1, 3)
    want, bound, wl, lb = O.attend(O.f64(q), k64, v64, b, scale, window)
    O.assert_within(O.f64(out), want, bound, "out")
    O.assert_within(O.f64(lse), wl, lb, "lse")
    for k in (1, 2):  # each kernel, whatever the call's size
        with kernel(k):
            pinned, pinned_lse = cache.attend(q, batch, scale=scale, window=window, return_lse=True)
            assert torch.equal(cache.attend(q, batch, scale=scale, window=window), pinned), "two runs differ"
        O.assert_within(O.f64(pinned), want, bound, f"out, kernel {k}")
        O.assert_within(O.f64(pinned_lse), wl, lb, f"lse, kernel {k}")
    return out, lse, b, cache, batch, q, (k64, v64)


SHAPES = [(64, 8, 2), (64, 5, 5), (128, 12, 4), (128, 8, 8), (256, 16, 8), (256, 6, 2), (512, 16, 1), (512, 4, 2), (64, 40, 1),
          (256, 20, 1), (512, 32, 1), (128, 48, 2)]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d,hq,hk", SHAPES)
def test_decode_lengths(gpu_lib, d, hq, hk, kind):
    """One new token each, contexts around every boundary of groups, tiles and pages."""
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 0, 300]
    attend_case(np.random.default_rng(d + hq), d, hq, hk, [1] * len(kv), kv, 16, kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d,hq,hk", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 16, 37])
def test_chunks(gpu_lib, d, hq, hk, kind, window):
    """Prompts, tails of prompts, verify blocks and single tokens in one batch, with padding
    rows and a request without new tokens."""
    attend_case(np.random.default_rng(7 * d + hq + window), d, hq, hk, [33, 1, 0, 8, 70, 2], [33, 90, 50, 41, 130, 2], 32, kind,
                window=window, padding=2)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d,hq,hk", [(64, 8, 2), (128, 12, 4), (256, 16, 8), (512, 16, 1)])
def test_long_contexts_are_split(gpu_lib, d, hq, hk, kind):
    """Few rows and long contexts: the split launch and its join, wide score ranges."""
    attend_case(np.random.default_rng(d), d, hq, hk, [1, 3], [5003, 777], 64, kind, spread=6.0)
    attend_case(np.random.default_rng(d), d, hq, hk, [2], [4000], 128, kind, window=1024, layout="pshd")


@pytest.mark.parametrize("d,hq,hk,kind", [(256, 16, 8, "bf16"), (512, 16, 1, "bf16"), (512, 16, 1, "e4m3"), (128, 4, 4, "bf16"),
                                          (64, 6, 2, "e4m3")])
@pytest.mark.parametrize("q_len,kv_len,window", [(257, 257, 0), (200, 901, 0), (300, 700, 64), (129, 640, 100)])
def test_prefill_tiles(gpu_lib, d, hq, hk, kind, q_len, kv_len, window):
    attend_case(np.random.default_rng(q_len), d, hq, hk, [q_len], [kv_len], 64, kind, window=window)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d,hq,hk", [(64, 8, 2), (128, 12, 4), (256, 16, 8), (512, 16, 1)])
@pytest.mark.parametrize("window", [0, 1500])
def test_chunks_far_into_their_contexts(gpu_lib, d, hq, hk, kind, window):
    """Chunks whose keys take many tiles and several rounds of table entries, beside single
    tokens; and one request alone."""
    rng = np.random.default_rng(d + window)
    attend_case(rng, d, hq, hk, [70, 1, 0, 9, 1], [3100, 2500, 7, 2049, 1], 16, kind, window=window, padding=1)
    attend_case(rng, d, hq, hk, [67], [4500], 32, kind, window=window, spread=4.0)


@pytest.mark.parametrize("d,hq,hk", [(64, 4, 2), (256, 4, 2), (512, 16, 1)])
def test_many_requests(gpu_lib, d, hq, hk):
    """More requests than a wave has lanes, of very different lengths and numbers of tokens."""
    rng = np.random.default_rng(d)
    q_lens = [int(v) for v in rng.choice([0, 1, 1, 1, 2, 5, 20], 150)] + [130, 1]
    kv_lens = [a + int(rng.integers(0, 60)) for a in q_lens[:-1]] + [3001]
    attend_case(rng, d, hq, hk, q_lens, kv_lens, 16, padding=4)
    attend_case(rng, d, hq, hk, [1] * 70, [int(v) for v in rng.integers(1, 200, 69)] + [2600], 32, "e4m3")


@pytest.mark.parametrize("page", [16, 64, 256, 1024])
@pytest.mark.parametrize("layout", ["phsd", "pshd"])
def test_pages(gpu_lib, page, layout):
    attend_case(np.random.default_rng(page), 256, 4, 2, [1, 20, 100], [page, 3 * page + 5, 2 * page + 100], page, layout=layout,
                window=2 * page)


def test_rows_without_keys(gpu_lib):
    """No tokens, more new tokens than positions, every page absent, a table too narrow."""
    import torch

    def change(b):
        b["tables"][2, :] = -1
        b["tables"][3, 0] = b["num_pages"]

    for d, hq, hk in ((256, 16, 8), (512, 16, 1)):
        out, lse, b, *_ = attend_case(np.random.default_rng(1), d, hq, hk, [1, 9, 5, 20], [0, 4, 60, 60], 16, padding=3, change=change)
        for row in [0] + list(range(1, 6)) + list(range(10, 15)) + list(range(35, 38)):
            assert bool((out[row] == 0).all()) and bool((lse[row] == float("-inf")).all()), row
        assert bool(torch.isfinite(lse[6:10]).all()) and bool(torch.isfinite(lse[15:35]).all())
    # positions past the table's pages have no keys of their own
    attend_case(np.random.default_rng(2), 128, 4, 2, [3, 1], [100, 40], 16, width=3)


@pytest.mark.parametrize("d,hq,hk,kind", [(256, 16, 8, "bf16"), (512, 16, 1, "bf16"), (64, 4, 4, "bf16"), (256, 4, 2, "e4m3")])
@pytest.mark.parametrize("q_len,kv_len,window", [(40, 40, 0), (8, 300, 0), (150, 400, 50), (3, 3000, 0), (300, 300, 0)])
def test_infinities_and_nan_in_hidden_places(gpu_lib, d, hq, hk, kind, q_len, kv_len, window):
    """A token's infinite or NaN key or value reaches the rows that see it and no other."""
    import torch

    rng = np.random.default_rng(q_len)
    *_, b, cache, batch, q, (k64, v64) = attend_case(rng, d, hq, hk, [q_len], [kv_len], 32, kind, window=window)
    odd = [float("nan")] * 3 if kind == "e4m3" else [float("inf"), float("-inf"), float("nan")]
    first = kv_len - q_len
    for n, (p, h, e) in enumerate([(first + q_len // 2, 0, 1), (kv_len - 1, hk - 1, d - 1), (max(0, first - max(0, window - 5)), 0, 2),
                                   (first + q_len // 2, 0, 3), (kv_len - 2 if kv_len > 1 else 0, 0, 1)]):
        page, slot = O.slot_of(b, 0, p)
        value = odd[n % 3]
        cache.v.view(torch.uint8 if kind == "e4m3" else torch.bfloat16)[page, h, slot, e] = 0x7F if kind == "e4m3" else value
        v64[page, h, slot, e] = value
    want, bound, wl, lb = O.attend(O.f64(q), k64, v64, b, d ** -0.5, window)
    group = hq // hk
    outs = {}
    for k in (1, 2):
        with kernel(k):
            outs[k], lse = cache.attend(q, batch, window=window, return_lse=True)
        O.assert_within(O.f64(outs[k]), want, bound, f"values, kernel {k}")
        O.assert_within(O.f64(lse), wl, lb, f"lse, kernel {k}")
    # a NaN key: rows that see it are NaN, the others as before
    page, slot = O.slot_of(b, 0, kv_len - 1)
    cache.k.view(torch.uint8 if kind == "e4m3" else torch.bfloat16)[page, 0, slot, 0] = 0x7F if kind == "e4m3" else float("nan")
    for k, out in outs.items():
        with kernel(k):
            got = cache.attend(q, batch, window=window)
        assert bool(got[-1, :group].isnan().all())
        assert torch.equal(got[:-1].nan_to_num(7, 8, 9), out[:-1].nan_to_num(7, 8, 9))
        assert torch.equal(got[-1, group:].nan_to_num(7, 8, 9), out[-1, group:].nan_to_num(7, 8, 9))


def test_scales_and_extreme_scores(gpu_lib):
    for scale in (0.0, -0.3, 1.0, 40.0):
        attend_case(np.random.default_rng(5), 128, 4, 2, [20, 1], [50, 600], 16, scale=scale)


def test_offsets_past_32_bits(gpu_lib):
    """Pages that lie more than 4 GiB (and 2^31 elements) into the tensors."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(11)
    d, hk, page, pages = 128, 2, 64, 5
    gap = (1 << 30) + 4096  # elements between pages: the last one starts past 2^32
    big = [torch.empty(gap * (pages - 1) + hk * page * d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = (t.as_strided((pages, hk, page, d), (gap, page * d, d, 1)) for t in big)
    k.copy_(randn(rng, *k.shape))
    v.copy_(randn(rng, *v.shape))
    b = O.make_batch(rng, [3, 130], [64, 200], page, extra_pages=0)
    assert b["num_pages"] == pages
    cache, batch = A.PagedKVCache(k, v), O.device_batch(b)
    new = randn(rng, b["rows"], 2 * hk, d)
    q = cache.append(new[:, :hk], new[:, hk:], batch, q=randn(rng, b["rows"], 4, d))
    k64, v64 = O.f64(k), O.f64(v)
    for i, r, p in O.rows_of(b):
        at = O.slot_of(b, r, p)
        assert np.array_equal(k64[at[0], :, at[1]], O.f64(new[i, :hk])) and np.array_equal(v64[at[0], :, at[1]], O.f64(new[i, hk:]))
    out = cache.attend(q, batch)
    want, bound, _, _ = O.attend(O.f64(q), k64, v64, b, d ** -0.5)
    O.assert_within(O.f64(out), want, bound, "out")


def test_caller_tensors_and_streams(gpu_lib):
    """out into a slice of a wider tensor whose other columns stay; another stream."""
    import torch

    rng = np.random.default_rng(21)
    out, lse, b, cache, batch, q, _ = attend_case(rng, 256, 16, 8, [30, 1], [100, 700], 32)
    wide = torch.full((b["rows"], 18, 256), -7.0, dtype=torch.bfloat16, device="cuda")
    got = cache.attend(q, batch, out=wide[:, 1:17])
    assert got.data_ptr() == wide[:, 1:17].data_ptr() and torch.equal(wide[:, 1:17], out)
    assert bool((wide[:, 0] == -7).all()) and bool((wide[:, 17] == -7).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = cache.attend(q, batch)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, out)
    named = cache.attend(q, batch, stream=side)
    side.synchronize()
    assert torch.equal(named, out)


def test_graph_replays_follow_the_device_arrays(gpu_lib):
    """A captured decoding step (append, attention) replayed as the sequences grow, against
    the eager calls, with eager work between the replays."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(31)
    d, hq, hk, page, n, steps = 256, 16, 8, 16, 5, 6
    lens = np.array([1, 15, 16, 40, 2000], np.int32)
    b = O.make_batch(rng, [1] * n, list(lens + steps), page)
    shape = (b["num_pages"], hk, page, d)
    first = [randn(rng, *shape) for _ in range(2)]
    caches = [A.PagedKVCache(*[t.clone() for t in first]) for _ in range(2)]
    rope, norm = A.Rope(dev(inv_freq(d // 2))), A.HeadNorm(None)
    batch = O.device_batch(b)
    x = torch.zeros(n, hq + 2 * hk, d, dtype=torch.bfloat16, device="cuda")

    def step(cache):
        q = cache.append(x[:, hq:hq + hk], x[:, hq + hk:], batch, rope=rope, k_norm=norm, v_norm=norm, q=x[:, :hq], q_norm=norm)
        return cache.attend(q, batch, window=1024)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(caches[0])
    torch.cuda.synchronize()
    for c, t in zip((caches[0].k, caches[0].v), first):
        c.copy_(t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        replayed = step(caches[0])
    for i in range(steps):
        x.copy_(randn(rng, *x.shape))
        batch.kv_lens.copy_(dev(lens + i + 1))
        eager = step(caches[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed, eager), f"step {i}"
        assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v), f"step {i}"


def test_refusals(gpu_lib):
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(41)
    b = O.make_batch(rng, [2], [9], 16)
    batch, k = O.device_batch(b), randn(rng, b["num_pages"], 2, 16, 128)
    cache = A.PagedKVCache(k, k.clone())
    q, new = randn(rng, 2, 4, 128), randn(rng, 2, 2, 128)
    refused = [
        lambda: cache.attend(q[:, :3], batch),                    # 3 query heads over 2
        lambda: cache.attend(q[..., :64], batch),                 # another head_dim
        lambda: cache.attend(q.float(), batch),
        lambda: cache.attend(q.transpose(1, 2), batch),
        lambda: cache.attend(q, batch, window=-1),
        lambda: cache.attend(q, batch, scale=float("nan")),
        lambda: cache.attend(q, batch, out=torch.empty_like(q).float()),
        lambda: cache.attend(q, batch, out=torch.empty_like(q)[:1]),
        lambda: cache.append(new[:1], new, batch),
        lambda: cache.append(q, q, batch),                        # too many heads
        lambda: cache.append(new, new, batch, q=q[:1]),
        lambda: cache.append(new, new, batch, k_norm=A.HeadNorm(torch.ones(64, device="cuda").bfloat16())),
        lambda: cache.append(new, new, batch, rope=A.Rope(dev(inv_freq(12)))),
        lambda: A.qk_norm_rope(q, new[:1], dev(np.zeros(2, np.int32))),
        lambda: A.qk_norm_rope(q, None, dev(np.zeros(3, np.int32)), A.Rope(dev(inv_freq(8)))),
        lambda: A.qk_norm_rope(q, None, None, A.Rope(dev(inv_freq(8)))),
        lambda: A.PagedKVCache(k, k.float()),
        lambda: A.PagedKVCache(k, k[:1]),
        lambda: A.PagedKVCache(k[..., :96].contiguous(), k[..., :96].contiguous()).attend(q[..., :96].contiguous(), batch),
        lambda: A.KVBatch(batch.query_starts, batch.kv_lens.long(), batch.block_tables),
        lambda: A.KVBatch(batch.query_starts[:1], batch.kv_lens, batch.block_tables),
        lambda: A.PagedKVCache(k, k, layout="hspd"),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(gpu_lib.Gemma4Error):
            call()
            pytest.fail(f"call {i} was taken")
    assert math.isfinite(float(cache.attend(q, batch).float().abs().max()))  # and still works


def test_random_batches(gpu_lib):
    """Small random batches over the whole range of shapes, types and layouts."""
    rng = np.random.default_rng(51)
    for _ in range(40):
        d = int(rng.choice([64, 128, 256, 512]))
        hk = int(rng.choice([1, 2, 3]))
        hq = hk * int(rng.choice([1, 2, 3, 5, 8, 16, 17]))
        n = int(rng.integers(1, 7))
        q_lens = [int(v) for v in rng.choice([0, 1, 1, 2, 7, 16, 40, 90], n)]
        kv_lens = [max(0, a + int(rng.choice([-1, 0, 0, 1, 5, 64, 200]))) for a in q_lens]
        if sum(q_lens) == 0:
            q_lens[0] = kv_lens[0] = 1
        page = int(rng.choice([16, 32, 64, 128]))
        kind, window = str(rng.choice(["bf16", "e4m3"])), int(rng.choice([0, 0, 1, 20, 64, 129]))
        layout = str(rng.choice(["phsd", "pshd"]))
        print(f"d={d} hq={hq} hk={hk} q={q_lens} kv={kv_lens} page={page} {kind} window={window} {layout}", flush=True)
        attend_case(rng, d, hq, hk, q_lens, kv_lens, page, kind, window=window, layout=layout, padding=int(rng.integers(0, 3)))
