"""The paged-cache calls on the GPU at the edges of what they take: outputs on a named stream,
infinities and NaN beside rotated pairs, scales that leave fp32's range,
more query heads to a KV head than a tile has rows."""

import numpy as np
import pytest

import attention_oracle as O
from test_gpu_attention import attend_case, dev, inv_freq, kernel, randn

pytestmark = pytest.mark.gpu


def stream_of(t):
    """The stream whose memory holds t (the allocator's own record; 0: the default stream's)."""
    import torch

    for s in torch.cuda.memory_snapshot():
        if s["address"] <= t.data_ptr() < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not the allocator's memory")


def test_outputs_on_a_named_stream(gpu_lib):
    """An output that a call makes belongs to the stream it is written on, and equals that of
    the call on the current stream."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(61)
    out, lse, b, cache, batch, q, _ = attend_case(rng, 128, 8, 4, [30, 1], [100, 700], 32)
    k = randn(rng, b["rows"], 4, 128)
    pos, rope = dev(np.arange(b["rows"], dtype=np.int32)), A.Rope(dev(inv_freq(64)))
    turned = A.qk_norm_rope(q, k, pos, rope)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    # attention before the append, which changes the cache
    got = list(cache.attend(q, batch, return_lse=True, stream=side)) + list(A.qk_norm_rope(q, k, pos, rope, stream=side))
    appended = cache.append(k, k, batch, q=q, stream=side)
    side.synchronize()
    for t in got + [appended]:
        assert stream_of(t) == side.cuda_stream
    for t, want in zip(got, (out, lse, *turned)):
        assert torch.equal(t, want)
    assert stream_of(out) != side.cuda_stream
    assert np.array_equal(O.f64(appended), O.f64(q))


@pytest.mark.parametrize("distance", [1, 8, 32])
def test_infinities_and_nan_beside_the_rotated_pairs(gpu_lib, distance):
    """An element outside the rotated pairs passes as it is, whatever lies next to it, and so do
    all of the values."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(71)
    d, pairs, rows = 128, 8, 3
    rope = A.Rope(dev(inv_freq(pairs)), distance)
    pos = dev(np.array([5, 1000, 77], np.int32))
    x = randn(rng, rows, 4, d)
    plain, _ = A.qk_norm_rope(x, None, pos, rope)
    odd = [float("inf"), float("-inf"), float("nan")]
    y, want = x.clone(), plain.clone()
    for row in range(rows):
        for e in (50, 71, 127):  # neither these nor their neighbours are rotated
            y[row, 1, e] = want[row, 1, e] = odd[row]
    got, _ = A.qk_norm_rope(y, None, pos, rope)
    same = lambda a, b: torch.equal(a.nan_to_num(7, 8, 9), b.nan_to_num(7, 8, 9)) and torch.equal(a.isnan(), b.isnan())  # noqa: E731
    assert same(got, want)
    # values are not rotated at all: neither their first pair nor the others
    v = y.clone()
    v[:, 0, 0], v[:, 2, 3], v[:, 3, distance] = odd[0], odd[1], odd[2]
    b = O.make_batch(rng, [rows], [rows], 16)
    cache = A.PagedKVCache.allocate(b["num_pages"], 16, 4, d)
    cache.append(x, v, O.device_batch(b), rope=rope)
    assert same(cache.v[int(b["tables"][0, 0]), :, :rows].transpose(0, 1), v)


@pytest.mark.parametrize("d,hq,hk", [(64, 8, 2), (128, 4, 2), (256, 4, 2), (512, 16, 1)])
@pytest.mark.parametrize("scale,k_scale,kind", [(1e-20, 1e-30, "e4m3"), (-1e-20, 1e-30, "e4m3"), (1.5e-45, 1.0, "bf16"), (1e-38, 1.0, "bf16")])
def test_scales_below_fp32s_range(gpu_lib, d, hq, hk, scale, k_scale, kind):
    """A scale that vanishes (with that of the keys) leaves every visible key the same weight,
    and the hidden ones none."""
    import torch

    from helios_amd import attention as A

    rng = np.random.default_rng(d)
    *_, b, cache, batch, q, (k64, v64) = attend_case(rng, d, hq, hk, [40, 1, 3], [90, 33, 2], 16, kind, window=37)
    small = A.PagedKVCache(cache.k, cache.v, k_scale, cache.v_scale)
    k64 = O.f64(cache.k) * k_scale
    want, bound, wl, lb = O.attend(O.f64(q), k64, v64, b, scale, 37)
    for kernel_ in (1, 2):
        with kernel(kernel_):
            out, lse = small.attend(q, batch, scale=scale, window=37, return_lse=True)
        O.assert_within(O.f64(out), want, bound, f"out, kernel {kernel_}")
        O.assert_within(O.f64(lse), wl, lb, f"lse, kernel {kernel_}")


@pytest.mark.parametrize("d,hq,hk,kind", [(64, 8, 2, "bf16"), (128, 4, 2, "e4m3"), (256, 4, 2, "bf16"), (512, 16, 1, "bf16")])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite_at_scale_zero(gpu_lib, d, hq, hk, kind, odd):
    """Zero times an infinite or NaN score is NaN: such a query's head is NaN in its row, and
    nothing else changes."""
    import torch

    rng = np.random.default_rng(d + 1)
    out, lse, b, cache, batch, q, _ = attend_case(rng, d, hq, hk, [40, 1], [60, 33], 16, kind, scale=0.0)
    for k in (1, 2):
        with kernel(k):
            before, before_lse = cache.attend(q, batch, scale=0.0, return_lse=True)
            q2 = q.clone()
            q2[7, 1, 5] = q2[40, 0, d - 1] = odd
            got, got_lse = cache.attend(q2, batch, scale=0.0, return_lse=True)
        for row, head in ((7, 1), (40, 0)):
            assert bool(got[row, head].isnan().all()) and bool(got_lse[row, head].isnan()), (k, row)
            got[row, head], got_lse[row, head] = before[row, head], before_lse[row, head]
        assert torch.equal(got, before) and torch.equal(got_lse, before_lse), k


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("d,hq,hk", [(64, 130, 1), (64, 300, 1), (128, 260, 2), (512, 130, 1)])
def test_more_heads_to_a_key_than_a_tile_has_rows(gpu_lib, d, hq, hk, kind):
    """A KV head's query heads in several runs of 128 (and of 16), the last one partly filled:
    uncut, and with items to join."""
    attend_case(np.random.default_rng(hq), d, hq, hk, [5, 1, 0, 2], [40, 33, 7, 2], 16, kind, window=20, padding=1)
    attend_case(np.random.default_rng(hq), d, hq, hk, [2, 1], [1500, 700], 32, kind)
    attend_case(np.random.default_rng(hq), d, hq, hk, [1], [2100], 64, kind, window=1800)
