"""Plain 64-bit implementations (numpy, on the host) of the head norms with rotation, the
append to a paged cache and the attention over it, with error bounds for the kernels'
types, and random batches for them.

Bounds: a bf16 result is half a step off at most (2^-8 of its size).  The kernels compute
in fp32: a few ulp (2^-24) of the terms of each sum.  In the attention the softmax weights
are rounded to bf16 for their product with the values (2^-8 of each term p |v|)."""

import numpy as np

BF16, E4M3, F32 = 2.0 ** -8, 2.0 ** -4, 2.0 ** -24


def f64(t):
    """A device tensor's values (bf16 or e4m3 too) as float64."""
    return t.detach().float().cpu().numpy().astype(np.float64)


def norm_rope(x, positions, inv_freq=None, distance=0, norm=False, weight=None, eps=1e-6):
    """x float64 [rows, heads, D] -> (y, bound of a bf16 result's error)."""
    n = x.copy()
    if norm:
        n = n / np.sqrt((n * n).mean(-1, keepdims=True) + eps)
        if weight is not None:
            n = n * weight
    y = n.copy()
    if inv_freq is not None:
        pairs = inv_freq.size
        ang = positions.astype(np.float64)[:, None] * inv_freq.astype(np.float64)[None, :]
        cos, sin = np.cos(ang)[:, None, :], np.sin(ang)[:, None, :]
        if distance == 1:
            a, b = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
        else:
            a, b = slice(0, pairs), slice(distance, distance + pairs)
        y[..., a] = n[..., a] * cos - n[..., b] * sin
        y[..., b] = n[..., b] * cos + n[..., a] * sin
    # fp32: the norm's sum and root, two products, the sine and cosine
    slack = 64 * F32 * np.abs(n).max(-1, keepdims=True)
    return y, BF16 * np.abs(y) + slack


def stored(y, slack, scale=None):
    """(value held, bound) of y in a bf16 page, or over `scale` in an e4m3 one."""
    if scale is None:
        return y, slack
    z = np.clip(y / scale, -448, 448)
    # half a step, of a normal (2^-4) or of the subnormals (2^-10), and fp32 error before it
    return z, np.maximum(E4M3 * np.abs(z), 2.0 ** -10) + 2 * np.abs(slack - BF16 * np.abs(y)) / scale + 1e-6 * np.abs(z)


def slot_of(batch, r, p):
    """(page, slot) of position p of request r, or None where there is no such page."""
    at = p // batch["page"]
    if p < 0 or at >= batch["tables"].shape[1]:
        return None
    page = int(batch["tables"][r, at])
    return (page, p % batch["page"]) if 0 <= page < batch["num_pages"] else None


def rows_of(batch):
    """(row, request, position) of every row of the batch; request None for padding."""
    s = batch["starts"]
    for r in range(len(s) - 1):
        for i in range(s[r], s[r + 1]):
            yield i, r, int(batch["kv_lens"][r]) - (s[r + 1] - i)
    for i in range(s[-1], batch["rows"]):
        yield i, None, 0


def attend(q, k_cache, v_cache, batch, scale, window=0):
    """q float64 [rows, heads, D], caches float64 [pages, kv_heads, page, D] (scales applied).
    Returns out, its bound, lse, its bound."""
    rows, heads, d = q.shape
    group = heads // k_cache.shape[1]
    out, bound = np.zeros_like(q), np.zeros_like(q)
    lse, lse_bound = np.full((rows, heads), -np.inf), np.zeros((rows, heads))
    held = {}  # a request's present positions, and its keys and values
    for i, r, p in rows_of(batch):
        if r is None:
            continue
        if r not in held:
            at = [(j, slot_of(batch, r, j)) for j in range(int(batch["kv_lens"][r]))]
            at = [(j, *w) for j, w in at if w is not None]
            places, pages, slots = (np.array(w, np.int64) for w in zip(*at)) if at else (np.zeros(0, np.int64),) * 3
            held[r] = places, [(k_cache[pages, h, slots], v_cache[pages, h, slots]) for h in range(k_cache.shape[1])]
        places, per_head = held[r]
        begin, end = np.searchsorted(places, [max(0, p - window + 1) if window else 0, p + 1])
        if begin >= end:
            continue
        for h in range(heads):
            k, v = (x[begin:end] for x in per_head[h // group])
            s = scale * (k @ q[i, h])
            top = s.max()
            e = np.exp(s - top)
            z = e.sum()
            pr = e / z
            with np.errstate(invalid="ignore"):
                out[i, h] = pr @ v
            lse[i, h] = top + np.log(z)
            # fp32 error of a score: its D products, the scale and the exponent's argument
            ds = 4 * F32 * (d ** 0.5 * abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max() + np.abs(s).max() + 4)
            mass = pr @ np.where(np.isfinite(v), np.abs(v), 0)
            bound[i, h] = BF16 * np.abs(np.where(np.isfinite(out[i, h]), out[i, h], 0)) + (1.01 * BF16 + 2 * ds) * mass + 1e-30
            lse_bound[i, h] = 2 * ds + 16 * F32 * (1 + abs(lse[i, h]))
    return out, bound, lse, lse_bound


def make_batch(rng, q_lens, kv_lens, page, padding=0, extra_pages=3, width=None):
    """A batch on the host with pages in random order; entries past a request's length are -1."""
    need = [-(-max(kv, 0) // page) for kv in kv_lens]
    width = width or max(1, max(need))
    num_pages = max(1, sum(min(n, width) for n in need)) + extra_pages
    order = rng.permutation(num_pages)
    tables = np.full((len(q_lens), width), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        n = min(n, width)
        tables[r, :n] = order[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    return {"starts": starts, "kv_lens": np.array(kv_lens, np.int32), "tables": tables, "page": page,
            "num_pages": num_pages, "rows": int(starts[-1]) + padding}


def device_batch(batch):
    import torch

    from helios_amd.attention import KVBatch

    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return KVBatch(dev(batch["starts"]), dev(batch["kv_lens"]), dev(batch["tables"]))


def assert_within(got, want, bound, what):
    bad_kind = (np.isnan(got) != np.isnan(want)) | (np.isinf(want) & (got != want)) | (np.isinf(got) & (got != want))
    assert not bad_kind.any(), f"{what}: {int(bad_kind.sum())} values differ in inf or NaN"
    fine = np.isfinite(want)
    err = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)), 0)
    over = err > np.broadcast_to(bound, err.shape)
    worst = float((err / np.maximum(np.broadcast_to(bound, err.shape), 1e-300)).max()) if err.size else 0.0
    assert not over.any(), f"{what}: {int(over.sum())} of {err.size} values off, worst {worst:.3g} of the bound"
