"""The calls that serving Gemma 4 12B makes between a layer's q|k|v projection and its o
projection, for timing: the norms and rotation of queries and keys, appending keys and
values to a paged cache, and the attention that reads it.

Layers are those of the decoder that ``bench.py`` runs (16 query and 8 KV heads of 256,
a window of 1024) and its full-attention layers (16 query heads and one KV head of 512,
the values made from the key projection, a quarter of each head rotated); a few drawn
cases have other head counts.  Caches hold [pages, kv_heads, page_size, head_dim] in bf16
or e4m3; a request's pages lie in any order, and a windowed layer keeps only the pages
that its window still reaches (-1 elsewhere).

Kinds of case:

* ``rope``: qk_norm_rope on the fused rows of a projection.
* ``append``: one launch that norms and rotates q and appends k and v.
* ``attend``: attention of each request's new tokens over its pages.
* ``step``: an append and the attention after it, as one layer runs them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
# name -> query heads, KV heads, head_dim, window, rope base, rotated pairs, pair distance
LAYERS = {
    "sliding": (16, 8, 256, 1024, 1.0e4, 128, 128),
    "full": (16, 1, 512, 0, 1.0e6, 64, 256),
    "mha128": (8, 8, 128, 0, 1.0e4, 64, 64),
    "gqa128": (12, 4, 128, 333, 1.0e5, 32, 32),
    "gqa64": (32, 4, 64, 0, 1.0e4, 32, 32),
}


def listed():
    return [
        # the smallest call: the query and key heads of one token
        {"name": "rope_token_1", "kind": "rope", "layer": "sliding", "requests": 1, "q_max": 1, "kv_max": 9001, "ragged": False},
        # a whole prefill chunk of a full-attention layer
        {"name": "rope_full_chunk_2048", "kind": "rope", "layer": "full", "requests": 1, "q_max": 2048, "kv_max": 131072, "ragged": False},
        # one decoding step of a batch: a token each, far into their contexts
        {"name": "append_decode_32", "kind": "append", "layer": "sliding", "requests": 32, "q_max": 1, "kv_max": 60000, "ragged": True, "page": 64, "dtype": "bf16"},
        # prompts of several requests into an 8-bit cache, ragged
        {"name": "append_e4m3_prompts", "kind": "append", "layer": "full", "requests": 5, "q_max": 777, "kv_max": 5000, "ragged": True, "page": 16, "dtype": "e4m3"},
        # one user decoding in a long context, full attention
        {"name": "decode_full_1", "kind": "attend", "layer": "full", "requests": 1, "q_max": 1, "kv_max": 32768, "ragged": False, "page": 64, "dtype": "bf16", "lse": False},
        # a decoding batch over the sliding layers
        {"name": "decode_sliding_64", "kind": "attend", "layer": "sliding", "requests": 64, "q_max": 1, "kv_max": 9000, "ragged": True, "page": 32, "dtype": "bf16", "lse": False},
        # a decoding batch over an 8-bit cache, ragged contexts, full attention
        {"name": "decode_full_e4m3_32", "kind": "attend", "layer": "full", "requests": 32, "q_max": 1, "kv_max": 16000, "ragged": True, "page": 64, "dtype": "e4m3", "lse": False},
        # blocks of drafted tokens verified for a few requests
        {"name": "verify_sliding_8", "kind": "attend", "layer": "sliding", "requests": 4, "q_max": 8, "kv_max": 4100, "ragged": False, "page": 64, "dtype": "bf16", "lse": False},
        # short prompts and decodes in one batch, ragged, with the log-sum-exp a later merge needs
        {"name": "mixed_full_lse", "kind": "attend", "layer": "full", "requests": 12, "q_max": 300, "kv_max": 3900, "ragged": True, "page": 16, "dtype": "bf16", "lse": True},
        # one decoding step of a layer, append and attention
        {"name": "step_sliding_8", "kind": "step", "layer": "sliding", "requests": 8, "q_max": 1, "kv_max": 1500, "ragged": True, "page": 64, "dtype": "bf16"},
        # a prefill chunk at the end of a 16K prompt: a sliding layer, then a full one
        {"name": "chunk_sliding_2048", "kind": "attend", "layer": "sliding", "requests": 1, "q_max": 2048, "kv_max": 16384, "ragged": False, "page": 64, "dtype": "bf16", "lse": False},
        {"name": "chunk_full_2048", "kind": "attend", "layer": "full", "requests": 1, "q_max": 2048, "kv_max": 16384, "ragged": False, "page": 64, "dtype": "bf16", "lse": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "step"])
    layer = rng.choice(["sliding", "sliding", "full", "full", "mha128", "gqa128", "gqa64"])
    shape = rng.choice(["decode", "verify", "chunk"])
    if shape == "decode":
        requests, q_max = _log_int(rng, 1, 96), 1
    elif shape == "verify":
        requests, q_max = _log_int(rng, 1, 32), rng.randint(2, 16)
    else:
        requests = rng.choice([1, 1, 2, 5])
        q_max = _log_int(rng, 17, 2048 // requests)
    # scores of the plain form and the caches stay under those of the largest listed cases
    kv_hi = max(64, min(32768, 524288 // requests, 33554432 // (requests * q_max)))
    case = {"kind": kind, "layer": layer, "requests": requests, "q_max": q_max,
            "kv_max": max(q_max, _log_int(rng, 1, kv_hi)), "ragged": rng.choice([True, True, False])}
    if kind != "rope":
        case.update(page=rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["bf16", "bf16", "e4m3"]))
    if kind == "attend":
        case["lse"] = rng.choice([True, False])
    return case


def _lens(case):
    """(new tokens, tokens in the cache with them) of each request: the case's alone."""
    n, q, kv = case["requests"], case["q_max"], case["kv_max"]
    if not case["ragged"]:
        return [q] * n, [kv] * n
    rng = random.Random("%d %d %d" % (n, q, kv))
    qs = [q] + [rng.randint(1, q) if rng.random() < 0.7 else 1 for _ in range(n - 1)]
    return qs, [kv] + [max(a, _log_int(rng, max(1, kv // 40), kv)) for a in qs[1:]]


def _span(case):
    """The positions of each request that a call touches: [first, kv_len)."""
    window = LAYERS[case["layer"]][3]
    qs, kvs = _lens(case)
    if case["kind"] == "append":
        return [(kv - q, kv) for q, kv in zip(qs, kvs)]
    return [(max(0, kv - q - window + 1) if window else 0, kv) for q, kv in zip(qs, kvs)]


def prepare(case, seed):
    hq, hk, d, window, base, pairs, dist = LAYERS[case["layer"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    qs, kvs = _lens(case)
    rows = sum(qs)
    # projections leave some heads louder than others
    loud = torch.exp(0.5 * randn(1, hq + 2 * hk, 1))
    x = (randn(rows, hq + 2 * hk, d) * loud).bfloat16().reshape(rows, -1)
    starts = [0]
    for q in qs:
        starts.append(starts[-1] + q)
    positions = [kv - q + i for q, kv in zip(qs, kvs) for i in range(q)]
    state = {
        "case": dict(case), "x": x, "rows": rows,
        "positions": torch.tensor(positions, dtype=torch.int32, device="cuda"),
        "inv_freq": torch.tensor([base ** (-2.0 * i / (2 * dist)) for i in range(pairs)], dtype=torch.float32, device="cuda"),
        "q_weight": (1 + 0.2 * randn(d)).bfloat16(), "k_weight": (1 + 0.2 * randn(d)).bfloat16(),
        "window": window, "scale": 2.0 / math.sqrt(d),
    }
    if case["kind"] == "rope":
        return state
    page, span = case["page"], _span(case)
    width = (max(kvs) + page - 1) // page
    held = [(a // page, (b + page - 1) // page) for a, b in span]
    count = sum(b - a for a, b in held)
    order = torch.randperm(count, device="cuda", generator=g).to(torch.int32).cpu()
    tables = torch.full((len(qs), width), -1, dtype=torch.int32)
    at = 0
    for r, (a, b) in enumerate(held):
        tables[r, a:b] = order[at:at + b - a]
        at += b - a
    shape = (count, hk, page, d)
    state["k_scale"], state["v_scale"] = (0.0625, 0.03125) if case["dtype"] == "e4m3" else (1.0, 1.0)
    kinds = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
    # what earlier steps left there: normed keys and values
    state["k_cache"] = (randn(*shape) / state["k_scale"]).clamp(-448, 448).to(kinds[case["dtype"]])
    state["v_cache"] = (randn(*shape) / state["v_scale"]).clamp(-448, 448).to(kinds[case["dtype"]])
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["kv_lens"] = torch.tensor(kvs, dtype=torch.int32, device="cuda")
    state["tables"] = tables.cuda()
    state["q"] = randn(rows, hq, d).bfloat16()
    # what a scheduler knows on the host
    state["q_max"], state["kv_max"] = max(qs), max(kvs)
    state["most_pages"] = max(b - a for a, b in held)
    state["first_page"] = torch.tensor([a for a, _ in held], dtype=torch.int64, device="cuda")
    return state


def _split(state):
    """q, k and v heads of the fused rows; a full layer's values come from its keys' projection."""
    hq, hk, d = LAYERS[state["case"]["layer"]][:3]
    x = state["x"]
    q, k = x[:, :hq * d].unflatten(1, (hq, d)), x[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    return q, k, k if state["case"]["layer"] == "full" else x[:, (hq + hk) * d:].unflatten(1, (hk, d))


# ---------------------------------------------------------------- the plain form

def _norm(x, weight):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x if weight is None else x * weight.float()


def _rotate(x, positions, inv_freq, dist):
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    pairs = inv_freq.numel()
    a, b = x[..., :pairs], x[..., dist:dist + pairs]
    return torch.cat([a * cos - b * sin, x[..., pairs:dist], b * cos + a * sin, x[..., dist + pairs:]], dim=-1)


def _plain_rope(state):
    q, k, _ = _split(state)
    dist = LAYERS[state["case"]["layer"]][6]
    turn = lambda x, w: _rotate(_norm(x, w), state["positions"], state["inv_freq"], dist)  # noqa: E731
    return turn(q, state["q_weight"]), turn(k, state["k_weight"])


def _store(x, scale, dtype):
    return x.to(dtype) if dtype == torch.bfloat16 else (x / scale).clamp(-448, 448).to(dtype)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_append(state):
    q, k = _plain_rope(state)
    v = _norm(_split(state)[2], None)
    starts, positions, page = state["starts"].long(), state["positions"].long(), state["case"]["page"]
    request = torch.searchsorted(starts, torch.arange(state["rows"], device="cuda"), right=True) - 1
    pages, slots = state["tables"][request, positions // page].long(), positions % page
    for_k, for_v = state["k_cache"], state["v_cache"]
    _bytes(for_k)[pages, :, slots] = _bytes(_store(k, state["k_scale"], for_k.dtype))
    _bytes(for_v)[pages, :, slots] = _bytes(_store(v, state["v_scale"], for_v.dtype))
    return q.bfloat16()


def _plain_attend(state, q):
    case = state["case"]
    hq, hk, d, window = LAYERS[case["layer"]][:4]
    n, group, page, q_max = case["requests"], hq // hk, case["page"], state["q_max"]
    starts, kv_lens = state["starts"].long(), state["kv_lens"].long()
    q_lens = starts[1:] - starts[:-1]
    # each request's pages, from the first one it holds
    at = state["first_page"][:, None] + torch.arange(state["most_pages"], device="cuda")[None, :]
    width = state["tables"].shape[1]
    pages = state["tables"].long().gather(1, at.clamp(max=width - 1))
    pages = torch.where(at < width, pages, -1)
    kv_pos = (at[:, :, None] * page + torch.arange(page, device="cuda")).reshape(n, -1)
    there = (pages >= 0)[:, :, None].expand(-1, -1, page).reshape(n, -1) & (kv_pos < kv_lens[:, None])

    def take(cache):
        t = _bytes(cache)[pages.clamp(min=0)].view(cache.dtype).float()  # [n, pages, hk, page, d]
        return t.permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)

    i = torch.arange(q_max, device="cuda")
    token = (starts[:-1, None] + i).clamp(max=state["rows"] - 1)
    rows = q.float()[token].reshape(n, q_max, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * q_max, d)
    s = torch.matmul(rows, take(state["k_cache"]).transpose(2, 3)) * (state["scale"] * state["k_scale"])
    q_pos = (kv_lens - q_lens)[:, None] + i
    seen = there[:, None, :] & (kv_pos[:, None, :] <= q_pos[:, :, None])
    if window:
        seen = seen & (kv_pos[:, None, :] > q_pos[:, :, None] - window)
    s = s.view(n, hk, group, q_max, -1).masked_fill(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = (e / total.clamp(min=1e-37)).view(n, hk, group * q_max, -1)
    o = torch.matmul(p, take(state["v_cache"])) * state["v_scale"]
    o = o.view(n, hk, group, q_max, d).permute(0, 3, 1, 2, 4).reshape(n, q_max, hq, d)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(n, q_max, hq)
    row = torch.arange(state["rows"], device="cuda")
    request = torch.searchsorted(starts, row, right=True) - 1
    at = row - starts[request]
    return o[request, at].bfloat16(), lse[request, at]


# ---------------------------------------------------------------- the framework's calls

def _held(state):
    """The objects that a server keeps: the rotation, the norms, the cache and the batch."""
    if "held" not in state:
        from helios_amd import attention

        held = {"rope": attention.Rope(state["inv_freq"], LAYERS[state["case"]["layer"]][6]),
                "q_norm": attention.HeadNorm(state["q_weight"], EPS), "k_norm": attention.HeadNorm(state["k_weight"], EPS),
                "v_norm": attention.HeadNorm(None, EPS)}
        if "k_cache" in state:
            held["cache"] = attention.PagedKVCache(state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"])
            held["batch"] = attention.KVBatch(state["starts"], state["kv_lens"], state["tables"])
        state["held"] = held
    return state["held"]


def _own_rope(state, h):
    from helios_amd import attention

    q, k, _ = _split(state)
    return attention.qk_norm_rope(q, k, state["positions"], h["rope"], q_norm=h["q_norm"], k_norm=h["k_norm"])


def _own_append(state, h):
    q, k, v = _split(state)
    return h["cache"].append(k, v, h["batch"], rope=h["rope"], k_norm=h["k_norm"], v_norm=h["v_norm"], q=q, q_norm=h["q_norm"])


def run(state):
    kind = state["case"]["kind"]
    if kind == "rope":
        if own:
            q, k = _own_rope(state, _held(state))
        else:
            q, k = (t.bfloat16() for t in _plain_rope(state))
        return {"q": q, "k": k}
    if kind == "append":
        q = _own_append(state, _held(state)) if own else _plain_append(state)
        return {"q": q, "k": state["k_cache"], "v": state["v_cache"]}
    if kind == "step":
        if own:
            h = _held(state)
            q = _own_append(state, h)
            out = h["cache"].attend(q, h["batch"], scale=state["scale"], window=state["window"])
        else:
            q = _plain_append(state)
            out, _ = _plain_attend(state, q)
        return {"out": out, "k": state["k_cache"], "v": state["v_cache"]}
    if own:
        h = _held(state)
        if state["case"]["lse"]:
            out, lse = h["cache"].attend(state["q"], h["batch"], scale=state["scale"], window=state["window"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": h["cache"].attend(state["q"], h["batch"], scale=state["scale"], window=state["window"])}
    out, lse = _plain_attend(state, state["q"])
    return {"out": out, "lse": lse} if state["case"]["lse"] else {"out": out}


def work(case):
    hq, hk, d, window = LAYERS[case["layer"]][:4]
    qs, kvs = _lens(case)
    rows, kind = sum(qs), case["kind"]
    size = 2 if case.get("dtype") != "e4m3" else 1
    heads_in = hq + hk if kind == "rope" or case["layer"] == "full" else hq + 2 * hk
    if kind == "rope":
        return {"bytes": rows * d * 4 * (hq + hk) + 4 * rows, "flops": 8 * rows * d * (hq + hk)}
    put = {"bytes": rows * d * (2 * heads_in + 2 * hq + 2 * hk * size), "flops": 8 * rows * d * (hq + 2 * hk)}
    if kind == "append":
        return put
    pairs = keys = 0
    for q, kv, (first, last) in zip(qs, kvs, _span(case)):
        keys += last - first
        for p in range(kv - q, kv):
            pairs += min(p + 1, window) if window else p + 1
    got = {"bytes": 2 * keys * hk * d * size + 4 * rows * hq * d + 4 * sum((b - a + case["page"] - 1) // case["page"] for a, b in _span(case))
           + (4 * rows * hq if case.get("lse") else 0), "flops": 4 * d * hq * pairs}
    if kind == "step":
        return {"bytes": got["bytes"] + put["bytes"] - 4 * rows * hq * d, "flops": got["flops"] + put["flops"]}
    return got


# ---------------------------------------------------------------- 64 bits

def _exact_heads(x, weight, positions, inv_freq, dist):
    """[rows, heads, d] in 64 bits, each pair turned as a complex number."""
    y = x.double()
    y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt()
    if weight is not None:
        y = y * weight.double()
    if inv_freq is None:
        return y
    n = inv_freq.numel()
    z = torch.complex(y[..., :n].contiguous(), y[..., dist:dist + n].contiguous())
    angle = torch.outer(positions.double(), inv_freq.double()).unsqueeze(1)
    z = z * torch.polar(torch.ones_like(angle), angle)
    y = y.clone()
    y[..., :n], y[..., dist:dist + n] = z.real, z.imag
    return y


def _exact_attend(state, q, k_cache, v_cache):
    case = state["case"]
    hq, hk, d, window = LAYERS[case["layer"]][:4]
    qs, kvs = _lens(case)
    page, outs, lses, at = case["page"], [], [], 0
    for r, (n, kv, (first, last)) in enumerate(zip(qs, kvs, _span(case))):
        j = torch.arange(first, last, device="cuda")
        pages, slots = state["tables"][r].long()[j // page], j % page
        kk, vv = (c[pages, :, slots] for c in (k_cache, v_cache))  # [keys, hk, d]
        i = torch.arange(kv - n, kv, device="cuda")
        hidden = j[None, :] > i[:, None]
        if window:
            hidden = hidden | (i[:, None] - j[None, :] >= window)
        o, l = [], []
        for h in range(hq):
            s = q[at:at + n, h].double() @ kk[:, h // (hq // hk)].double().t() * (state["scale"] * state["k_scale"])
            s = s.masked_fill(hidden, float("-inf"))
            z = torch.logsumexp(s, 1)
            l.append(z)
            o.append(torch.exp(s - z[:, None]) @ vv[:, h // (hq // hk)].double() * state["v_scale"])
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(l, 1))
        at += n
    return torch.cat(outs), torch.cat(lses)


def exact(case, seed):
    state = prepare(case, seed)
    kind, dist = case["kind"], LAYERS[case["layer"]][6]
    if kind == "attend":
        out, lse = _exact_attend(state, state["q"], _wide(state["k_cache"]), _wide(state["v_cache"]))
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    x, k, v = _split(state)
    q = _exact_heads(x, state["q_weight"], state["positions"], state["inv_freq"], dist)
    k = _exact_heads(k, state["k_weight"], state["positions"], state["inv_freq"], dist)
    if kind == "rope":
        return {"q": q, "k": k}
    v = _exact_heads(v, None, None, None, 0)
    k_cache, v_cache = _wide(state["k_cache"]).double(), _wide(state["v_cache"]).double()
    at = 0
    for r, (n, kv) in enumerate(zip(*_lens(case))):
        j = torch.arange(kv - n, kv, device="cuda")
        pages = state["tables"][r].long()[j // case["page"]]
        for cache, new, scale in ((k_cache, k, state["k_scale"]), (v_cache, v, state["v_scale"])):
            cache[pages, :, j % case["page"]] = (new[at:at + n] / scale).clamp(-448, 448) if case["dtype"] == "e4m3" else new[at:at + n]
        at += n
    if kind == "append":
        return {"q": q, "k": k_cache, "v": v_cache}
    out, _ = _exact_attend(state, q, k_cache, v_cache)
    return {"out": out, "k": k_cache, "v": v_cache}


def _wide(cache):
    return cache.bfloat16()
