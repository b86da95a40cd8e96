"""What a serving step with drafted tokens adds around the projections, for timing: page
tables and slot maps made on the GPU, a key/value cache of e4m3 with a scale for each block
of tokens and KV head, the attention over it, and the check of drafted tokens against the
target's probabilities.

Layers are those of the decoder that ``bench.py`` runs (16 query and 8 KV heads of 256, a
window of 1024) and its full-attention layers (16 query heads and one KV head of 512, the
values made from the key projection, a quarter of each head rotated); a few drawn cases have
other head counts.  The vocabulary is the head's 262144, or drawn.

Kinds of case:

* ``pages``: a batch's new tokens get pages and slots (``PagePool.reserve``), then what was
  not kept goes back (``PagePool.release``): a step whose drafts were all refused, or
  prompts that come and go.
* ``append``: one launch that norms and rotates q and appends k and v to block-scaled pages.
* ``attend``: attention of each request's new tokens over such pages.
* ``verify``: drafted tokens of a batch against the logits of their rows.
* ``sample``: a token from each row of logits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
LOW, HIGH = -100, 80  # exponents of a block's scale
# name -> query heads, KV heads, head_dim, window, rope base, rotated pairs, pair distance
LAYERS = {
    "sliding": (16, 8, 256, 1024, 1.0e4, 128, 128),
    "full": (16, 1, 512, 0, 1.0e6, 64, 256),
    "mha128": (8, 8, 128, 0, 1.0e4, 64, 64),
    "gqa128": (12, 4, 128, 333, 1.0e5, 32, 32),
    "gqa64": (32, 4, 64, 0, 1.0e4, 32, 32),
}
VOCAB = 262144


def listed():
    return [
        # the smallest call: one token for each of a few requests, far into their contexts
        {"name": "pages_decode_8", "kind": "pages", "requests": 8, "q_max": 1, "kv_max": 9000, "ragged": True, "page": 64, "window": 1024},
        # prompts and decodes of a large batch over small pages, no window
        {"name": "pages_mixed_96", "kind": "pages", "requests": 96, "q_max": 2048, "kv_max": 32768, "ragged": True, "page": 16, "window": 0},
        # one decoding step of a batch: a token each into blocks that hold some already
        {"name": "append_decode_32", "kind": "append", "layer": "sliding", "requests": 32, "q_max": 1, "kv_max": 60000, "ragged": True, "page": 64, "block": 16},
        # prompts of several requests, ragged, one scale to a block of 32 tokens
        {"name": "append_prompts_5", "kind": "append", "layer": "full", "requests": 5, "q_max": 777, "kv_max": 5000, "ragged": True, "page": 64, "block": 32},
        # a decoding batch over the sliding layers
        {"name": "decode_sliding_64", "kind": "attend", "layer": "sliding", "requests": 64, "q_max": 1, "kv_max": 9000, "ragged": True, "page": 32, "block": 32, "lse": False},
        # a decoding batch over full layers, ragged contexts
        {"name": "decode_full_32", "kind": "attend", "layer": "full", "requests": 32, "q_max": 1, "kv_max": 16000, "ragged": True, "page": 64, "block": 16, "lse": False},
        # blocks of drafted tokens of a few requests, with the log-sum-exp a later merge needs
        {"name": "drafts_full_8", "kind": "attend", "layer": "full", "requests": 8, "q_max": 8, "kv_max": 4100, "ragged": True, "page": 16, "block": 16, "lse": True},
        # a prefill chunk at the end of a 16K prompt, full attention
        {"name": "chunk_full_2048", "kind": "attend", "layer": "full", "requests": 1, "q_max": 2048, "kv_max": 16384, "ragged": False, "page": 64, "block": 64, "lse": False},
        # one user: a token from the head's logits
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": VOCAB, "dtype": "bf16", "softcap": 30.0},
        # a batch without drafts, 32-bit logits
        {"name": "sample_48_f32", "kind": "sample", "rows": 48, "vocab": VOCAB, "dtype": "f32", "softcap": 0.0},
        # drafts of a greedy drafter (no distribution), some requests greedy themselves
        {"name": "verify_greedy_drafts_4", "kind": "verify", "requests": 4, "q_max": 5, "ragged": True, "vocab": VOCAB, "dtype": "bf16", "softcap": 30.0, "drafter": False},
        # a batch of sampled drafts with the drafter's logits
        {"name": "verify_32", "kind": "verify", "requests": 32, "q_max": 8, "ragged": False, "vocab": VOCAB, "dtype": "bf16", "softcap": 0.0, "drafter": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["pages", "append", "append", "attend", "attend", "attend", "verify", "verify", "sample"])
    if kind in ("verify", "sample"):
        vocab = rng.choice([VOCAB, _log_int(rng, 1000, VOCAB)])
        case = {"kind": kind, "vocab": vocab, "dtype": rng.choice(["bf16", "f32"]), "softcap": rng.choice([0.0, 30.0])}
        if kind == "sample":
            return {**case, "rows": _log_int(rng, 1, 224)}
        requests = _log_int(rng, 1, 48)
        # no more bytes than the largest listed case reads
        return {**case, "requests": requests, "q_max": rng.randint(2, max(2, min(16, 120 // requests))), "ragged": rng.choice([True, True, False]),
                "drafter": rng.choice([True, False])}
    shape = rng.choice(["decode", "drafts", "chunk"])
    if shape == "decode":
        requests, q_max = _log_int(rng, 1, 96), 1
    elif shape == "drafts":
        requests, q_max = _log_int(rng, 1, 32), rng.randint(2, 16)
    else:
        requests = rng.choice([1, 1, 2, 5])
        q_max = _log_int(rng, 17, 2048 // requests)
    # scores of the plain form and the caches stay under those of the largest listed cases
    kv_hi = max(64, min(32768, 524288 // requests, 33554432 // (requests * q_max)))
    page = rng.choice([16, 32, 64, 128, 256])
    case = {"kind": kind, "requests": requests, "q_max": q_max, "kv_max": max(q_max, _log_int(rng, 1, kv_hi)), "ragged": rng.choice([True, True, False]),
            "page": page}
    if kind == "pages":
        return {**case, "window": rng.choice([0, 0, 333, 1024])}
    case.update(layer=rng.choice(["sliding", "sliding", "full", "full", "mha128", "gqa128", "gqa64"]),
                block=rng.choice([b for b in (16, 32, 64, 128, 256) if b <= page]))
    if kind == "attend":
        case["lse"] = rng.choice([True, False])
    return case


def _lens(case):
    """(new tokens, tokens in the cache with them) of each request: the case's alone."""
    n, q, kv = case["requests"], case["q_max"], case.get("kv_max", case["q_max"])
    if not case["ragged"]:
        return [q] * n, [kv] * n
    rng = random.Random("%d %d %d" % (n, q, kv))
    qs = [q] + [rng.randint(1, q) if rng.random() < 0.7 else 1 for _ in range(n - 1)]
    return qs, [kv] + [max(a, _log_int(rng, max(1, kv // 40), kv)) for a in qs[1:]]


def _span(case):
    """The positions of each request that a call touches or keeps: [first, kv_len)."""
    window = LAYERS[case["layer"]][3] if "layer" in case else case["window"]
    qs, kvs = _lens(case)
    if case["kind"] == "append":
        return [((kv - q) // case["block"] * case["block"], kv) for q, kv in zip(qs, kvs)]
    return [(max(0, kv - q - window + 1) if window else 0, kv) for q, kv in zip(qs, kvs)]


def _starts(qs):
    starts = [0]
    for q in qs:
        starts.append(starts[-1] + q)
    return starts


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 31)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    rand = lambda *s: torch.rand(s, device="cuda", generator=g)  # noqa: E731
    state = {"case": dict(case)}
    if case["kind"] in ("verify", "sample"):
        _prepare_logits(state, case, randn, rand)
        return state
    qs, kvs = _lens(case)
    rows, page, n = sum(qs), case["page"], len(qs)
    state["rows"] = rows
    width = (max(kvs) + page - 1) // page
    held = [(a // page, (b + page - 1) // page) for a, b in _span(case)]
    if case["kind"] == "pages":
        # held are the tokens of earlier steps; their pages lie in any order, the others are free
        before = [kv - q for q, kv in zip(qs, kvs)]
        held = [(a, (b + page - 1) // page) for (a, _), b in zip(held, before)]
        held = [(min(a, b), b) for a, b in held]
        count = sum((kv + page - 1) // page - a for (a, _), kv in zip(held, kvs)) + 7
    else:
        count = sum(b - a for a, b in held)
    order = torch.randperm(count, device="cuda", generator=g).to(torch.int32).cpu()
    tables = torch.full((n, width), -1, dtype=torch.int32)
    at = 0
    for r, (a, b) in enumerate(held):
        tables[r, a:b] = order[at:at + b - a]
        at += b - a
    state["tables"] = tables.cuda()
    if case["kind"] == "pages":
        free = torch.zeros(count, dtype=torch.int32)
        free[:count - at] = order[at:]
        state.update(free=free.cuda(), free_count=_ints([count - at]), lens=_ints(before), kept=_ints(before), new=_ints(qs),
                     window=case["window"], num_pages=count)
        return state
    hq, hk, d, window, base, pairs, dist = LAYERS[case["layer"]]
    per = page // case["block"]
    # what earlier steps left there: normed keys and values, each block by a scale of its own
    codes = lambda: (randn(count, hk, page, d) * 96).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    scales = lambda: torch.randint(118, 122, (count, hk, per), device="cuda", generator=g).to(torch.uint8).view(torch.float8_e8m0fnu)  # noqa: E731
    state.update(k_cache=codes(), v_cache=codes(), k_scales=scales(), v_scales=scales(), starts=_ints(_starts(qs)), kv_lens=_ints(kvs),
                 window=window, scale=2.0 / math.sqrt(d), q_max=max(qs), kv_max=max(kvs), most_pages=max(b - a for a, b in held),
                 first_page=_ints([a for a, _ in held], torch.int64))
    if case["kind"] == "attend":
        state["q"] = randn(rows, hq, d).bfloat16()
        return state
    # projections leave some heads louder than others
    loud = torch.exp(0.5 * randn(1, hq + 2 * hk, 1))
    state["x"] = (randn(rows, hq + 2 * hk, d) * loud).bfloat16().reshape(rows, -1)
    state["positions"] = _ints([kv - q + i for q, kv in zip(qs, kvs) for i in range(q)])
    state["inv_freq"] = torch.tensor([base ** (-2.0 * i / (2 * dist)) for i in range(pairs)], dtype=torch.float32, device="cuda")
    state["q_weight"], state["k_weight"] = (1 + 0.2 * randn(d)).bfloat16(), (1 + 0.2 * randn(d)).bfloat16()
    return state


def _prepare_logits(state, case, randn, rand):
    kinds = {"bf16": torch.bfloat16, "f32": torch.float32}
    vocab = case["vocab"]
    qs = [1] * case["rows"] if case["kind"] == "sample" else _lens(case)[0]
    rows, n = sum(qs), len(qs)
    # a tail, and some tokens that the context makes likely
    target = randn(rows, vocab) * 2
    likely = (rand(rows, 24) * vocab).long()
    target.scatter_add_(1, likely, 8 + 3 * randn(rows, 24))
    logits = target.to(kinds[case["dtype"]])
    # greedy requests stand beside sampled ones
    state["temperature"] = torch.tensor([0.8, 1.0, 0.0, 0.6], device="cuda")[(rand(n) * 4).long()]
    state.update(rows=rows, logits=logits, softcap=case["softcap"])
    if case["kind"] == "sample":
        state["uniforms"] = rand(rows)
        return
    state["uniforms"] = rand(rows, 2)
    state["starts"] = _ints(_starts(qs))
    # the drafter is near the target; its tokens are drawn from its own distribution
    draft = (target + 0.7 * randn(rows, vocab)).to(kinds[case["dtype"]])
    heat = torch.repeat_interleave(state["temperature"], state["starts"].long().diff(), output_size=rows)[:, None]
    z = _capped(draft.float(), case["softcap"]) / torch.where(heat > 0, heat, torch.ones_like(heat))
    if case["drafter"]:
        z = z - torch.where(heat > 0, torch.log(-torch.log(rand(rows, vocab).clamp(1e-12, 1 - 1e-7))), torch.zeros_like(z))
        state["draft_logits"] = draft
    state["tokens"] = torch.roll(z.argmax(1), 1).to(torch.int32)


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


def _row_request(starts, rows):
    return torch.searchsorted(starts, torch.arange(rows, device="cuda"), right=True) - 1


def _exponents(scales):
    return scales.view(torch.uint8).int() - 127


def _least_exponent(top):
    """The least e with top <= 448 * 2^e."""
    part, e = torch.frexp(top)  # top = part * 2^e, part in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(top > 0, e - 9 + (part > 0.875).int(), LOW).clamp(LOW, HIGH)


def _plain_store(cache, scales, x, pages, slots, block):
    """x [rows, heads, d] into its slots; the blocks' scales grow, and what they held follows."""
    count, hk, page, d = cache.shape
    per = page // block
    by_block = lambda t: t.permute(0, 2, 1, *range(3, t.dim())).flatten(0, 1)  # noqa: E731  [pages * per, heads, ...]
    in_page = lambda t: t.unflatten(0, (count, per)).transpose(1, 2)  # noqa: E731
    raw, was = by_block(cache.view(torch.uint8).unflatten(2, (per, block))), by_block(_exponents(scales))
    unit = pages * per + slots // block  # [rows]
    top = torch.zeros(count * per, hk, device="cuda").index_reduce_(0, unit, x.abs().amax(-1), "amax")
    first = torch.full((count * per,), block, device="cuda").scatter_reduce_(0, unit, slots % block, "amin")[:, None]
    new = torch.maximum(torch.where(first > 0, was, LOW), _least_exponent(top))
    now = torch.where(first < block, new, was)  # blocks without a new token stay
    # what a block held before its first new token, by the new scale
    held = (raw.view(cache.dtype).float() * torch.exp2((was - now).float())[..., None, None]).to(cache.dtype)
    before = (torch.arange(block, device="cuda") < first)[:, None, :, None] & (first < block)[..., None, None]
    raw = torch.where(before, held.view(torch.uint8), raw)
    codes = (x * torch.exp2(-now[unit].float())[..., None]).clamp(-448, 448).to(cache.dtype)
    raw[unit, :, slots % block] = codes.view(torch.uint8)
    cache.view(torch.uint8).unflatten(2, (per, block)).copy_(in_page(raw))
    scales.view(torch.uint8).copy_(in_page((now + 127).to(torch.uint8)))


def _plain_append(state):
    case = state["case"]
    q, k, v = _split(state)
    dist = LAYERS[case["layer"]][6]
    turn = lambda x, w: _rotate(_norm(x, w), state["positions"], state["inv_freq"], dist)  # noqa: E731
    positions, page = state["positions"].long(), case["page"]
    request = _row_request(state["starts"].long(), state["rows"])
    pages, slots = state["tables"][request, positions // page].long(), positions % page
    _plain_store(state["k_cache"], state["k_scales"], turn(k, state["k_weight"]), pages, slots, case["block"])
    _plain_store(state["v_cache"], state["v_scales"], _norm(v, None), pages, slots, case["block"])
    return turn(q, state["q_weight"]).bfloat16()


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

    def take(cache, scales):
        at = pages.clamp(min=0)
        t = cache.view(torch.uint8)[at].view(cache.dtype).float()  # [n, pages, hk, page, d]
        s = torch.exp2(_exponents(scales)[at].float())             # [n, pages, hk, blocks]
        t = t.unflatten(3, (-1, case["block"])) * s[..., None, None]
        return t.flatten(3, 4).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)

    i = torch.arange(q_max, device="cuda")
    token = (starts[:-1, None] + i).clamp(max=state["rows"] - 1)
    rows = q.float()[token].reshape(n, q_max, hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * q_max, d)
    s = torch.matmul(rows, take(state["k_cache"], state["k_scales"]).transpose(2, 3)) * state["scale"]
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
    o = torch.matmul(p, take(state["v_cache"], state["v_scales"]))
    o = o.view(n, hk, group, q_max, d).permute(0, 3, 1, 2, 4).reshape(n, q_max, hq, d)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(n, q_max, hq)
    row = torch.arange(state["rows"], device="cuda")
    request = _row_request(starts, state["rows"])
    at = row - starts[request]
    return o[request, at].bfloat16(), lse[request, at]


def _plain_pages(state):
    page, tables, free, free_count, lens = state["case"]["page"], state["tables"], state["free"], state["free_count"], state["lens"]
    n, width = tables.shape
    # reserve: pages for the new tokens, taken from the end of the free ones
    new, old = state["new"].long(), lens.long()
    starts = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    kv = old + new
    first, end = (old + page - 1) // page, (kv + page - 1) // page
    fits = end <= width
    need = (end - first) * fits
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= free_count))
    j = torch.arange(width, device="cuda")[None, :]
    fresh = granted[:, None] & (j >= first[:, None]) & (j < end[:, None])
    nth = (upto - need)[:, None] + j - first[:, None]
    tables.copy_(torch.where(fresh, free[(free_count - 1 - nth).clamp(0, free.numel() - 1)], tables))
    free_count.sub_((need * granted).sum().int())
    row = torch.arange(state["rows"], device="cuda")
    request = _row_request(starts, state["rows"])
    positions = old[request] + row - starts[request]
    at = tables[request, positions // page].long()
    slots = torch.where(at >= 0, at * page + positions % page, -1)
    out = {"positions": positions.int(), "slots": slots, "starts": starts.int(), "kv_lens": kv.int(), "granted": granted.int()}
    # release: what the kept tokens do not reach goes back, the last one on top
    kept, window = state["kept"].long(), state["window"]
    lo = ((kept - window + 1).clamp(min=0) // page if window else torch.zeros_like(kept))[:, None]
    gone = (tables >= 0) & ((j < lo) | (j >= ((kept + page - 1) // page)[:, None]))
    flat = gone.reshape(-1)
    count = flat.sum()
    nth = free_count + count - 1 - (flat.long().cumsum(0) - 1)
    longer = torch.cat([free, free.new_zeros(1)])
    longer.scatter_(0, torch.where(flat, nth, free.numel()), tables.reshape(-1))
    free.copy_(longer[:-1])
    free_count.add_(count.int())
    tables.copy_(torch.where(gone, -1, tables))
    lens.copy_(kept.int())
    return {**out, "free": free, "free_count": free_count, "tables": tables, "lens": lens}


def _capped(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def _chances(logits, cap, heat):
    """Probabilities in 64 bits; one place only where the temperature is 0."""
    x = logits.double()
    z = _capped(x, cap) / torch.where(heat > 0, heat, torch.ones_like(heat))
    e = torch.exp(z - z.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    best = torch.zeros_like(p).scatter_(1, x.argmax(1, keepdim=True), 1.0)
    return torch.where(heat > 0, p, best)


def _pick(weights, u):
    """The first place where the sum of the weights up to it exceeds u times all of them."""
    upto = weights.cumsum(1)
    places = torch.arange(weights.shape[1], device="cuda")
    last = torch.where(weights > 0, places, 0).amax(1)
    at = torch.searchsorted(upto, upto[:, -1:] * u.double()[:, None], right=True).squeeze(1)
    return torch.minimum(at, last)


def _plain_sample(state):
    heat = state["temperature"].double()[:, None]
    return _pick(_chances(state["logits"], state["softcap"], heat), state["uniforms"]).int()


def _plain_verify(state):
    starts, rows, tokens, u = state["starts"].long(), state["rows"], state["tokens"].long(), state["uniforms"]
    row = torch.arange(rows, device="cuda")
    request = _row_request(starts, rows)
    heat = state["temperature"].double()[request][:, None]
    p = _chances(state["logits"], state["softcap"], heat)
    last = row == starts[request + 1] - 1
    draft = torch.roll(tokens, -1)  # the token that row's distribution has to answer for
    if "draft_logits" in state:
        q = _chances(state["draft_logits"], state["softcap"], heat)
    else:
        q = torch.zeros_like(p).scatter_(1, draft[:, None], 1.0)
    at = lambda t: t.gather(1, draft[:, None]).squeeze(1)  # noqa: E731
    refused = ~last & ~(u[:, 0].double() * at(q) < at(p))
    stop = torch.where(refused | last, row - starts[request], rows)
    accepted = torch.full_like(starts[1:], rows).scatter_reduce_(0, request, stop, "amin")
    spot = starts[:-1] + accepted
    rest = torch.where(last[spot][:, None], p[spot], (p[spot] - q[spot]).clamp(min=0))
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p[spot])
    token = _pick(rest, u[spot, 1])
    i = row - starts[request]
    out = torch.where(i < accepted[request], draft, torch.where(i == accepted[request], token[request], -1))
    return {"tokens": out.int(), "accepted": accepted.int()}


# ---------------------------------------------------------------- the framework's calls

def _held(state):
    """The objects that a server keeps: the pool, the cache, the batch, the rotation and the norms."""
    if "held" not in state:
        from helios_amd import HeadNorm, KVBatch, PagedKVCache, PagePool, Rope

        held = {}
        if "free" in state:
            held["pool"] = PagePool(state["free"], state["free_count"], state["lens"], state["tables"], state["case"]["page"])
        if "k_cache" in state:
            held["cache"] = PagedKVCache(state["k_cache"], state["v_cache"], state["k_scales"], state["v_scales"])
            held["batch"] = KVBatch(state["starts"], state["kv_lens"], state["tables"])
        if "x" in state:
            held.update(rope=Rope(state["inv_freq"], LAYERS[state["case"]["layer"]][6]), q_norm=HeadNorm(state["q_weight"], EPS),
                        k_norm=HeadNorm(state["k_weight"], EPS), v_norm=HeadNorm(None, EPS))
        state["held"] = held
    return state["held"]


def _own_pages(state):
    pool = _held(state)["pool"]
    positions, slots = pool.reserve(state["new"], state["rows"])
    pool.release(state["kept"], window=state["window"])
    return {"positions": positions, "slots": slots, "starts": pool.batch.query_starts, "kv_lens": pool.batch.kv_lens, "granted": pool.granted,
            "free": pool.free_pages, "free_count": pool.free_count, "tables": pool.block_tables, "lens": pool.lens}


def _own_append(state):
    h = _held(state)
    q, k, v = _split(state)
    return h["cache"].append(k, v, h["batch"], rope=h["rope"], k_norm=h["k_norm"], v_norm=h["v_norm"], q=q, q_norm=h["q_norm"])


def _own_attend(state):
    h = _held(state)
    return h["cache"].attend(state["q"], h["batch"], scale=state["scale"], window=state["window"], return_lse=state["case"]["lse"])


def _own_sample(state):
    from helios_amd import sample

    return sample(state["logits"], state["uniforms"], state["temperature"], softcap=state["softcap"])


def _own_verify(state):
    from helios_amd import verify_drafts

    tokens, accepted = verify_drafts(state["logits"], state["tokens"], state["starts"], state["uniforms"], state["temperature"],
                                     draft_logits=state.get("draft_logits"), softcap=state["softcap"], draft_softcap=state["softcap"])
    return {"tokens": tokens, "accepted": accepted}


def run(state):
    kind = state["case"]["kind"]
    if kind == "pages":
        return _own_pages(state) if own else _plain_pages(state)
    if kind == "sample":
        return {"tokens": _own_sample(state) if own else _plain_sample(state)}
    if kind == "verify":
        return _own_verify(state) if own else _plain_verify(state)
    if kind == "append":
        q = _own_append(state) if own else _plain_append(state)
        return {"q": q, "k": state["k_cache"], "v": state["v_cache"], "k_scales": state["k_scales"], "v_scales": state["v_scales"]}
    if own:
        got = _own_attend(state)
        return {"out": got[0], "lse": got[1]} if state["case"]["lse"] else {"out": got}
    out, lse = _plain_attend(state, state["q"])
    return {"out": out, "lse": lse} if state["case"]["lse"] else {"out": out}


def work(case):
    kind = case["kind"]
    if kind in ("verify", "sample"):
        rows = case["rows"] if kind == "sample" else sum(_lens(case)[0])
        n = rows if kind == "sample" else case["requests"]
        size = 2 if case["dtype"] == "bf16" else 4
        # the last row of a request has no draft to answer for
        drafted = rows - n if case.get("drafter") else 0
        return {"bytes": (rows + drafted) * case["vocab"] * size + 16 * rows + 12 * n, "flops": 4 * (rows + drafted) * case["vocab"]}
    qs, kvs = _lens(case)
    rows, n, page = sum(qs), len(qs), case["page"]
    if kind == "pages":
        fresh = sum((kv + page - 1) // page - (kv - q + page - 1) // page for q, kv in zip(qs, kvs))
        # lengths in and out, each new page off the stack, into a table, and back, a position and a slot a row
        return {"bytes": 12 * rows + 24 * n + 16 * fresh, "flops": 4 * rows + 8 * n}
    hq, hk, d, window = LAYERS[case["layer"]][:4]
    block = case["block"]
    if kind == "append":
        heads_in = hq + hk if case["layer"] == "full" else hq + 2 * hk
        blocks = sum((kv + block - 1) // block - (kv - q) // block for q, kv in zip(qs, kvs))
        return {"bytes": rows * d * (2 * heads_in + 2 * hq + 2 * hk) + 4 * blocks * hk, "flops": 8 * rows * d * (hq + 2 * hk)}
    pairs = keys = blocks = tables = 0
    for q, kv, (first, last) in zip(qs, kvs, _span(case)):
        keys += last - first
        blocks += (last + block - 1) // block - first // block
        tables += (last + page - 1) // page - first // page
        for p in range(kv - q, kv):
            pairs += min(p + 1, window) if window else p + 1
    return {"bytes": 2 * keys * hk * d + 2 * blocks * hk + 4 * rows * hq * d + 4 * tables + (4 * rows * hq if case["lse"] else 0),
            "flops": 4 * d * hq * pairs}


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


def _exact_append(state):
    case = state["case"]
    page, block, dist = case["page"], case["block"], LAYERS[case["layer"]][6]
    x, k, v = _split(state)
    where = (state["positions"], state["inv_freq"], dist)
    new = {"k": _exact_heads(k, state["k_weight"], *where), "v": _exact_heads(v, None, None, None, 0)}
    out = {"q": _exact_heads(x, state["q_weight"], *where)}
    tables = state["tables"].tolist()
    for which in ("k", "v"):
        codes = state[which + "_cache"].float().double()
        size = torch.exp2(state[which + "_scales"].view(torch.uint8).double() - 127)
        at = 0
        for r, (n, kv) in enumerate(zip(*_lens(case))):
            p = kv - n
            while p < kv:
                b0 = p // block * block
                end = min(kv, b0 + block)
                rows = new[which][at:at + end - p].transpose(0, 1)  # [heads, tokens, d]
                pg, unit, slot = tables[r][b0 // page], b0 % page // block, b0 % page
                top = rows.abs().flatten(1).amax(1).clamp(min=448 * 2.0 ** LOW)
                least = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(LOW, HIGH))
                was = size[pg, :, unit] if p > b0 else torch.zeros_like(least)
                now = torch.maximum(was, least)
                if p > b0:
                    codes[pg, :, slot:slot + p - b0] *= (was / now)[:, None, None]
                codes[pg, :, slot + p - b0:slot + end - b0] = rows / now[:, None, None]
                size[pg, :, unit] = now
                at, p = at + end - p, end
        out[which], out[which + "_scales"] = codes, size
    return out


def _exact_attend(state):
    case = state["case"]
    hq, hk, d, window = LAYERS[case["layer"]][:4]
    page, block = case["page"], case["block"]
    outs, lses, at = [], [], 0
    wide = [(c.bfloat16(), s.view(torch.uint8).double()) for c, s in ((state["k_cache"], state["k_scales"]), (state["v_cache"], state["v_scales"]))]
    for r, (n, kv, (first, last)) in enumerate(zip(*_lens(case), _span(case))):
        j = torch.arange(first, last, device="cuda")
        pages, slots = state["tables"][r].long()[j // page], j % page
        kk, vv = (c[pages, :, slots].double() * torch.exp2(s[pages, :, slots // block] - 127)[..., None] for c, s in wide)  # [keys, hk, d]
        i = torch.arange(kv - n, kv, device="cuda")
        hidden = j[None, :] > i[:, None]
        if window:
            hidden = hidden | (i[:, None] - j[None, :] >= window)
        o, l = [], []
        for h in range(hq):
            s = state["q"][at:at + n, h].double() @ kk[:, h // (hq // hk)].t() * state["scale"]
            s = s.masked_fill(hidden, float("-inf"))
            z = torch.logsumexp(s, 1)
            l.append(z)
            o.append(torch.exp(s - z[:, None]) @ vv[:, h // (hq // hk)])
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(l, 1))
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)} if case["lse"] else {"out": torch.cat(outs)}


def exact(case, seed):
    if case["kind"] in ("pages", "verify", "sample"):
        return None  # whole numbers
    state = prepare(case, seed)
    return _exact_append(state) if case["kind"] == "append" else _exact_attend(state)
