"""Tokens from logits and drafted tokens checked against them, on the GPU, against the
definitions in float64 on the host: tokens and counts have to be equal.  A token is a place in
a cumulative sum, found in float64 on both sides (about 1e-15 apart), so two of them differ
with a probability of some vocab * 1e-15 a draw."""

import numpy as np
import pytest

from pooled_streams import streams  # noqa: F401

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def chances(x, heat, cap=0.0):
    """p of one row of float64 logits; all zero where none has any."""
    live = x > -np.inf
    p = np.zeros(x.shape)
    if not live.any():
        return p
    if not heat > 0:
        p[int(np.where(live, x, -np.inf).argmax())] = 1.0
        return p
    top = x[live].max()
    if np.isinf(top):
        p[x == top] = 1.0
        return p / p.sum()
    z = (cap * np.tanh(x[live] / cap) if cap else x[live]) / heat
    e = np.exp(z - z.max())
    p[live] = e / e.sum()
    return p


def pick(w, u):
    at = np.nonzero(w > 0)[0]
    if at.size == 0:
        return -1
    upto = np.cumsum(w)
    past = np.nonzero(upto > float(u) * upto[-1])[0]
    past = past[w[past] > 0] if past.size else past
    return int(past[0]) if past.size else int(at[-1])


def verify(x, tokens, starts, u, heats, y=None, cap=0.0, draft_cap=0.0):
    rows, vocab = x.shape
    out, accepted = np.full(rows, -1), np.zeros(len(starts) - 1, np.int64)
    for r, heat in enumerate(heats):
        a, b = starts[r], starts[r + 1]
        for i in range(a, b):
            p = chances(x[i], heat, cap)
            if i == b - 1:
                out[i] = pick(p, u[i, 1])
                break
            d = int(tokens[i + 1])
            q = chances(y[i], heat, draft_cap) if y is not None else np.eye(1, vocab, d)[0] if 0 <= d < vocab else np.zeros(vocab)
            inside = 0 <= d < vocab
            q_d = 1.0 if y is None else (q[d] if inside else 0.0)
            if inside and float(u[i, 0]) * q_d < p[d]:
                out[i] = d
                accepted[r] += 1
                continue
            rest = np.clip(p - q, 0, None)
            out[i] = pick(rest if rest.sum() > 0 else p, u[i, 1])
            break
    return out, accepted


def logits(rng, rows, vocab, dtype):
    """A tail and a few likely tokens, as float64 and on the device."""
    x = rng.standard_normal((rows, vocab)) * 2
    for r in range(rows):
        x[r, rng.integers(0, vocab, 8)] += 6
    t = dev(x.astype(np.float32), dtype)
    return t, t.float().cpu().numpy().astype(np.float64)


def kinds():
    import torch

    return {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 255), (4, 2048), (4, 2049), (70, 4097), (3, 50001), (33, 8191), (260, 16385), (1, 262144),
                                        (40, 262144)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_sample(gpu_lib, rows, vocab, kind, cap):
    from helios_amd import sample

    rng = np.random.default_rng(rows * 7 + vocab)
    t, x = logits(rng, rows, vocab, kinds()[kind])
    u = rng.random(rows).astype(np.float32)
    u[0] = 0.0
    heats = rng.choice([0.0, 0.3, 1.0, 2.5], rows).astype(np.float32)
    got = sample(t, dev(u), dev(heats), softcap=cap).tolist()
    assert got == [pick(chances(x[r], heats[r], cap), u[r]) for r in range(rows)]
    assert sample(t, dev(u), dev(heats), softcap=cap).tolist() == got
    one = sample(t, dev(u), 0.7, softcap=cap).tolist()
    assert one == [pick(chances(x[r], np.float32(0.7), cap), u[r]) for r in range(rows)]
    assert sample(t, dev(u), 0.0).tolist() == x.argmax(1).tolist()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,heat", [(17, 1.0), (4100, 1.0), (4100, 0.05), (262144, 1.0)])
def test_every_place_can_be_drawn(gpu_lib, vocab, heat, kind):
    """Uniforms over [0, 1) on one distribution: each token as the host finds it, at borders too."""
    from helios_amd import sample

    rng = np.random.default_rng(vocab)
    t, x = logits(rng, 1, vocab, kinds()[kind])
    p = chances(x[0], heat)
    upto = np.cumsum(p)
    inside = (upto[:-1] + upto[1:])[:: max(1, vocab // 60)] / 2  # the middle of places' ranges
    u = np.concatenate([inside, rng.random(60), [0.0, np.nextafter(np.float32(1), np.float32(0))]]).astype(np.float32)
    u = u[u < 1]
    got = sample(t.expand(len(u), vocab).contiguous(), dev(u), heat).tolist()
    # Uniforms made from the sums themselves lie on borders, where two float64 sums may differ: a
    # weight is off by (2 z + 4) half steps of 2^-52 (the quotient z, up to |x| / T, and the
    # exponential), a sum of n terms by n more, on either side.  Off a border the token is the host's.
    z = np.abs(x[0]).max() * 2 / heat
    off = 2 * (2 * z + 4 + vocab) * 2.0 ** -53
    before = np.concatenate([[0], upto[:-1]])
    for v, token in zip(u.astype(np.float64), got):
        assert token == pick(p, v) or (p[token] > 0 and before[token] - off <= v <= upto[token] + off), (v, token, pick(p, v))
    assert sum(token != pick(p, v) for v, token in zip(u, got)) <= len(u) // 4


def test_rows_of_masks(gpu_lib):
    """-inf everywhere, in all places but one, the type's lowest value, infinities, NaN."""
    import torch

    from helios_amd import sample

    vocab = 5000
    x = np.full((8, vocab), -np.inf, np.float32)
    x[1, 4321] = -50.0
    x[3, 7:9] = np.inf
    x[3, 100] = 5
    x[4] = np.nan
    x[4, 17] = 1.0
    x[5] = np.nan
    x[6] = -3.0e38
    x[6, 4999] = 3.0e38
    x[7, [3, 2060, 4090]] = 2.0
    for cap in (0.0, 30.0):
        for kind in kinds().values():
            t = dev(x, kind)
            t[2] = torch.finfo(kind).min  # (float32's would round to -inf in bf16)
            u = np.array([0.5, 0.5, 0.5, 0.75, 0.9, 0.1, 0.3, 0.5], np.float32)
            got = sample(t, dev(u), 1.0, softcap=cap).tolist()
            assert got[:2] == [-1, 4321] and got[2] == vocab // 2
            assert got[3] == (8 if cap == 0 else got[3]) and got[3] in (7, 8)
            assert got[4] == 17 and got[5] == -1 and got[7] == 2060
            if cap == 0:
                assert got[6] == 4999
            assert sample(t, dev(u), 0.0, softcap=cap).tolist() == [-1, 4321, 0, 7, 17, -1, 4999, 3]
    # uniforms that are none: a token with a probability all the same
    t = dev(np.where(np.arange(vocab) % 3 == 0, 0.0, -np.inf).astype(np.float32)[None].repeat(4, 0), torch.float32)
    assert sample(t, dev(np.array([1.0, 7.0, -1.0, np.nan], np.float32))).tolist() == [4998, 4998, 0, 4998]


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(4, 5000), (260, 16385)])
@pytest.mark.parametrize("cap,draft_cap", [(0.0, 0.0), (30.0, 30.0), (30.0, 0.0), (0.0, 20.0)])
def test_masks_among_logits(gpu_lib, rows, vocab, kind, cap, draft_cap):
    """NaN and -inf beside ordinary logits, of the target and of the drafter, have no part in the sums."""
    from helios_amd import sample, verify_drafts

    rng = np.random.default_rng(rows + vocab)
    starts, heats = np.arange(0, rows + 1, 4), np.full(rows // 4, 0.8, np.float32)
    t, x = logits(rng, rows, vocab, kinds()[kind])
    y, tokens = drafts(rng, x, heats, starts, 0.3)
    yt = dev(y.astype(np.float32), kinds()[kind])
    for one in (t, yt):
        for mask in (np.nan, -np.inf):
            one[dev(rng.random((rows, vocab)) < 0.1)] = mask
    x, y = (one.float().cpu().numpy().astype(np.float64) for one in (t, yt))
    u = rng.random((rows, 2)).astype(np.float32)
    assert sample(t, dev(u[:, 0]), 0.8, softcap=cap).tolist() == [pick(chances(x[r], np.float32(0.8), cap), u[r, 0]) for r in range(rows)]
    got, count = verify_drafts(t, dev(tokens), dev(starts.astype(np.int32)), dev(u), dev(heats), draft_logits=yt, softcap=cap, draft_softcap=draft_cap)
    want, accepted = verify(x, tokens, starts, u, heats, y, cap, draft_cap)
    assert count.tolist() == accepted.tolist() and got.tolist() == want.tolist()


@pytest.mark.parametrize("rows,vocab", [(3, 6000), (200, 30000)])
def test_far_temperatures_and_logits(gpu_lib, rows, vocab):
    """Quotients of 2^40 and more, temperatures near both ends of float32: ties alone, or all alike."""
    import torch

    from helios_amd import sample

    places = [5, vocab // 2, vocab - 2]
    for kind in kinds().values():
        x = torch.zeros(rows, vocab, device="cuda", dtype=kind)
        x[:, places] = 2.0 ** 41
        for u, want in ((0.0, 0), (0.3, 0), (0.5, 1), (0.7, 2), (0.99, 2)):
            uu = torch.full((rows,), u, device="cuda")
            for t, heat in ((x, 1.0), (x, 4.0), (x, 1e-3), (x / 2 ** 41, 1e-42), (x / 2 ** 41, 1e-38), (x * 2.0 ** 80, 1e30)):
                assert sample(t, uu, heat).tolist() == [places[want]] * rows, (u, heat)
            # all weights are 1 to the last bit: the first place whose number of weights exceeds u n
            assert sample(x / 2 ** 41, uu, 3e38).tolist() == [int(np.float64(np.float32(u)) * vocab)] * rows


def test_large_vocabularies(gpu_lib):
    """More parts to a row than a workgroup has threads, and the largest vocabulary."""
    from helios_amd import sample, verify_drafts

    rng = np.random.default_rng(11)
    for vocab in (1 << 21, (1 << 20) + 12345, 1 << 24):
        x = (rng.standard_normal((3, vocab), np.float32) * 0.5).astype(np.float32)
        x[:, -1] += 12.0
        t, x = dev(x), x.astype(np.float64)
        p = [chances(v, 1.0) for v in x]
        for u in ([0.0, 0.31, 0.999], [0.5, 0.05, 0.77]):
            u = np.array(u, np.float32)
            assert sample(t, dev(u)).tolist() == [pick(p[r], u[r]) for r in range(3)]
            assert sample(t, dev(u), 0.0).tolist() == x.argmax(1).tolist()
        tokens, starts = np.array([1, vocab - 1, 5], np.int32), np.array([0, 3])
        for u in ([[0.0, 0.3], [0.99, 0.6], [0.1, 0.2]], [[0.999, 0.4], [0.0, 0.0], [0.0, 0.0]]):
            u = np.array(u, np.float32)
            for y in (None, x[::-1].copy()):
                got, count = verify_drafts(t, dev(tokens), dev(starts.astype(np.int32)), dev(u), 1.0,
                                           draft_logits=None if y is None else t.flip(0).contiguous())
                want, accepted = verify(x, tokens, starts, u, [1.0], y)
                assert got.tolist() == want.tolist() and count.tolist() == accepted.tolist()


def test_two_threads_two_streams(gpu_lib, streams):
    """Calls of two threads, each on a stream of its own, keep out of each other's scratch memory."""
    import threading

    import torch

    from helios_amd import sample, verify_drafts

    rng = np.random.default_rng(13)
    work = []
    for rows in (12, 64):
        t, _ = logits(rng, rows, 60000, torch.bfloat16)
        y, _ = logits(rng, rows, 60000, torch.bfloat16)
        starts = dev(np.arange(0, rows + 1, 4).astype(np.int32))
        tokens, u = dev(rng.integers(0, 60000, rows).astype(np.int32)), dev(rng.random((rows, 2)).astype(np.float32))
        want = verify_drafts(t, tokens, starts, u, draft_logits=y) + (sample(t, u[:, 0].contiguous()),)
        work.append((t, y, starts, tokens, u, want, streams()))
    torch.cuda.synchronize()
    failed = []

    def run(t, y, starts, tokens, u, want, stream):
        try:
            for _ in range(50):
                with torch.cuda.stream(stream):
                    first = u[:, 0].contiguous()
                got = verify_drafts(t, tokens, starts, u, draft_logits=y, stream=stream) + (sample(t, first, stream=stream),)
                stream.synchronize()
                assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_captured_sampling(gpu_lib, streams):
    """A captured call draws anew from what its inputs hold at the replay."""
    import torch

    from helios_amd import sample

    rng = np.random.default_rng(17)
    x, u, heats = torch.zeros(3, 40000, device="cuda"), torch.zeros(3, device="cuda"), torch.ones(3, device="cuda")
    stream = streams()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sample(x, u, heats)  # takes the stream's scratch memory before the capture
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = sample(x, u, heats)
    for _ in range(8):
        x.copy_(torch.from_numpy(rng.standard_normal((3, 40000), np.float32)))
        u.copy_(torch.from_numpy(rng.random(3, np.float32)))
        heats.copy_(torch.from_numpy(rng.choice(np.array([0, 0.5, 1], np.float32), 3)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sample(x, u, heats))
        torch.rand(1000, device="cuda").sum().item()  # work of the program's own between replays


def test_ties_and_saturated_softcap(gpu_lib):
    """Greedy: the first of equals, whatever the chunk; logits far past the softcap keep their order."""
    from helios_amd import sample

    for vocab in (9000, 262144):
        x = np.zeros((3, vocab), np.float32)
        x[0, [vocab - 1, 5000, 8999]] = 4.0
        x[1, vocab - 1] = 2000.0
        x[1, 3] = 1000.0
        for kind in kinds().values():
            assert sample(dev(x, kind), dev(np.zeros(3, np.float32)), 0.0, softcap=30.0).tolist() == [5000, vocab - 1, 0]


def drafts(rng, x, heats, starts, near):
    """A drafter's logits near the target's and tokens drawn from them."""
    y = x + near * rng.standard_normal(x.shape)
    y = y.astype(np.float32).astype(np.float64)
    tokens = np.zeros(len(x), np.int32)
    for r, heat in enumerate(heats):
        for i in range(starts[r], starts[r + 1] - 1):
            tokens[i + 1] = pick(chances(y[i], heat), rng.random())
        if starts[r + 1] > starts[r]:
            tokens[starts[r]] = rng.integers(0, x.shape[1])
    return y, tokens


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("lens,vocab", [([1], 100), ([2], 2049), ([5, 1, 0, 8, 3], 5000), ([16], 20001), ([4] * 70, 1000), ([5, 4, 5, 5], 262144)])
@pytest.mark.parametrize("drafter", ["logits", "none"])
def test_verify(gpu_lib, lens, vocab, kind, drafter):
    from helios_amd import verify_drafts

    rng = np.random.default_rng(sum(lens) + vocab)
    padding = 2
    starts = np.concatenate([[0], np.cumsum(lens)])
    rows = int(starts[-1]) + padding
    t, x = logits(rng, rows, vocab, kinds()[kind])
    heats = rng.choice([0.0, 0.5, 1.0, 1.7], len(lens)).astype(np.float32)
    y, tokens = drafts(rng, x, heats, starts, 0.5)
    yt = dev(y.astype(np.float32), kinds()[kind])
    y = yt.float().cpu().numpy().astype(np.float64)
    for trial in range(4):
        u = rng.random((rows, 2)).astype(np.float32) * (1.0 if trial else 0.3)  # the first time most drafts stand
        cap = 30.0 if trial == 2 else 0.0
        draft_cap = 20.0 if trial >= 2 else 0.0
        given = dict(draft_logits=yt, draft_softcap=draft_cap) if drafter == "logits" else {}
        got, count = verify_drafts(t, dev(tokens), dev(starts.astype(np.int32)), dev(u), dev(heats), softcap=cap, **given)
        want, accepted = verify(x, tokens, starts, u, heats, y if drafter == "logits" else None, cap, draft_cap)
        assert count.tolist() == accepted.tolist()
        assert got.tolist() == want.tolist()


def test_equal_distributions_always_stand(gpu_lib):
    """p and q from the same logits are the same numbers: any uniform under 1 accepts."""
    import torch

    from helios_amd import verify_drafts

    rng = np.random.default_rng(1)
    for vocab in (300, 40000):
        t, x = logits(rng, 6, vocab, torch.bfloat16)
        tokens = np.array([pick(chances(r, 1.0), 0.4) for r in x], np.int32)
        u = np.full((6, 2), np.nextafter(np.float32(1), np.float32(0)), np.float32)
        got, count = verify_drafts(t, dev(tokens), dev(np.array([0, 6], np.int32)), dev(u), 1.0, draft_logits=t)
        assert count.tolist() == [5] and got[:5].tolist() == tokens[1:].tolist()


def test_borders_of_acceptance(gpu_lib):
    """u q against p where they are equal: with p and q exact in binary, equality refuses."""
    import torch

    from helios_amd import verify_drafts

    # p: four equal logits of a row, 1/4 each; no drafter's logits: u < 1/4 accepts
    x = torch.full((2, 64), float("-inf"), device="cuda")
    x[:, 10:14] = 0.0
    tokens, starts = dev(np.array([0, 12], np.int32)), dev(np.array([0, 2], np.int32))
    for u, want in ((0.25, 0), (np.nextafter(np.float32(0.25), np.float32(0)), 1), (0.0, 1)):
        uu = dev(np.array([[u, 0.5], [0.0, 0.0]], np.float32))
        got, count = verify_drafts(x, tokens, starts, uu, 1.0)
        assert count.tolist() == [want]
        # the refused one has no weight left: the middle of 10, 11 and 13
        assert got.tolist() == ([12, 10] if want else [11, -1])
    # a draft that the target cannot give, and ones that are no tokens
    for bad in (3, -1, 64, 2 ** 31 - 1, -2 ** 31):
        got, count = verify_drafts(x, dev(np.array([0, bad], np.int32)), starts, dev(np.zeros((2, 2), np.float32)), 1.0)
        assert count.tolist() == [0] and got.tolist() == [10, -1]


def test_greedy_verification(gpu_lib):
    """Temperature 0: a draft stands where it is the first largest logit, whatever the uniforms."""
    import torch

    from helios_amd import verify_drafts

    rng = np.random.default_rng(4)
    t, x = logits(rng, 8, 30000, torch.bfloat16)
    best = x.argmax(1)
    for wrong in range(8):
        tokens = np.concatenate([[0], best[:7]]).astype(np.int32)
        if wrong:
            tokens[wrong] = (tokens[wrong] + 1) % 30000
        u = dev(rng.random((8, 2)).astype(np.float32))
        for more in ({}, {"draft_logits": dev(rng.standard_normal((8, 30000)).astype(np.float32), torch.bfloat16)}):
            got, count = verify_drafts(t, dev(tokens), dev(np.array([0, 8], np.int32)), u, 0.0, **more)
            n = wrong - 1 if wrong else 7
            assert count.tolist() == [n]
            assert got.tolist() == best[:n + 1].tolist() + [-1] * (7 - n)


def test_the_target_distribution_is_kept(gpu_lib):
    """Whatever the drafter, the first token of a block is distributed as the target's: 20000
    blocks of one draft over 5 tokens, counts within five standard deviations."""
    import torch

    from helios_amd import verify_drafts

    rng = np.random.default_rng(6)
    x, y = np.array([1.0, 0.0, -1.0, 2.0, 0.5]), np.array([0.0, 2.0, -1.0, 0.5, -np.inf])
    p, q = chances(x, 1.0), chances(y, 1.0)
    n = 20000
    tokens = np.zeros(2 * n, np.int32)
    tokens[1::2] = rng.choice(5, n, p=q)
    rows = lambda v: dev(np.tile(v, (2 * n, 1)).astype(np.float32), torch.float32)  # noqa: E731
    got, _ = verify_drafts(rows(x), dev(tokens), dev(np.arange(0, 2 * n + 1, 2, dtype=np.int32)), dev(rng.random((2 * n, 2)).astype(np.float32)), 1.0,
                           draft_logits=rows(y))
    counts = np.bincount(got.cpu().numpy()[::2], minlength=5)
    assert np.all(np.abs(counts - n * p) <= 5 * np.sqrt(n * p * (1 - p))), (counts, n * p)


def test_strides_and_alignment(gpu_lib):
    """Rows of a wider tensor, at odd offsets, of odd lengths."""
    from helios_amd import sample, verify_drafts

    rng = np.random.default_rng(9)
    for kind in kinds().values():
        for vocab, offset, width in ((5001, 1, 5010), (4096, 3, 4103), (2047, 0, 2048), (8192, 8, 8200), (999, 5, 1004)):
            t, x = logits(rng, 6, width, kind)
            t, x = t[:, offset:offset + vocab], x[:, offset:offset + vocab]
            u = rng.random((6, 2)).astype(np.float32)
            assert sample(t, dev(u[:, 0]), 1.0).tolist() == [pick(chances(x[r], 1.0), u[r, 0]) for r in range(6)]
            starts = np.array([0, 4, 6])
            y, tokens = drafts(rng, x, [1.0, 1.0], starts, 0.4)
            yt = dev(y.astype(np.float32), kind)
            got, count = verify_drafts(t, dev(tokens), dev(starts.astype(np.int32)), dev(u), 1.0, draft_logits=yt)
            want, accepted = verify(x, tokens, starts, u, [1.0, 1.0], yt.float().cpu().numpy().astype(np.float64))
            assert got.tolist() == want.tolist() and count.tolist() == accepted.tolist()


def test_empty_calls_and_starts_that_are_none(gpu_lib):
    import torch

    from helios_amd import sample, verify_drafts

    z = torch.zeros(0, 100, device="cuda")
    assert sample(z, torch.zeros(0, device="cuda")).shape == (0,)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    out, accepted = verify_drafts(z, ints().int(), ints(0, 0, 0), torch.zeros(0, 2, device="cuda"))
    assert out.shape == (0,) and accepted.tolist() == [0, 0]
    # starts past the rows, falling ones, a first one that is not 0: clamped
    x = torch.randn(4, 100, device="cuda")
    u = torch.rand(4, 2, device="cuda")
    for starts in ((0, 100), (0, 3, 1, 4), (2, 4), (-5, 4), (0, 0, 0)):
        out, accepted = verify_drafts(x, ints(1, 2, 3, 4), ints(*starts), u)
        assert bool((accepted >= 0).all()) and bool((accepted < 4).all())
    out, _ = verify_drafts(x, ints(1, 2, 3, 4), ints(0, 0, 0), u)
    assert out.tolist() == [-1] * 4


def test_refusals(gpu_lib):
    import torch

    from helios_amd import Gemma4Error, sample, verify_drafts

    x, u = torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda")
    for args in ((x.half(), u), (x[0], u), (x.t(), u), (x.cpu(), u), (x, u[:3]), (x, u.double()), (x, u.cpu()), (x, u, -1.0), (x, u, float("nan")),
                 (x, u, u[:2]), (x, u, 1.0, -3.0), (x, u, 1.0, float("inf")), (x[:, :0], u)):
        with pytest.raises(Gemma4Error):
            sample(*args)
    ints = torch.zeros(4, dtype=torch.int32, device="cuda")
    u2 = torch.zeros(4, 2, device="cuda")
    verify_drafts(x, ints, ints[:2], u2)
    for args, kw in (((x, ints[:3], ints[:2], u2), {}), ((x, ints.long(), ints[:2], u2), {}), ((x, ints, ints[:1], u2), {}), ((x, ints, ints[:0], u2), {}),
                     ((x, ints, ints[:2], u), {}), ((x, ints, ints[:2], u2, u), {}), ((x, ints, ints[:2], u2), dict(draft_logits=x[:, :9])),
                     ((x, ints, ints[:2], u2), dict(draft_logits=x.bfloat16())), ((x, ints, ints[:2], u2), dict(draft_logits=x, draft_softcap=-1.0))):
        with pytest.raises(Gemma4Error):
            verify_drafts(*args, **kw)
