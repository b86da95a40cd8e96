"""Sampling and verification at the ends of what they take, on the GPU against the definitions in
float64 (or in decimals of 60 digits) on the host: uniforms of 0 and from 1 on beside places without
weight, temperatures and softcaps over float32's range.

Tokens have to be equal: uniforms are drawn at random, and a token differs only where one lies within the
kernels' error of a border (2e-13 of the sum, with a softcap up to 3e-9), which happens once in 10^5 runs
with other numbers than these."""

import decimal

import numpy as np
import pytest

from test_gpu_sampling import chances, dev, drafts, pick, verify

pytestmark = pytest.mark.gpu

ONE_LESS = np.nextafter(np.float32(1), np.float32(0))
# rows and vocabularies whose rows are cut into parts of 512, and of 2048
SIZES = [(2, 3000, 512), (512, 8192, 2048)]


def test_the_first_of_two_neighbours(gpu_lib):
    """A uniform of 0 takes the first place with any weight, however little beside the next one's."""
    from helios_amd import sample

    for vocab in (600, 5000):
        for at in (0, 1, 2, 510, 511, 512, 513, 590):
            x = np.full((1, vocab), -np.inf, np.float32)
            x[0, at] = -60.0
            x[0, at + 1:at + 3] = 0.0
            u = dev(np.zeros(1, np.float32))
            assert sample(dev(x), u, 1.0).tolist() == [at], at
            assert sample(dev(x), u, 1.0, softcap=100.0).tolist() == [at], at


def blocks(rows):
    """Requests of two rows: one draft each."""
    return np.arange(0, rows + 1, 2)


def check(x, tokens, starts, u, heats, y=None, cap=0.0):
    """verify_drafts of float64 logits that are exact in float32, against the host's."""
    from helios_amd import verify_drafts

    on_gpu = lambda v: dev(v.astype(np.float32))  # noqa: E731
    given = {} if y is None else dict(draft_logits=on_gpu(y), draft_softcap=cap)
    got, count = verify_drafts(on_gpu(x), dev(tokens), dev(starts.astype(np.int32)), dev(u), dev(heats), softcap=cap, **given)
    want, accepted = verify(x, tokens, starts, u, heats, y, cap, cap)
    assert count.tolist() == accepted.tolist()
    assert got.tolist() == want.tolist()
    return got, count


@pytest.mark.parametrize("rows,vocab,size", SIZES)
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("end", ["first", "last"])
def test_parts_of_nothing_with_a_drafter(gpu_lib, rows, vocab, size, cap, end):
    """Parts that are masked in both, or far below, have no remainder, whatever u: the token comes
    from the others (the first with any at 0, the last from 1 on)."""
    rng = np.random.default_rng(rows + vocab)
    x = np.round(rng.standard_normal((rows, vocab)) * 8) / 8
    y = x * 0.5
    here = slice(0, size) if end == "first" else slice(vocab - size, vocab)
    kind = rng.integers(0, 3, size)
    low = np.where(kind == 0, -np.inf, np.where(kind == 1, np.nan, -3000.0 if not cap else -np.inf))
    x[:, here] = y[:, here] = low
    middle = np.arange(size + 4, vocab - size)
    tokens = rng.choice(middle, rows).astype(np.int32)
    x[np.arange(rows - 1), tokens[1:]] = -5.0  # every draft falls
    y[np.arange(rows - 1), tokens[1:]] = 9.0
    x[:, size + 3] = 19.0  # the target is the more certain one
    starts, heats = blocks(rows), np.full(rows // 2, 0.7, np.float32)
    u = np.zeros((rows, 2), np.float32)
    u[:, 0] = ONE_LESS
    for v in (0.0, 1.0, 7.0, 0.5):
        u[:, 1] = v
        got, count = check(x, tokens, starts, u, heats, y, cap)
        assert int(count.sum()) == 0 and bool((got[::2] >= 0).all())


@pytest.mark.parametrize("rows,vocab,size", SIZES)
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("low", [-np.inf, -100.0])
def test_a_part_of_nothing_but_the_draft(gpu_lib, rows, vocab, size, cap, low):
    """Without a drafter's logits the fallen draft's part may hold nothing else: masked places, or
    at a temperature of 0.05 ones 2000 below the top."""
    if cap and low > -np.inf:
        low = -20.0  # capped at -17.5, some 900 below the top at a temperature of 0.03
    rng = np.random.default_rng(rows + vocab + 1)
    x = np.round(rng.standard_normal((rows, vocab)) * 8) / 8
    heats = np.full(rows // 2, 0.05 if not cap else 0.03, np.float32)
    for end in ("first", "last"):
        z = x.copy()
        here = slice(0, size) if end == "first" else slice((vocab - 1) // size * size, vocab)
        z[:, here] = low
        z[:, size + 5] = 10.0
        inside = np.arange(vocab)[here]
        tokens = rng.choice(inside, rows).astype(np.int32)
        u = np.zeros((rows, 2), np.float32)
        u[:, 0] = ONE_LESS
        for v in (0.0, 1.0, 0.3):
            u[:, 1] = v
            got, count = check(z, tokens, blocks(rows), u, heats, None, cap)
            assert int(count.sum()) == 0 and bool((got[::2] >= 0).all())
        # the draft has nearly all of the row's weight, and still falls
        z[np.arange(rows - 1), tokens[1:]] = 10.5  # all but 4e-5 or 4e-7 of it
        for v in (0.0, 1.0, 0.3):
            u[:, 1] = v
            got, count = check(z, tokens, blocks(rows), u, heats, None, cap)
            assert int(count.sum()) == 0 and bool((got[::2] >= 0).all())


@pytest.mark.parametrize("rows,vocab,size", SIZES)
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_remainders_of_roundings_alone(gpu_lib, rows, vocab, size, cap):
    """p and q that differ by roundings alone in most parts: whatever u, a token that the target can give."""
    import torch

    from helios_amd import verify_drafts

    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    y = np.roll(x, 1, axis=1)
    y[:, :2 * size] = x[:, :2 * size]
    y[:, 2 * size] = x[:, vocab - 1]  # the same values in another order
    x[:, 7::16] = y[:, 7::16] = -np.inf
    tokens = np.full(rows, 7, np.int32)
    u = np.zeros((rows, 2), np.float32)
    for v in (0.0, 1e-20, 1.0):
        u[:, 1] = v
        got, count = verify_drafts(dev(x), dev(tokens), dev(blocks(rows).astype(np.int32)), dev(u), 0.9, draft_logits=dev(y), softcap=cap, draft_softcap=cap)
        assert int(count.sum()) == 0 and bool((got[::2] >= 0).all())
        assert bool(torch.isfinite(dev(x)[::2].gather(1, got[::2, None].long())).all())


def random_uniforms(rng, n):
    u = rng.random(n).astype(np.float32)
    return np.minimum(u, ONE_LESS)


def draw_all(x, u, heat, cap=0.0, kind=None):
    """The same row for each uniform."""
    from helios_amd import sample

    t = dev(np.broadcast_to(x.astype(np.float32), (len(u), len(x))).copy(), kind)
    return sample(t, dev(u), heat, softcap=cap).tolist()


HEATS = [1e-3, 3e-7, 1e-10, 1e-11, 3e-12, 1e-13, 1e-16, 1e-18, 1e-20, 1e-27, 1e-37, 1e-42]


@pytest.mark.parametrize("heat", HEATS)
@pytest.mark.parametrize("cap", [0.0, 30.0, 5.0])
@pytest.mark.parametrize("vocab", [3000, 40000])
def test_small_temperatures(gpu_lib, heat, cap, vocab):
    """What is equal to the largest logit has its weight; of the smaller ones those have one that a
    temperature of 3e-7 and more leaves within e^-700."""
    rng = np.random.default_rng(int(-np.log10(heat) * 10) + vocab)
    for trial in range(6):
        x = rng.uniform(5.0, 30.0, vocab).astype(np.float32)
        top = np.float32(rng.uniform(30.5, 34.0))
        places = np.sort(rng.choice(vocab, 3, replace=False))
        x[places] = top
        u = random_uniforms(rng, 20)
        u[0] = 0.0
        if heat >= 3e-7:
            p = chances(x.astype(np.float64), np.float32(heat), cap)
            want = [pick(np.where(p >= p.max() * np.exp(-700.0), p, 0.0), v) for v in u]
        else:
            want = [int(places[int(v * 3)]) for v in u.astype(np.float64)]
        assert draw_all(x, u, heat, cap) == want, trial


@pytest.mark.parametrize("step,over", [(1, 0.8), (1, 3.0), (3, 2.0)])
def test_temperatures_of_a_step(gpu_lib, step, over):
    """Logits one or some float32 steps under the top, and a temperature of that size."""
    rng = np.random.default_rng(step)
    for top in (0.7, 19.3, 5e-6, 3e20):
        top = np.float32(top)
        ulp = float(np.spacing(top))
        heat = np.float32(ulp * over)
        x = np.full(4000, 0.0, np.float32) - np.float32(top)
        some = rng.choice(4000, 30, replace=False)
        x[some] = (float(top) - rng.integers(0, 4, 30) * step * ulp).astype(np.float32)
        u = random_uniforms(rng, 40)
        z = (x.astype(np.float64) - float(x.max())) / float(heat)  # exact differences
        e = np.exp(z)
        p = e / e.sum()
        assert draw_all(x, u, float(heat)) == [pick(p, v) for v in u], (top, heat)


@pytest.mark.parametrize("cap,heat", [(30.0, 1e-6), (0.0, 1e-18), (1e12, 1.0), (3.4e38, 0.7), (30.0, 1e-17)])
def test_drafts_at_far_softcaps_and_temperatures(gpu_lib, cap, heat):
    """The check of drafts by the same weights: a large cap is none, a small temperature the first largest."""
    rng = np.random.default_rng(31)
    for rows, vocab, _ in SIZES:
        x = (np.round(rng.standard_normal((rows, vocab)) * 64) / 64).astype(np.float32).astype(np.float64)
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 9.0  # one largest logit
        y = np.roll(x, 3, axis=1)
        y[::4] = x[::4]
        starts, heats = blocks(rows), np.full(rows // 2, heat, np.float32)
        greedy = heat < 1e-3
        _, tokens = drafts(rng, x, [0.0 if greedy else float(h) for h in heats], starts, 0.0)
        from helios_amd import verify_drafts

        u = random_uniforms(rng, 2 * rows).reshape(rows, 2)
        on_gpu = lambda v: dev(v.astype(np.float32))  # noqa: E731
        for drafter in (None, y):
            given = {} if drafter is None else dict(draft_logits=on_gpu(y), draft_softcap=cap)
            got, count = verify_drafts(on_gpu(x), dev(tokens), dev(starts.astype(np.int32)), dev(u), dev(heats), softcap=cap, **given)
            want, accepted = verify(x, tokens, starts, u, heats * 0 if greedy else heats, drafter)
            assert count.tolist() == accepted.tolist() and got.tolist() == want.tolist()


def exact_chances(x, heat, cap):
    """softmax(cap tanh(x / cap) / heat) with 60 digits."""
    with decimal.localcontext() as c:
        c.prec, c.Emin, c.Emax = 60, -10 ** 9, 10 ** 9
        D = decimal.Decimal
        cap, heat = D(float(np.float32(cap))), D(float(np.float32(heat)))
        cache = {}
        for v in set(x.tolist()):
            w = D(v) / cap
            if abs(w) < D("1e-15"):
                t = w - w ** 3 / 3
            else:
                e = (-2 * abs(w)).exp()
                t = ((1 - e) / (1 + e)).copy_sign(w)
            cache[v] = cap * t / heat
        top = max(cache.values())
        e = {v: (z - top).exp() for v, z in cache.items()}
        weights = [e[v] for v in x.tolist()]
        total = sum(weights)
        return [w / total for w in weights]


def exact_pick(p, u):
    with decimal.localcontext() as c:
        c.prec = 60
        goal, at = decimal.Decimal(float(u)) * sum(p), decimal.Decimal(0)
        for i, w in enumerate(p):
            at += w
            if at > goal:
                return i
        return max(i for i, w in enumerate(p) if w > 0)


CAPS = [(1e3, 1.0), (1e6, 1.0), (1e9, 1.0), (1e12, 1.0), (1e15, 1.0), (1e17, 1.0), (1e30, 1.0), (3.4e38, 1.0),
        (1e12, 1e10), (3.4e38, 3e38), (30.0, 0.3), (30.0, 0.03), (30.0, 0.02), (30.0, 1e-3), (30.0, 1e-6), (30.0, 1e-9), (30.0, 1e-13), (30.0, 1e-15),
        (1.0, 1.0), (1e-3, 1e-3), (1e-3, 1e-6), (1e-20, 1e-20), (1e-38, 1e-38), (1e-38, 1.0), (1e-45, 1e-45), (1e-45, 1e-40)]


@pytest.mark.parametrize("cap,heat", CAPS)
def test_softcaps(gpu_lib, cap, heat):
    """Any finite softcap and temperature: the logits lie where cap tanh(x / cap) / T spreads."""
    rng = np.random.default_rng(int(np.log10(cap) * 7 - np.log10(heat) * 3) + 1000)
    vocab = 1500
    for low, high in ((0.0, 1.0), (-2.0, 2.0), (6.0, 8.0)):
        # z over a range of about 12 below some largest logit
        at = rng.uniform(low, high)
        if cap > 1e4:
            at *= heat / cap * 5
        slope = 1 - np.tanh(at) ** 2
        x = cap * at - rng.uniform(0, 12, vocab) * heat / max(slope, 1e-6)
        x = np.clip(x, -3.4e38, 3.4e38).astype(np.float32)
        u = random_uniforms(rng, 24)
        p = exact_chances(x.astype(np.float64), heat, cap)
        got = draw_all(x, u, heat, cap)
        assert got == [exact_pick(p, v) for v in u], (low, high)


@pytest.mark.parametrize("heat", [1e28, 1e30, 1e31, 1e37, 3e38])
def test_large_temperatures(gpu_lib, heat):
    """Logits of float32's largest values over temperatures of that size."""
    rng = np.random.default_rng(int(np.log10(heat)))
    for cap in (0.0, 3e38):
        x = np.clip(rng.uniform(-12, 12, 3000) * heat, -3.4e38, 3.4e38).astype(np.float32)
        u = random_uniforms(rng, 40)
        p = chances(x.astype(np.float64), float(np.float32(heat)), float(np.float32(cap)))
        assert draw_all(x, u, heat, cap) == [pick(p, v) for v in u], cap


def test_an_infinite_temperature_is_uniform(gpu_lib):
    """In the array of temperatures: every place that can be given is as likely as another."""
    from helios_amd import sample

    x = np.linspace(-3e38, 3e38, 3000).astype(np.float32)
    x[::2] = -np.inf
    u = np.array([0.0, 0.25, 0.5, 0.75, ONE_LESS], np.float32)
    got = sample(dev(np.tile(x, (5, 1))), dev(u), dev(np.full(5, np.inf, np.float32))).tolist()
    assert got == [2 * int(float(v) * 1500) + 1 for v in u]
