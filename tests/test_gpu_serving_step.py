"""A serving step with drafted tokens, wholly on the GPU: pages for the new tokens, the append
and the attention over a block-scaled cache, logits, which drafts stand, what is kept.  A
captured step replays as the eager one runs, and both do what the steps' definitions say."""

import numpy as np
import pytest

import attention_oracle as O
from pooled_streams import streams  # noqa: F401
from test_gpu_paging import Host
from test_gpu_sampling import verify as verify_host

pytestmark = pytest.mark.gpu

REQUESTS, DRAFTS, PAGE, WIDTH, BLOCK = 5, 3, 32, 12, 16
HQ, HK, D, VOCAB, WINDOW = 8, 2, 128, 6001, 70


class Server:
    """One layer between an embedding and a head, both random; a step's rows are each request's
    last token and its drafts (a request that is full stands still)."""

    def __init__(self, seed):
        import torch

        from helios_amd import HeadNorm, PagedKVCache, PagePool, Rope

        g = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
        self.embed = randn(VOCAB, (HQ + 2 * HK) * D).bfloat16()
        self.head = randn(HQ * D, VOCAB).bfloat16() * 0.02
        self.pool = PagePool.allocate(REQUESTS * WIDTH // 2, PAGE, REQUESTS, WIDTH)
        self.cache = PagedKVCache.allocate(self.pool.num_pages, PAGE, HK, D, torch.float8_e4m3fn, scale_block=BLOCK)
        self.cache.k.view(torch.uint8).fill_(0x7F)  # NaN: what no token is stored to is never read into a result
        self.cache.v.view(torch.uint8).fill_(0x7F)
        for t in (self.cache.k_scale, self.cache.v_scale):
            t.view(torch.uint8).fill_(255)
        self.rope = Rope(1e4 ** (-torch.arange(D // 2, device="cuda") / (D // 2)))
        self.norm = HeadNorm()
        rows = REQUESTS * (1 + DRAFTS)
        self.rows = rows
        self.tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(REQUESTS, dtype=torch.int32, device="cuda")
        self.uniforms = torch.zeros(rows, 2, device="cuda")
        self.draft_logits = torch.zeros(rows, VOCAB, dtype=torch.bfloat16, device="cuda")
        self.heat = torch.tensor([0.0, 0.7, 1.0, 1.3, 0.7], device="cuda")

    def step(self):
        from helios_amd import verify_drafts

        positions, slots = self.pool.reserve(self.new, self.rows)
        x = self.embed[self.tokens.long()]
        q, k, v = (x[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, HQ), (HQ, HQ + HK), (HQ + HK, HQ + 2 * HK)))
        batch = self.pool.batch
        q = self.cache.append(k, v, batch, rope=self.rope, k_norm=self.norm, v_norm=self.norm, q=q, q_norm=self.norm)
        y = self.cache.attend(q, batch, window=WINDOW)
        logits = (y.flatten(1).float() @ self.head.float()).bfloat16()
        out, accepted = verify_drafts(logits, self.tokens, batch.query_starts, self.uniforms, self.heat, draft_logits=self.draft_logits, softcap=30.0)
        kept = self.pool.lens + (accepted + 1) * self.pool.granted * (self.new > 0)
        self.pool.release(kept, window=WINDOW)
        return {"positions": positions, "slots": slots, "q": q, "y": y, "logits": logits, "out": out, "accepted": accepted}

    def inputs(self, rng):
        import torch

        new = rng.integers(0, DRAFTS + 2, REQUESTS)
        self.new.copy_(torch.from_numpy(new).int())
        self.tokens.copy_(torch.from_numpy(rng.integers(0, VOCAB, self.rows)).int())
        self.uniforms.copy_(torch.from_numpy(rng.random((self.rows, 2)) * rng.choice([0.001, 1.0])).float())
        self.draft_logits.copy_(torch.from_numpy(rng.standard_normal((self.rows, VOCAB))))
        return new

    def state(self):
        import torch

        p, c = self.pool, self.cache
        return {"free": p.free_pages, "count": p.free_count, "lens": p.lens, "tables": p.block_tables, "starts": p.batch.query_starts,
                "kv_lens": p.batch.kv_lens, "granted": p.granted, "k": c.k.view(torch.uint8), "v": c.v.view(torch.uint8),
                "k_scale": c.k_scale.view(torch.uint8), "v_scale": c.v_scale.view(torch.uint8)}


def test_captured_steps_replay_as_eager_ones(gpu_lib, streams):
    import torch

    eager, captured = Server(1), Server(1)
    stream = streams()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        captured.step()  # takes the stream's scratch memory before the capture; no tokens are new
    stream.synchronize()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outputs = captured.step()
    rngs = [np.random.default_rng(3) for _ in range(2)]
    for step in range(60):
        new = eager.inputs(rngs[0])
        captured.inputs(rngs[1])
        want = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        live = int(new.sum())
        for name, t in want.items():
            rows = t.shape[0] if name == "accepted" else live
            assert torch.equal(outputs[name][:rows], t[:rows]), (step, name)
        for name, t in eager.state().items():
            assert torch.equal(captured.state()[name], t), (step, name)
        assert bool((outputs["out"][live:] == -1).all()) and bool((outputs["y"][live:] == 0).all())
        torch.rand(100, device="cuda").sum().item()  # work of the program's own between replays


def test_steps_do_what_they_say(gpu_lib):
    """Each step's parts against the host's: the pool's state, the attention over the values that
    the cache then holds, the tokens that follow from the logits."""
    import torch

    server, host = Server(2), Host(REQUESTS * WIDTH // 2, PAGE, REQUESTS, WIDTH)
    host.free = server.pool.free_pages.tolist()
    rng = np.random.default_rng(7)
    for step in range(60):
        new = server.inputs(rng)
        got = server.step()
        live = int(new.sum())
        starts, kv, granted, positions, slots = host.reserve(new, server.rows)
        assert np.array_equal(got["positions"].cpu().numpy(), positions) and np.array_equal(got["slots"].cpu().numpy(), slots)
        assert server.pool.granted.tolist() == granted
        b = {"starts": np.array(starts), "kv_lens": np.array(kv), "tables": host.tables.copy(), "page": PAGE, "num_pages": host.num_pages,
             "rows": server.rows}
        wide = [O.f64(t) * 2.0 ** np.repeat(np.clip(s.view(torch.uint8).cpu().numpy().astype(np.int64) - 127, -100, 80), BLOCK, 2)[..., None]
                for t, s in ((server.cache.k, server.cache.k_scale), (server.cache.v, server.cache.v_scale))]
        want, bound, _, _ = O.attend(O.f64(got["q"]), *wide, b, D ** -0.5, WINDOW)
        O.assert_within(O.f64(got["y"]), want, bound, f"step {step}")
        x, y = (t.float().cpu().numpy().astype(np.float64) for t in (got["logits"], server.draft_logits))
        out, accepted = verify_host(x, server.tokens.cpu().numpy(), starts, server.uniforms.cpu().numpy(), server.heat.cpu().numpy(), y, 30.0)
        assert got["out"][:live].tolist() == out[:live].tolist() and got["accepted"].tolist() == accepted.tolist()
        host.release([int(host.lens[r] + (accepted[r] + 1) * granted[r] * (new[r] > 0)) for r in range(REQUESTS)], WINDOW)
        assert server.pool.lens.tolist() == host.lens.tolist() and server.pool.free_pages[:len(host.free)].tolist() == host.free
        assert np.array_equal(server.pool.block_tables.cpu().numpy(), host.tables)
    assert int(host.lens.max()) > WINDOW  # pages went back behind the window


@pytest.mark.parametrize("args", [["--block", "16"], ["--layer", "full", "--block", "64"]])
def test_the_example_runs_over_block_scales(gpu_lib, args):
    import os
    import subprocess
    import sys

    example = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_attention.py")
    run = subprocess.run([sys.executable, example, "--e4m3", "--requests", "3", "--prompt", "150", "--chunk", "64", "--steps", "5", *args],
                         capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr
    assert "prompts: 300 tokens" in run.stdout and "decoding: 12 tokens" in run.stdout
