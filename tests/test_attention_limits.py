"""CPU checks of what the paged-cache calls take and refuse at the edges of their types:
sizes past 32 bits, tensors on several GPUs.  No kernel runs: pointers are checked, never
followed, and the tensors of the Python checks are fake ones (shapes, strides and devices
without memory)."""

import contextlib
import warnings

import pytest
from torch.utils._python_dispatch import TorchDispatchMode

from helios_amd import attention as A
from helios_amd import qmm
from test_attention_abi import BAD, NO, append, attention, batch, lib  # noqa: F401


@pytest.mark.parametrize("stride", [1 << 31, (1 << 32) - 4])
def test_a_table_stride_past_31_bits_is_refused(lib, stride):  # noqa: F811
    """The kernels' stride is an int: read as negative, it would lead before the table."""
    for call in (attention, append):
        assert call(lib, b=batch(table_stride=stride)) == NO
        assert "table_stride" in qmm.last_error()


# ------------------------------------------------------------------ tensors on several GPUs

class Took(Exception):
    """The call went through to the library."""


class NoLibrary:
    def __getattr__(self, name):
        def call(*args):
            raise Took(name)

        return call


@pytest.fixture
def fake(monkeypatch):
    """Fake CUDA tensors on a machine without a GPU; device 0 is current."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(A.qmm, "load_library", NoLibrary)
    monkeypatch.setattr(A.qmm, "_stream_ptr", lambda stream: 0)
    with warnings.catch_warnings(), FakeTensorMode():
        warnings.simplefilter("ignore")  # fake tensors' addresses are 0
        yield lambda *shape, dtype=torch.bfloat16, gpu=0: torch.empty(shape, dtype=dtype, device=f"cuda:{gpu}")


def calls(fake, **gpu):
    """(name, call) of every entry point, with tensor `name` of each on GPU gpu[name]."""
    import torch

    at = lambda name: gpu.get(name, 0)  # noqa: E731
    i32 = lambda name, *shape: fake(*shape, dtype=torch.int32, gpu=at(name))  # noqa: E731
    rope = A.Rope(fake(64, dtype=torch.float32, gpu=at("inv_freq")))
    norms = {f"{w}_norm": A.HeadNorm(fake(128, gpu=at(f"{w}_norm"))) for w in "qkv"}
    q, k, v = (fake(3, n, 128, gpu=at(w)) for n, w in ((4, "q"), (2, "k"), (2, "v")))
    two = norms["q_norm"], norms["k_norm"]
    yield "qk_norm_rope", lambda: A.qk_norm_rope(q, k, i32("positions", 3), rope, *two)
    cache = A.PagedKVCache(*[fake(5, 2, 16, 128, gpu=at("pages")) for _ in "kv"])
    def batch():
        return A.KVBatch(i32("query_starts", 3), i32("kv_lens", 2), i32("block_tables", 2, 4))
    yield "append", lambda: cache.append(k, v, batch(), rope=rope, q=q, **norms)
    yield "attend", lambda: cache.attend(q, batch())


def test_tensors_on_the_current_gpu_are_taken(fake):
    for name, call in calls(fake):
        with pytest.raises(Took):
            call()


@pytest.mark.parametrize("where", ["q", "k", "v", "positions", "inv_freq", "q_norm", "k_norm", "v_norm", "pages", "query_starts",
                                   "kv_lens", "block_tables"])
def test_a_tensor_on_another_gpu_is_refused(fake, where):
    """Whichever it is: its address would be handed to a kernel of the current GPU."""
    used = {"qk_norm_rope": {"q", "k", "positions", "inv_freq", "q_norm", "k_norm"},
            "append": {"q", "k", "v", "inv_freq", "q_norm", "k_norm", "v_norm", "pages", "query_starts", "kv_lens", "block_tables"},
            "attend": {"q", "pages", "query_starts", "kv_lens", "block_tables"}}
    for name, call in calls(fake, **{where: 1}):
        if where in used[name]:
            with pytest.raises(qmm.Gemma4Error) as e:
                call()
            assert e.value.status == BAD, name
        else:
            with pytest.raises(Took):
                call()


# ------------------------------------------------------------------ outputs on a named stream

class Made(TorchDispatchMode):
    """Records, for each tensor operation, the stream that is current."""

    def __init__(self, current):
        super().__init__()
        self.current, self.on = current, []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "aten":
            self.on.append((str(func), self.current[-1]))
        return func(*args, **(kwargs or {}))


@pytest.fixture
def made(fake, monkeypatch):
    """(fake, record(call)): the operations of `call` up to the library's own, with their streams."""
    import torch

    current = ["current"]

    @contextlib.contextmanager
    def stream(s):
        current.append(s)
        yield
        current.pop()

    monkeypatch.setattr(torch.cuda, "stream", stream)

    def record(call):
        with Made(current) as mode, pytest.raises(Took):
            call()
        return mode.on

    return fake, record


def test_outputs_belong_to_the_stream_that_writes_them(made):
    """Memory taken on the current stream may still be in use there when another stream writes it."""
    import torch

    fake, record = made
    i32 = lambda *shape: fake(*shape, dtype=torch.int32)  # noqa: E731
    batch = A.KVBatch(i32(3), i32(2), i32(2, 4))
    cache = A.PagedKVCache(fake(5, 2, 16, 128), fake(5, 2, 16, 128))
    q, k = fake(3, 4, 128), fake(3, 2, 128)
    for call in (lambda s: A.qk_norm_rope(q, k, None, stream=s), lambda s: cache.append(k, k, batch, q=q, stream=s),
                 lambda s: cache.attend(q, batch, return_lse=True, stream=s)):
        for s in (None, "side"):
            on = record(lambda: call(s))
            assert on and all(where == (s or "current") for _, where in on), on


# ------------------------------------------------------------------ numbers past 32 bits in Python

@pytest.mark.parametrize("window", [(1 << 30) + 1, 1 << 32, (1 << 32) + 5, 1 << 70])
def test_a_window_past_the_librarys_limit_is_refused(fake, window):
    """Cut to 32 bits, 2^32 would mean no window and 2^32 + 5 one of 5."""
    import torch

    i32 = lambda *shape: fake(*shape, dtype=torch.int32)  # noqa: E731
    cache = A.PagedKVCache(fake(5, 2, 16, 128), fake(5, 2, 16, 128))
    batch = A.KVBatch(i32(3), i32(2), i32(2, 4))
    with pytest.raises(qmm.Gemma4Error) as e:
        cache.attend(fake(3, 4, 128), batch, window=window)
    assert "window" in str(e.value) and e.value.status == NO
    with pytest.raises(Took):
        cache.attend(fake(3, 4, 128), batch, window=1 << 30)


@pytest.mark.parametrize("distance", [1 << 32, (1 << 32) + 1, (1 << 32) + 64, 1 << 70, -1])
def test_a_distance_past_32_bits_is_refused(fake, distance):
    """Cut to 32 bits, 2^32 + 1 would mean adjacent pairs."""
    import torch

    with pytest.raises(qmm.Gemma4Error) as e:
        A.Rope(fake(64, dtype=torch.float32), distance)
    assert "distance" in str(e.value)
    A.Rope(fake(64, dtype=torch.float32), 256)


# ------------------------------------------------------------------ strides that say nothing

@pytest.mark.parametrize("width", [4 * 128 + 4, 4 * 128 + 1, (1 << 33) + 8])
def test_a_single_rows_stride_says_nothing(fake, width):
    """One token's heads may be cut from a row of any width."""
    one = fake(1, 4, 128).as_strided((1, 4, 128), (width, 128, 1))
    assert A._heads_tensor(one, "q")[1] == 4 * 128
    assert A._heads_tensor(fake(2, 5, 128)[:, :4], "q")[1] == 5 * 128
