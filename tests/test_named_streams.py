"""CPU check of the quantized linear calls with ``stream=``: what they make (outputs, contiguous
copies of strided inputs) is made on that stream, not on torch's current one.  No kernel runs:
the tensors are fake and the library only says that it was reached."""

import contextlib
import ctypes

import pytest

from helios_amd import qmm
from test_attention_limits import NoLibrary, fake, made  # noqa: F401


def handle(cls):
    h = object.__new__(cls)
    h._lib, h._handle, h.in_features, h.out_features = NoLibrary(), ctypes.c_void_p(), 128, 64
    h.info = lambda: {"device": 0}
    return h


@pytest.mark.parametrize("stream", [None, "side"])
def test_what_a_call_makes_is_made_on_its_stream(made, stream, monkeypatch):  # noqa: F811
    import torch

    fake, record = made  # noqa: F811
    lin, pair = handle(qmm.QuantizedLinear), handle(qmm.QuantizedGeGLU)
    x = fake(3, 256)[:, ::2]  # strided: the calls copy it
    triple = fake(64, 32, dtype=torch.int32)[:, ::2], fake(64, 4)[:, ::2], fake(64, 4)[:, ::2]
    ids = fake(5, dtype=torch.int64)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    calls = {
        "forward": lambda: lin.forward(x, stream=stream),
        "fp32": lambda: lin.forward(x, out_dtype=torch.float32, stream=stream),
        "lora": lambda: lin.forward_lora(x, None, stream=stream),
        "greedy": lambda: lin.forward_greedy(x, return_logits=True, stream=stream),
        "embed": lambda: lin.embed(ids, stream=stream),
        "dequantize": lambda: lin.dequantize(stream=stream),
        "geglu": lambda: pair.forward(x, stream=stream),
        "mlp": lambda: pair.forward_mlp(lin, x, stream=stream),
        "geglu dequantize": lambda: pair.dequantize(stream=stream),
        "create": lambda: qmm.QuantizedLinear(*triple, stream=stream),
        "create pair": lambda: qmm.QuantizedGeGLU(triple, triple, stream=stream),
    }
    for name, call in calls.items():
        on = record(call)
        assert on and all(where == (stream or "current") for _, where in on), (name, on)
