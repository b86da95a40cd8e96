"""The quantized linear calls with ``stream=`` on the GPU: outputs that a call makes belong to
that stream's memory, strided inputs are copied there, and the results are those of the
current stream."""

import pytest

from oracle import affine as A
from test_gpu_attention_edges import stream_of
from test_gpu_parity import dev_triple, dev_x, random_triple

pytestmark = pytest.mark.gpu


def test_outputs_and_copies_on_a_named_stream(gpu_lib):
    import torch

    n, k = 512, 256
    lin = gpu_lib.QuantizedLinear(*dev_triple(*random_triple(n, k, 91)))
    pair = gpu_lib.QuantizedGeGLU(dev_triple(*random_triple(n, k, 92)), dev_triple(*random_triple(n, k, 93)))
    down = gpu_lib.QuantizedLinear(*dev_triple(*random_triple(k, n, 94)))
    x = dev_x(A.make_activations(10, k, seed=95))[::2]  # every other row
    ids = torch.arange(7, device="cuda")

    def run(stream):
        return [lin.forward(x, stream=stream), lin.forward(x, out_dtype=torch.float32, stream=stream), pair.forward(x, stream=stream),
                *pair.forward_mlp(down, x, stream=stream), *lin.forward_greedy(x, return_logits=True, stream=stream),
                lin.embed(ids, stream=stream), lin.dequantize(stream=stream), pair.dequantize(stream=stream)]

    want = run(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = run(side)
    side.synchronize()
    for i, (a, b) in enumerate(zip(got, want)):
        assert stream_of(a) == side.cuda_stream and stream_of(b) != side.cuda_stream, i
        assert torch.equal(a, b), i
    for h in (lin, pair, down):
        h.close()
