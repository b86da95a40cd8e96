"""Sampling and verification at the ends of what they take, on the GPU against the definitions in
float64 on the host: uniforms of 0 and from 1 on beside places without weight.  Tokens have to be equal."""

import numpy as np
import pytest

from test_gpu_sampling import dev

pytestmark = pytest.mark.gpu


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
