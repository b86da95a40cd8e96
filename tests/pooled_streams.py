"""Streams for a test that leave torch's pool as it was.

``torch.cuda.Stream()`` hands out 32 streams in turn, and scratch memory is kept per stream: a
test that expects a stream without any would meet one that another test has used, depending on
how many were taken between the two.  The ``streams`` fixture gives back its streams' scratch
memory and takes the turn on to where it was."""

import pytest

POOL = 32


@pytest.fixture
def streams(gpu_lib):
    import torch

    made = []

    def make():
        made.append(torch.cuda.Stream())
        return made[-1]

    yield make
    torch.cuda.synchronize()
    for s in made:
        gpu_lib.release_scratch(s)
    for _ in range(-len(made) % POOL):
        torch.cuda.Stream()
