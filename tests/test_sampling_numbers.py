"""CPU checks of the numbers that the sampling calls take from Python's 64 bits to the library's 32."""

import numpy as np
import pytest

from helios_amd import sampling
from helios_amd.qmm import Gemma4Error

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("v", [0.0, 0, 1, 0.7, 30.0, 1e30, 3.4e38, 1e-38, 1e-45, 2.0 ** -149, float(np.nextafter(2.0 ** -150, 1.0))])
def test_numbers_that_stay_what_they_are(v):
    assert sampling._number(v, "temperature", "greedy") == v
    assert (np.float32(v) == 0) == (v == 0)
    assert sampling._temperature(v, 3) == (v, None)


@pytest.mark.parametrize("v", [-1.0, -1e-300, INF, -INF, NAN])
def test_numbers_that_are_none(v):
    with pytest.raises(Gemma4Error, match="finite and >= 0"):
        sampling._temperature(v, 3)


@pytest.mark.parametrize("v", [1e-46, 5e-324, 1e-300, 2.0 ** -150])
def test_numbers_that_would_become_zero(v):
    """0 is another call: greedy, or uncapped."""
    assert np.float32(v) == 0
    with pytest.raises(Gemma4Error, match="2\\^-150"):
        sampling._temperature(v, 3)
    with pytest.raises(Gemma4Error, match="softcap must be 0"):
        sampling._number(v, "logits' softcap", "none")
