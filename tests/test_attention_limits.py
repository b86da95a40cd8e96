"""CPU checks of what the paged-cache calls take and refuse at the edges of their types:
sizes past 32 bits, tensors on several GPUs.  No kernel runs: pointers are checked, never
followed, and the tensors of the Python checks are fake ones (shapes, strides and devices
without memory)."""

import pytest

from helios_amd import qmm
from test_attention_abi import NO, append, attention, batch, lib  # noqa: F401


@pytest.mark.parametrize("stride", [1 << 31, (1 << 32) - 4])
def test_a_table_stride_past_31_bits_is_refused(lib, stride):  # noqa: F811
    """The kernels' stride is an int: read as negative, it would lead before the table."""
    for call in (attention, append):
        assert call(lib, b=batch(table_stride=stride)) == NO
        assert "table_stride" in qmm.last_error()
