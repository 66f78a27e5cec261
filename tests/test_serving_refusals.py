"""What the entries of the batched decode step refuse before any device access."""
import ctypes

import pytest

import tmac_zynq_fpga_b200 as tm
from test_serving import append, attend, cache, draw

NODEV = -9


@pytest.mark.parametrize("device", [-1, -(1 << 31), 1 << 30, (1 << 31) - 1])
def test_no_such_device(device):
    c = cache(device=device)
    assert append(c) == NODEV
    assert attend(c, prefix=40000) == NODEV
    assert draw(device=device) == NODEV
    n = ctypes.c_size_t(0)
    rc = tm.lib().tmac_prefix_attention_workspace(ctypes.addressof(c), 14, 3, 3, 1, 40000, 64, ctypes.addressof(n))
    assert rc == (NODEV if device < 0 else 0)  # a size needs no device


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_attention_refuses_a_scale_that_is_not_finite(scale):
    assert attend(scale=scale) == -1
    assert attend(scale=scale, prefix=40000) == -1
