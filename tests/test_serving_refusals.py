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


def reader(dtype, heads, kv_heads, dim, batch, prefix, own, page=16, max_q=1):
    c = cache(type=dtype, kv_heads=kv_heads, page_size=page, head_dim=dim)
    return tm.lib().tmac_prefix_attention_engine(ctypes.addressof(c), heads, batch * max_q, batch, max_q, prefix, own)


def test_who_reads_the_prefix():
    """A short prefix is read by each of a few sequences, but once for many whose reading would be most of the work."""
    F32, F16, BF16 = 0, 1, 30
    assert reader(BF16, 14, 2, 64, 2, 96, 17) == 0 and reader(F16, 16, 4, 128, 48, 192, 64) == 0
    assert reader(BF16, 32, 8, 128, 192, 320, 64) >= 1 and reader(F16, 32, 8, 128, 128, 448, 64) >= 1
    assert reader(BF16, 8, 8, 64, 192, 192, 64) >= 1 and reader(F32, 32, 8, 128, 192, 192, 64) == 1
    assert reader(BF16, 14, 2, 64, 384, 192, 64) == 0  # many query rows to a key
    assert reader(F16, 14, 2, 64, 48, 2051, 509) == 1 and reader(BF16, 14, 2, 64, 128, 32768, 1024) == 2
    assert reader(BF16, 14, 2, 64, 128, 32768, 1024, page=4) == 1
    assert reader(BF16, 14, 2, 64, 300, 0, 4000) == 0
    assert reader(BF16, 14, 3, 64, 2, 96, 17) == -3
