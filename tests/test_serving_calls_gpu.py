"""How the operators of the batched decode step are called: devices, streams, gradients."""
import pytest

import tmac_zynq_fpga_b200 as tm
from test_serving import append, cache, draw
from test_serving_gpu import BF16, append_case, check_append

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_a_refused_device_leaves_nothing_behind():
    """The refusal is the call's alone: the next launch does not report it."""
    for device in (99, -1):
        assert draw(device=device) == -9 and append(cache(device=device)) == -9
        check_append(append_case(BF16, BF16, 14, 2, 64, 64, 16, 5))
        torch.zeros(3, device="cuda").add_(1)
