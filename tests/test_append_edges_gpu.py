"""rope_append: what must not depend on how its arguments lie."""
import pytest

import tmac_zynq_fpga_b200 as tm
from test_serving_gpu import BF16, F16, F32, append_case, no_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,ctype", [(F32, F32), (BF16, F32), (F32, F16), (F16, F16)])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(14, 2, 64, 64), (16, 4, 128, 96), (6, 2, 64, 0)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_results_do_not_depend_on_strides_and_alignment(dtype, ctype, heads, kv_heads, dim, rot, interleaved):
    results = []
    for shift in (0, 1):  # the second layout takes no 16-byte access
        c = append_case(dtype, ctype, heads, kv_heads, dim, rot, 16, 200, interleaved)
        k, v = (p.clone() for p in c["pools"])
        rows = torch.empty(200 * (heads + 2 * kv_heads) * dim + shift, dtype=dtype, device="cuda")[shift:].view(200, -1)
        q3 = []
        for part, at in zip("qkv", (0, heads * dim, (heads + kv_heads) * dim)):
            there = rows[:, at:at + c[part].shape[1] * dim].unflatten(1, (-1, dim))
            q3.append(there.copy_(c[part]))
        out = tm.rope_append(tm.PagedCache(k, v), *q3, c["pos"], c["tables"], c["cos"], c["sin"], seq=c["seq"], starts=c["starts"],
                             interleaved=interleaved, bias=c["bias"])
        no_error()
        results.append((out, k, v))
    for a, b in zip(*results):
        assert torch.equal(a, b)
