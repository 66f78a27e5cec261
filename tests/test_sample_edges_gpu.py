"""sample at the ends of its ranges, against the definition in 64 bits."""
import pytest

import tmac_zynq_fpga_b200 as tm
from test_serving_gpu import BF16, F32, INF, check_sample, random_logits, sample_one

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [359999, 360000, 360001, 500003, 719999, 720000])
@pytest.mark.parametrize("f", [dict(), dict(k=1), dict(k=40), dict(k=900, p=0.9), dict(p=0.7), dict(m=0.05)], ids=str)
def test_large_vocabularies(vocab, f):
    """Rows of 8 and of 16 CTAs, held, and (more rows than the SMs hold) read anew."""
    for dtype, draws in ((F32, 6), (BF16, 3), (F32, 160)):
        check_sample(random_logits(1, vocab, dtype), draws=draws, **f)


def test_the_largest_logit_is_the_last():
    for vocab in (360000, 720000):
        logits = torch.zeros((1, vocab), device="cuda")
        logits[0, -1] = 30.0
        for kw in (dict(temperature=[0.0]), dict(top_k=[3]), dict(top_p=[0.5]), dict(min_p=[0.5])):
            tokens, probs = sample_one(logits, u=[0.5], **kw)
            assert tokens == [vocab - 1]


def test_scaled_logits_past_the_range_of_32_bits():
    """x = logit / temperature counts as infinite past the range: the infinite share the weight, and a row of -inf is empty."""
    logits = torch.tensor([[5.0, 4.0, 1.0, -INF], [-5.0, -4.0, -6.0, -7.0], [5.0, 4.0, 1.0, -INF], [-5.0, -4.0, -6.0, -7.0]], device="cuda")
    tokens, probs = sample_one(logits, u=[0.7] * 4, temperature=[1e-38, 1e-38, 1e-39, 1e-39])
    assert tokens == [1, -1, 0, 1] and probs == [0.5, 0.0, 1.0, 1.0]
