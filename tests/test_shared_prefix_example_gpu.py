"""The batched decode operators run together (examples/shared_prefix_batch.py): greedy
answers of the batch are the decode engine's own tokens, over a prompt computed once."""
import importlib.util
import os

import numpy as np
import pytest

import tmac_zynq_fpga_b200 as tm
from tmac_zynq_fpga_b200 import model

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "shared_prefix_batch.py")
PROMPT, STEPS, ANSWERS = 21, 6, 5


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("shared_prefix_batch", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def want():
    m = tm.Model(model.default_model_path(0), switches=tm.SW_ALL, max_seq=512)
    tokens, hidden = m.generate(model.prompt_tokens(PROMPT, seed=3), STEPS, want_hidden=True)
    m.free()
    return tokens, hidden


@pytest.mark.parametrize("cache", ["float32", "float16", "bfloat16"])
def test_greedy_answers_are_the_decode_engines(example, want, cache):
    tokens, hidden = want
    batch = example.SharedPrefixBatch(model.default_model_path(0), ANSWERS, PROMPT + 3, STEPS, getattr(torch, cache), page=8)
    states = []
    batch._logits = lambda x, f=batch._logits: (states.append(x[-1].cpu().numpy()), f(x))[1]
    got = example.generate(batch, model.prompt_tokens(PROMPT, seed=3), STEPS, temperature=torch.zeros(ANSWERS, device="cuda"))
    assert tm.device_error(0) == 0
    if cache == "float32":
        for i in range(ANSWERS):
            np.testing.assert_array_equal(got[:, i], tokens)
    # the engine's hidden states: 24 layers of int16 activations, whose rounding steps a last bit can move (2^-15 of the
    # largest value each), and of the cache's own rounding
    tol = {"float32": 2e-3, "float16": 5e-3, "bfloat16": 3e-2}[cache]
    for x, h in zip(states, hidden):
        if not np.array_equal(got[:, 0], tokens):
            break  # another token leads elsewhere
        assert np.linalg.norm(x - h) <= tol * np.linalg.norm(h)


def test_drawn_answers_differ_and_repeat(example):
    batch = example.SharedPrefixBatch(model.default_model_path(0), ANSWERS, PROMPT, STEPS)
    top_k = torch.full((ANSWERS,), 1000, dtype=torch.int32, device="cuda")
    prompt = model.prompt_tokens(PROMPT)
    a, b = (example.generate(batch, prompt, STEPS, seed=7, top_k=top_k) for _ in range(2))
    np.testing.assert_array_equal(a, b)
    assert len({tuple(t) for t in a.T}) > 1
