"""The batched decode operators without a GPU: the position table against its formula,
and the C entries' refusals, all of which come before any device access."""
import ctypes
import math

import numpy as np
import pytest

import tmac_zynq_fpga_b200 as tm
from tmac_zynq_fpga_b200.serving import PagedCacheStruct

torch = pytest.importorskip("torch")

INVALID, TYPE, SHAPE = -1, -2, -3
A = 0x10000  # stands for an aligned device address that is never read


def cache(k=A, v=A, n_pages=8, type=0, kv_heads=2, page_size=16, head_dim=64, device=0):
    return PagedCacheStruct(k, v, n_pages, type, kv_heads, page_size, head_dim, device)


def append(c=None, **kw):
    d = dict(type=0, q=A, qs=14 * 64, k=A, ks=128, v=A, vs=128, heads=14, tokens=3, bias=None, seq=A, pos=A, starts=None,
             tables=A, n_seq=3, width=4, cos=A, sin=A, max_pos=100, rot=64, inter=1, q_out=A)
    d.update(kw)
    c = c or cache()
    return tm.lib().tmac_rope_append(ctypes.addressof(c), *d.values(), None)


def attend(c=None, **kw):
    d = dict(q=A, qs=14 * 64, heads=14, tokens=3, batch=3, q_start=None, max_q=1, pages=A, prefix=40, prefix_lens=None,
             tables=A, width=4, lens=A, max_own=64, scale=0.125, out=A, os=14 * 64, work=A, work_bytes=1 << 40)
    d.update(kw)
    c = c or cache()
    return tm.lib().tmac_prefix_attention(ctypes.addressof(c), *d.values(), None)


def draw(**kw):
    d = dict(logits=A, type=0, stride=100, batch=2, vocab=100, u=A, t=None, k=None, p=None, m=None, tokens=A, probs=A, device=0)
    d.update(kw)
    return tm.lib().tmac_sample(*d.values(), None)


BAD_CACHES = [(dict(k=0), INVALID), (dict(v=None), INVALID), (dict(type=8), TYPE), (dict(n_pages=0), SHAPE),
              (dict(kv_heads=0), SHAPE), (dict(page_size=0), SHAPE), (dict(page_size=24), SHAPE), (dict(page_size=512), SHAPE),
              (dict(head_dim=63), SHAPE), (dict(head_dim=0), SHAPE), (dict(k=A + 8), INVALID), (dict(v=A + 2), INVALID)]


@pytest.mark.parametrize("what,code", BAD_CACHES)
def test_bad_caches_are_refused(what, code):
    assert append(cache(**what)) == code
    assert attend(cache(**what)) == code
    assert tm.lib().tmac_last_error()


@pytest.mark.parametrize("what,code", [
    (dict(type=8), TYPE), (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(pos=None), INVALID),
    (dict(tables=None), INVALID), (dict(q_out=None), INVALID), (dict(cos=None), INVALID), (dict(sin=None), INVALID),
    (dict(tokens=-1), SHAPE), (dict(heads=0), SHAPE), (dict(n_seq=0), SHAPE), (dict(width=0), SHAPE), (dict(rot=63), SHAPE),
    (dict(rot=66), SHAPE), (dict(rot=-2), SHAPE), (dict(max_pos=0), SHAPE), (dict(qs=14 * 64 - 1), SHAPE), (dict(ks=127), SHAPE),
    (dict(vs=0), SHAPE), (dict(seq=None, n_seq=2), SHAPE), (dict(q=A + 2), INVALID), (dict(q_out=A + 2), INVALID)])
def test_append_refusals(what, code):
    assert append(**what) == code


def test_append_of_no_token_is_ok():
    assert append(tokens=0, q=None, q_out=None) == 0


@pytest.mark.parametrize("what,code", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(pages=None), INVALID), (dict(tables=None), INVALID),
    (dict(lens=None), INVALID), (dict(prefix=40000, work=None), INVALID), (dict(prefix=40000, work_bytes=8), INVALID),
    (dict(prefix=40000, work=A + 8), INVALID),
    (dict(heads=13), SHAPE), (dict(heads=0), SHAPE), (dict(tokens=-1), SHAPE), (dict(batch=2), SHAPE), (dict(max_q=0), SHAPE),
    (dict(max_q=2), SHAPE), (dict(prefix=-1), SHAPE), (dict(max_own=-1), SHAPE), (dict(max_own=65), SHAPE), (dict(qs=64), SHAPE),
    (dict(os=64), SHAPE), (dict(batch=0, q_start=A), SHAPE), (dict(q=A + 2), INVALID)])
def test_attention_refusals(what, code):
    assert attend(**what) == code


def test_attention_refuses_other_head_dims():
    assert attend(cache(head_dim=96), qs=14 * 96, os=14 * 96) == SHAPE


def test_attention_of_no_token_is_ok():
    assert attend(tokens=0, batch=0, q=None, out=None) == 0
    n = ctypes.c_size_t(7)
    assert tm.lib().tmac_prefix_attention_workspace(ctypes.addressof(cache()), 14, 0, 0, 1, 40, 64, ctypes.addressof(n)) == 0
    assert n.value == 0
    assert tm.lib().tmac_prefix_attention_workspace(ctypes.addressof(cache()), 14, 3, 3, 1, 40, 64, None) == INVALID


@pytest.mark.parametrize("what,code", [
    (dict(type=12), TYPE), (dict(logits=None), INVALID), (dict(u=None), INVALID), (dict(tokens=None), INVALID),
    (dict(probs=None), INVALID), (dict(batch=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(vocab=720001, stride=720001), SHAPE),
    (dict(stride=99), SHAPE), (dict(logits=A + 2), INVALID)])
def test_sample_refusals(what, code):
    assert draw(**what) == code


def test_sample_of_no_row_is_ok():
    assert draw(batch=0, logits=None) == 0


def test_python_refusals_without_a_gpu():
    k = torch.zeros(4, 2, 16, 64)
    for bad in ((k, k), (k[0], k[0]), (k, k[:2]), (k.int(), k.int()), (k, k.half())):
        with pytest.raises(tm.TmacError):
            tm.PagedCache(*bad)
    with pytest.raises(tm.TmacError):
        tm.sample(torch.zeros(2, 10), torch.zeros(2))
    with pytest.raises(tm.TmacError):
        tm.sample(torch.zeros(2, 10, dtype=torch.int32), torch.zeros(2))
    for bad in (dict(max_pos=0), dict(rot_dim=63), dict(rot_dim=0), dict(factor=0.0), dict(theta=-1.0), dict(original=4, low=3.0, high=3.0)):
        with pytest.raises(tm.TmacError):
            tm.rope_table(**{"max_pos": 8, "rot_dim": 64, **bad}, device="cpu")


def test_rope_table_is_the_rounded_formula():
    # both sides form cos and sin in 64 bits: at most one unit of the 32-bit rounding apart (1/2 each), at |value| <= 1.5
    cos, sin = tm.rope_table(5000, 64, device="cpu")
    for pos in (0, 1, 77, 4999):
        for i in (0, 1, 13, 31):
            angle = pos * 1e6 ** (-2 * i / 64)
            assert abs(cos[pos, i].item() - math.cos(angle)) <= 2 ** -23 and abs(sin[pos, i].item() - math.sin(angle)) <= 2 ** -23


def test_rope_table_scaled_for_long_contexts():
    f = 1e4 ** (-np.arange(0, 32, 2) / 32)
    cos, _ = tm.rope_table(100, 32, theta=1e4, factor=4.0, device="cpu")
    np.testing.assert_allclose(cos[80].numpy(), np.cos(20 * f), atol=2 ** -22)  # a quarter of the position
    cos, sin = tm.rope_table(100, 32, theta=1e4, factor=4.0, original=256, low=1.0, high=8.0, scale=1.5, device="cpu")
    turns = 256 * f / (2 * math.pi)
    for i, n in enumerate(turns):
        g = f[i] if n >= 8 else f[i] / 4 if n <= 1 else f[i] * ((n - 1) / 7) + f[i] / 4 * (1 - (n - 1) / 7)
        assert abs(cos[99, i].item() - 1.5 * math.cos(99 * g)) <= 2 ** -22 and abs(sin[99, i].item() - 1.5 * math.sin(99 * g)) <= 2 ** -22
    assert (turns >= 8).any() and (turns <= 1).any() and ((turns > 1) & (turns < 8)).any()
