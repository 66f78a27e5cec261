"""prefix_attention where numbers, lengths or layouts are out of the ordinary, against 64 bits.
Tolerances as derived in test_serving_gpu.py; every sequence here sees one list of keys."""
import math

import pytest

import tmac_zynq_fpga_b200 as tm
from test_serving_gpu import BF16, F16, F32, INF, NAN, TINY, U, attention_case, bounds_error, ints, no_error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# (sequences, keys): each sequence reads the prefix itself; shared and joined; on tcgen05 (16 bits)
LAYOUTS = [(2, 200), (9, 1100), (40, 1100), (100, 6000)]
HEADS = {64: (14, 2), 128: (8, 2)}


def random_rows(dim, batch, n, dtype, seed=0):
    """q [batch, heads, dim], k and v [n, kv_heads, dim]"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, hk = HEADS[dim]
    return [(torch.randn(s, generator=g, device="cuda") * f).to(dtype) for s, f in (((batch, h, dim), 2.0), ((n, hk, dim), 1.0), ((n, hk, dim), 1.0))]


def paged(rows, page, seed=1):
    """Pools that hold rows [n, kv_heads, dim] in pages at random places, and the pages' numbers."""
    n, hk, dim = rows[0].shape
    count = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = torch.randperm(count + 2, generator=g, device="cuda")[:count].int()
    at = torch.arange(n, device="cuda")
    pools = []
    for r in rows:
        pool = torch.full((count + 2, hk, page, dim), NAN, device="cuda", dtype=r.dtype)
        pool[pages.long()[at // page], :, at % page] = r
        pools.append(pool)
    return pools, pages


def attend(q, k, v, page=16, **kw):
    """Every row over all keys."""
    (kp, vp), pages = paged([k, v], page)
    none = torch.zeros((len(q), 1), dtype=torch.int32, device="cuda")
    out = tm.prefix_attention(q, tm.PagedCache(kp, vp), none, none[:, 0].contiguous(), prefix_pages=pages, prefix_len=len(k), max_own=0, **kw)
    no_error()
    return out


def formula(q, k, v, scale=None):
    """The result in 64 bits and its tolerance; a key whose score is -inf weighs nothing."""
    h, dim = q.shape[1:]
    scale = dim ** -0.5 if scale is None else scale
    kd, vd = (x.double().repeat_interleave(h // k.shape[1], 1) for x in (k, v))
    want, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for t in range(len(q)):
        terms = q[t].double() * kd * scale
        score = terms.sum(2)
        p = torch.softmax(score, 0)
        want[t] = torch.einsum("kh,khd->hd", p, vd)
        size = torch.einsum("kh,khd->hd", p, vd.abs())
        most = torch.where(score == -INF, 0.0, terms.abs().sum(2)).amax(0)[:, None]
        off = 2 * (dim + 4) * 2.0 ** -24 * most + (len(k) + 16) * 2.0 ** -24
        tol[t] = U[q.dtype] * want[t].abs() + (off + (U[q.dtype] if q.dtype != F32 else 0)) * size + TINY[q.dtype]
    return want, tol


def check(out, want, tol):
    off = (out.double() - want).abs() - tol
    assert torch.isfinite(want).all() and (off <= 0).all(), f"worst {off.max().item():.3g} past the tolerance"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,n", LAYOUTS)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_of_minus_infinity_weighs_nothing(dtype, batch, n, dim):
    q, k, v = random_rows(dim, batch, n, dtype)
    q[..., 3] = q[..., 3].abs() + 0.5
    k[5::7, :, 3] = -INF
    check(attend(q, k, v), *formula(q, k, v))


@pytest.mark.parametrize("batch,n", LAYOUTS)
def test_keys_as_large_as_the_type_allows(batch, n):
    q, k, v = random_rows(64, batch, n, F32)
    q[..., 9] = 2.0 ** -126
    k[::3, :, 9] = torch.finfo(F32).max
    k[1::3, :, 9] = -torch.finfo(F32).max
    check(attend(q, k, v), *formula(q, k, v))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch,n", LAYOUTS)
def test_large_values_whose_weights_grow_along_the_keys(dtype, batch, n):
    """The first 64 keys weigh 2^-24 of the others each; sums of weight times value pass 32 bits' range
    unless weights stay near 1."""
    q, k, v = random_rows(64, batch, n, dtype)
    q[:], k[:] = 0, 0
    q[..., 0] = 8.0
    k[64:, :, 0] = 24 * math.log(2)  # times 8 / sqrt(64)
    v = (v.float() * 2.0 ** 110).to(dtype)
    check(attend(q, k, v), *formula(q, k, v))


# float32 NaNs as Python writes them, as the GPU's arithmetic gives them, and their negatives
NANS = {F32: [0x7FC00000, 0x7FFFFFFF, -1, -0x400000, 0x7F800001, 0x7FFFF000], F16: [0x7E00, 0x7FFF, -1, 0x7C01], BF16: [0x7FC0, 0x7FFF, -1, 0x7F81]}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,n", LAYOUTS)
@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_every_nan_reaches_the_rows_that_see_it(dtype, batch, n, where):
    whole = torch.int32 if dtype == F32 else torch.int16
    for bits in NANS[dtype]:
        rows = dict(zip("qkv", random_rows(64, batch, n, dtype)))
        at = 1 if where == "q" else n - 20
        rows[where].view(whole)[at, :, 6] = bits
        out = attend(**rows)
        if where == "q":
            assert torch.isnan(out[at]).all()
            others = torch.arange(batch, device="cuda") != at
            want, tol = formula(rows["q"][others], rows["k"], rows["v"])
            check(out[others], want, tol)
        elif where == "k":
            assert torch.isnan(out).all()
        else:
            assert torch.isnan(out[..., 6]).all() and torch.isfinite(out[..., 7]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_nan_far_below_the_largest_score_is_not_lost_in_the_join(dtype):
    """The NaN's neighbours in its range of keys weigh nothing against a key of another range."""
    q, k, v = random_rows(64, 9, 3000, dtype)
    q[..., 0], k[:, :, 0] = 16.0, -60.0
    k[0, :, 0] = 60.0
    k[2500, :, 5] = NAN
    assert torch.isnan(attend(q, k, v)).all()


@pytest.mark.parametrize("batch,n", LAYOUTS)
def test_nans_of_the_gpu_do_not_reach_rows_that_see_less(batch, n):
    q, k, v = random_rows(64, batch, n, F32)
    seen = n - 30
    for x in (k, v):
        x.view(torch.int32)[seen:, :, 6] = 0x7FFFFFFF
    out = attend(q, k, v, prefix_lens=ints([seen] * batch))
    check(out, *formula(q, k[:seen], v[:seen]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,n", LAYOUTS)
@pytest.mark.parametrize("gap", [12.0, 15.0, 17.5])
@pytest.mark.parametrize("at", ["first", "last"])
def test_many_small_weights_beside_a_key_without_value(dtype, batch, n, gap, at):
    """One key takes nearly all of the weight and its value is 0: the result is the small weights' alone."""
    q, k, v = random_rows(64, batch, n, dtype)
    q[:], k[:] = 0, 0
    q[..., 0] = 8.0  # times k / sqrt(64)
    one = 0 if at == "first" else n - 1
    k[one, :, 0], v[one] = gap, 0
    v = v.abs()
    check(attend(q, k, v), *formula(q, k, v))


# (prefix, own keys): every sequence reads the prefix itself; own keys alone, in one job and in several; joined;
# one job over the prefix alone; on tcgen05 (16 bits), joined and in one job
def rows_of_no_sequence_cases():
    few, many = [2, 3, 0, 1], [2, 3, 0, 1] * 80
    return [(75, [5, 40, 0, 17], few), (0, [5, 40, 0, 17], few), (0, [600] * 320, many), (0, [900, 700, 0, 1000], few), (1000, [5, 40, 0, 17], few),
            (600, [0] * 320, many), (600, [0] * 2400, many[:240] * 10), (3500, [3, 9, 0, 2] * 30, many[:120])]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(8))
def test_rows_of_no_sequence_are_zeros(dtype, case):
    prefix, own, queries = rows_of_no_sequence_cases()[case]
    c = attention_case(dtype, 14, 2, 64, 16, prefix, own, queries)
    before, after = 3, 70
    q = torch.cat([c["q"][:1].expand(before, -1, -1), c["q"], c["q"][:1].expand(after, -1, -1)])
    out = torch.full_like(q, NAN)
    kw = {**c["kw"], "q_start": c["kw"]["q_start"] + before, "max_own": max(own)}
    tm.prefix_attention(q, tm.PagedCache(c["k"], c["v"]), c["tables"], c["lens"], out=out, **kw)
    no_error()  # padding is no error
    assert not out[:before].any() and not out[-after:].any()
    check(out[before:-after], c["want"], c["tol"])
    # tokens past max_q
    out.fill_(NAN)
    tm.prefix_attention(q, tm.PagedCache(c["k"], c["v"]), c["tables"], c["lens"], out=out, **{**kw, "max_q": 2})
    bounds_error()
    third = torch.tensor([sum(queries[:b]) + before + 2 for b, n in enumerate(queries) if n == 3], device="cuda")
    assert torch.isfinite(out).all() and not out[third].any() and out[third - 1].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("prefix,own", [(75, 9), (1000, 9)])
@pytest.mark.parametrize("starts", [[0, 2, 7], [0, 3, 2], [-1, 2, 3], [5, 5, 5]])
def test_bad_starts_are_errors(dtype, prefix, own, starts):
    c = attention_case(dtype, 14, 2, 64, 16, prefix, [own] * 2, [2, 1])
    out = torch.full_like(c["q"], NAN)
    tm.prefix_attention(c["q"], tm.PagedCache(c["k"], c["v"]), c["tables"], c["lens"], out=out, **{**c["kw"], "q_start": ints(starts), "max_q": 3})
    bounds_error()
    assert torch.isfinite(out).all()
