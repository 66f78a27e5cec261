"""prefix_attention where the prefix's jobs run on the tcgen05 kernel, beside the own keys' kernel and
before the join.  Every case asserts that this kernel is the one that is chosen; results against 64
bits, tolerances as derived in test_serving_gpu.py."""
import ctypes

import pytest

import tmac_zynq_fpga_b200 as tm
from test_attention_edges_gpu import check, formula, paged, random_rows
from test_serving_gpu import BF16, F16, INF, NAN, attend, attention_case, bounds_error, check_attention, ints, no_error
from tmac_zynq_fpga_b200.serving import PagedCacheStruct

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [F16, BF16])
HEADS = pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (16, 4, 128)])


def engine(q, k, batch, prefix, max_own, max_q=1):
    n, hk, page, dim = k.shape
    c = PagedCacheStruct(k.data_ptr(), k.data_ptr(), n, {torch.float32: 0, F16: 1, BF16: 30}[k.dtype], hk, page, dim, 0)
    return tm.lib().tmac_prefix_attention_engine(ctypes.addressof(c), q.shape[1], q.shape[0], batch, max_q, prefix, max_own)


def on_tc(c):
    batch, width = c["tables"].shape
    assert engine(c["q"], c["k"], batch, c["kw"]["prefix_len"], width * c["k"].shape[2], c["kw"].get("max_q", 1)) == 2
    return c


def shared(q, k, v, page=16, lens=None, **kw):
    """All rows over the first lens[b] of all keys, no own ones."""
    (kp, vp), pages = paged([k, v], page)
    assert engine(q, kp, len(q), len(k), 0) == 2
    none = torch.zeros((len(q), 1), dtype=torch.int32, device="cuda")
    out = tm.prefix_attention(q, tm.PagedCache(kp, vp), none, none[:, 0].contiguous(), prefix_pages=pages, prefix_len=len(k), max_own=0,
                              prefix_lens=None if lens is None else ints(lens), **kw)
    no_error()
    return out


@TYPES
@HEADS
@pytest.mark.parametrize("batch", [67, 100, 128])
def test_rows_and_own_keys(dtype, heads, kv_heads, dim, batch):
    check_attention(on_tc(attention_case(dtype, heads, kv_heads, dim, 16, 9001, [b * 13 % 70 for b in range(batch)])))


@TYPES
@HEADS
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_pages(dtype, heads, kv_heads, dim, page):
    check_attention(on_tc(attention_case(dtype, heads, kv_heads, dim, page, 6007, [b % 9 for b in range(100)])))


def test_small_pages_stay_with_the_other_kernel():
    for page in (1, 2, 4):
        c = attention_case(BF16, 14, 2, 64, page, 6007, [3] * 100)
        assert engine(c["q"], c["k"], 100, 6007, page * c["tables"].shape[1]) == 1
        check_attention(c)


# ends inside a tile, at its end, at and before a key range's, and none
LENS = [6000, 0, 1, 63, 64, 65, 128, 255, 256, 257, 320, 1000, 1024, 2500, 2560, 3333, 4096, 5999, 5952, 5934]


@TYPES
@HEADS
@pytest.mark.parametrize("queries", [False, True])
def test_sequences_that_leave_the_prefix(dtype, heads, kv_heads, dim, queries):
    n_q = [1, 5, 0, 3, 7, 2, 1] * 14 if queries else None
    c = attention_case(dtype, heads, kv_heads, dim, 16, 6000, [b % 11 for b in range(98)], n_q, prefix_lens=[LENS[b * 7 % 20] for b in range(98)])
    check_attention(on_tc(c))


@TYPES
@HEADS
def test_several_query_tokens(dtype, heads, kv_heads, dim):
    check_attention(on_tc(attention_case(dtype, heads, kv_heads, dim, 32, 3500, [9 + b % 50 for b in range(60)], [1, 5, 0, 9, 2, 3] * 10)))
    check_attention(on_tc(attention_case(dtype, heads, kv_heads, dim, 32, 3500, [b % 3 for b in range(60)], [1, 5, 0, 9, 2, 3] * 10)))


@TYPES
@HEADS
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_unseen_values_do_not_reach_a_row(dtype, heads, kv_heads, dim, bad):
    """Sequences see the prefix up to 2000, 5950 or 6000; what lies behind does not reach them."""
    lens = [(2000, 5950, 6000)[b % 3] for b in range(99)]
    for tail in ((5950, 6000), (2000, 2001), (2000, 6000)):
        c = on_tc(attention_case(dtype, heads, kv_heads, dim, 16, 6000, [b % 4 for b in range(99)], prefix_lens=lens))
        p = c["kw"]["prefix_pages"].long()
        at = torch.arange(*tail, device="cuda")
        for pool in (c["k"], c["v"]):
            pool[p[at // 16], :, at % 16] = bad
        out = attend(c)
        no_error()
        blind = torch.tensor([n <= tail[0] for n in lens], device="cuda")
        assert ((out.double() - c["want"]).abs() <= c["tol"])[blind].all()
        assert not torch.isfinite(out[~blind]).any() or bad == -INF


@TYPES
@pytest.mark.parametrize("spread", [0.0, 8.0, 30.0])
def test_flat_and_peaked_scores(dtype, spread):
    check_attention(on_tc(attention_case(dtype, 14, 2, 64, 16, 7301, [b % 20 for b in range(80)], spread=spread)))
    check_attention(on_tc(attention_case(dtype, 16, 4, 128, 16, 3000, [b % 20 for b in range(80)], spread=spread)))


@TYPES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("every,step", [(130, 25.0), (64, 4.0), (200, 12.0), (1000, 60.0)])
def test_scores_that_rise_along_the_keys(dtype, dim, every, step):
    """Later tiles pass the limit on weights: a new maximum, and the sums so far scaled down, in some rows of a warp."""
    q, k, v = random_rows(dim, 100, 6000, dtype)
    sign = torch.tensor([(-1.0, 1.0, 0.0)[b % 3] for b in range(100)], device="cuda")
    q[..., 0] = (sign * dim ** 0.5)[:, None].to(dtype)
    k[:, :, 0] = ((torch.arange(6000, device="cuda") // every) * step)[:, None].to(dtype)
    check(shared(q, k, v), *formula(q, k, v))
    lens = [LENS[b * 7 % 20] or 6000 for b in range(100)]
    out = shared(q, k, v, lens=lens)
    for b in (0, 1, 2, 7, 12, 19, 55, 98):
        want, tol = formula(q[b:b + 1], k[:lens[b]], v[:lens[b]])
        check(out[b:b + 1], want, tol)


@TYPES
@pytest.mark.parametrize("scale", [-0.125, -1.0, 0.0, 0.3])
def test_other_scales(dtype, scale):
    q, k, v = random_rows(64, 100, 6000, dtype)
    check(shared(q, k, v, scale=scale), *formula(q, k, v, scale))


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("batch,n", [(2, 200), (9, 1100)])
@pytest.mark.parametrize("scale", [-0.125, 0.0])
def test_other_scales_on_the_other_kernel(dtype, batch, n, scale):
    q, k, v = random_rows(64, batch, n, dtype)
    (kp, vp), pages = paged([k, v], 16)
    none = torch.zeros((batch, 1), dtype=torch.int32, device="cuda")
    assert engine(q, kp, batch, n, 0) < 2
    out = tm.prefix_attention(q, tm.PagedCache(kp, vp), none, none[:, 0].contiguous(), prefix_pages=pages, prefix_len=n, max_own=0, scale=scale)
    no_error()
    check(out, *formula(q, k, v, scale))


@TYPES
@HEADS
@pytest.mark.parametrize("pad", [8, 4, 3, 1])
def test_strided_rows(dtype, heads, kv_heads, dim, pad):
    c = on_tc(attention_case(dtype, heads, kv_heads, dim, 16, 8300, [b % 5 for b in range(70)], pad=pad))
    plain = check_attention(c)
    wide = torch.zeros((70, heads * dim + pad), dtype=dtype, device="cuda")
    out = wide[:, pad:].unflatten(1, (heads, dim))
    assert attend(c, out=out) is out
    no_error()
    assert torch.equal(out, plain) and not wide[:, :pad].any()


@TYPES
@pytest.mark.parametrize("batch,prefix", [(100, 6000), (2400, 600)])
def test_the_prefix_alone(dtype, batch, prefix):
    """Joined, and (many rows) one job a row that writes the result."""
    q, k, v = random_rows(64, batch, prefix, dtype)
    for pad in (0, 1):
        wide = torch.zeros((batch, 14 * 64 + pad), dtype=dtype, device="cuda")
        out = wide[:, pad:].unflatten(1, (14, 64))
        shared(q, k, v, out=out)
        few = torch.arange(0, batch, 1 + batch // 100, device="cuda")
        check(out[few], *formula(q[few], k, v))
        assert not wide[:, :pad].any()


@TYPES
def test_pages_outside_the_pool_count_as_zeros(dtype):
    c = on_tc(attention_case(dtype, 14, 2, 64, 16, 8300, [b % 5 for b in range(70)]))
    pages = c["kw"]["prefix_pages"].clone()
    for at, bad in ((1, 10 ** 6), (100, -1), (312, 2 ** 31 - 1)):
        c["k"][pages[at].long()], c["v"][pages[at].long()] = 0, 0
        want = attend(c)
        no_error()
        broken = pages.clone()
        broken[at] = bad
        out = attend(c, prefix_pages=broken)
        bounds_error()
        assert torch.equal(out, want)
    out = attend(c, prefix_lens=ints([10 ** 6] * 70))
    bounds_error()
    assert torch.equal(out, attend(c))
    no_error()


def test_past_32_bit_offsets():
    # 2^31 elements lie before the prefix's pages of these pools (4.3 GB each)
    page, hk, dim = 64, 2, 64
    q, rows_k, rows_v = random_rows(dim, 100, 6000, BF16)
    count = -(-6000 // page)
    n = 2 ** 31 // (page * hk * dim) + count
    k, v = (torch.zeros((n, hk, page, dim), dtype=BF16, device="cuda") for _ in range(2))
    at = torch.arange(6000, device="cuda")
    pages = torch.arange(n - count, n, device="cuda")
    for pool, rows in ((k, rows_k), (v, rows_v)):
        pool[pages[at // page], :, at % page] = rows
    none = torch.zeros((100, 1), dtype=torch.int32, device="cuda")
    assert engine(q, k, 100, 6000, 0) == 2
    out = tm.prefix_attention(q, tm.PagedCache(k, v), none, none[:, 0].contiguous(), prefix_pages=pages.int(), prefix_len=6000, max_own=0)
    no_error()
    check(out, *formula(q, rows_k, rows_v))


@TYPES
def test_the_same_every_time(dtype):
    c = on_tc(attention_case(dtype, 14, 2, 64, 16, 8300, [b * 37 % 300 for b in range(70)], prefix_lens=[LENS[b % 20] for b in range(70)]))
    a = attend(c)
    assert all(torch.equal(a, attend(c)) for _ in range(10))


@TYPES
def test_on_another_stream(dtype):
    """The three kernels in order on a stream that is not torch's current one, between others that write their inputs."""
    c = on_tc(attention_case(dtype, 14, 2, 64, 16, 6500, [b % 30 for b in range(90)]))
    want = attend(c)
    q, k = c["q"].clone(), c["k"].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            q.fill_(NAN), k.fill_(NAN)
            q.copy_(c["q"]), k.copy_(c["k"])
        out = attend({**c, "q": q, "k": k}, stream=stream)
        with torch.cuda.stream(side):
            q.fill_(NAN), k.fill_(NAN)
        side.synchronize()
        assert torch.equal(out, want)
    no_error()


@TYPES
def test_in_a_graph(dtype):
    """Captured once, replayed on other lengths and queries, several calls behind one another."""
    c = on_tc(attention_case(dtype, 14, 2, 64, 16, 6500, [40] * 90))
    q, lens, seen = c["q"].clone(), c["lens"].clone(), ints([6500] * 90)
    args = {**c, "q": q, "lens": lens}
    attend(args, prefix_lens=seen)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = attend(args, prefix_lens=seen)
        second = attend({**args, "q": first}, prefix_lens=seen)  # reads what the first has written
    for round in range(3):
        q.copy_(torch.randn_like(q.float()).to(dtype))
        lens.copy_(ints([(b * 7 + round) % 41 for b in range(90)]))
        seen.copy_(ints([LENS[(b + round) % 20] for b in range(90)]))
        graph.replay()
        torch.cuda.synchronize()
        a, b = first.clone(), second.clone()
        want = attend(args, prefix_lens=seen)
        assert torch.equal(a, want) and torch.equal(b, attend({**args, "q": want}, prefix_lens=seen))
    no_error()
