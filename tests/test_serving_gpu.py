"""The batched decode operators (rope_append, prefix_attention, sample) on the GPU against
plain implementations in 64 bits.

Tolerances follow from the arithmetic, with u(type) = 2^-24, 2^-11, 2^-8 the unit roundoff
of F32, F16, BF16: each result is rounded once to its type (u |result|), on top of
* rope_append: at most four 32-bit roundings of terms bounded by |a| + |z| + |bias|;
* prefix_attention: scores within (head_dim + 4) 2^-24 of sum |scale q k|, which moves a
  weight by that much relatively, numerator and sum alike; each weight may be rounded to
  the values' type before the product with them (u of a 16-bit type), and the sum over n
  keys adds n 2^-24; all relative to sum p |v|;
* sample: whole numbers, equal; a draw or a cut is placed midway between two running sums,
  so that the last bits of exp cannot move it; a probability has two roundings of exp.
"""
import math

import pytest

import tmac_zynq_fpga_b200 as tm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}  # steps of the subnormals
NAN, INF = math.nan, math.inf


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def no_error():
    torch.cuda.synchronize()
    assert tm.device_error(0) == 0


def bounds_error():
    torch.cuda.synchronize()
    assert tm.device_error(0) == -4


# ------------------------------------------------------------- rope_append --

def plain_rope(x, cos, sin, pos, interleaved):
    """float64 rotation of [tokens, heads, dim], and the bound |a| + |z| of each value's terms."""
    y, size = x.clone(), x.abs()
    half = cos.shape[1]
    for i in range(half):
        a, z = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos.double()[pos, i][:, None], sin.double()[pos, i][:, None]
        y[..., a], y[..., z] = x[..., a] * c - x[..., z] * s, x[..., a] * s + x[..., z] * c
        size[..., a] = size[..., z] = x[..., a].abs() + x[..., z].abs()
    return y, size


def append_case(dtype, ctype, heads, kv_heads, dim, rot, page, tokens, interleaved=True, bias=True, pad=0, offset=0, n_seq=3, seed=0):
    """Random inputs whose q, k, v lie in one buffer of `pad` extra values per token, from value `offset` on."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    row = (heads + 2 * kv_heads) * dim
    buf = torch.randn(tokens * (row + pad) + offset, generator=g, device="cuda").to(dtype)
    rows = buf[offset:].view(tokens, row + pad)
    nq, nk = heads * dim, kv_heads * dim
    q, k, v = (rows[:, a:b].unflatten(1, (-1, dim)) for a, b in ((0, nq), (nq, nq + nk), (nq + nk, row)))
    seq = ints([t % n_seq for t in range(tokens)])
    starts = ints([5 * s for s in range(n_seq)])
    pos = ints([5 * (t % n_seq) + 2 + t // n_seq for t in range(tokens)])
    width = -(-(3 + tokens // n_seq) // page)
    total = n_seq * width + 2
    tables = torch.randperm(total, generator=g, device="cuda")[:n_seq * width].int().view(n_seq, width).contiguous()
    cos, sin = tm.rope_table(int(pos.max()) + 1, rot) if rot else (torch.zeros(int(pos.max()) + 1, 0, device="cuda"),) * 2
    pools = [torch.randn((total, kv_heads, page, dim), generator=g, device="cuda").to(ctype) for _ in range(2)]
    b = torch.randn(row, generator=g, device="cuda") if bias else None
    return dict(q=q, k=k, v=v, seq=seq, pos=pos, starts=starts, tables=tables, cos=cos, sin=sin, pools=pools, bias=b, interleaved=interleaved)


def check_append(c):
    kc, vc = (p.clone() for p in c["pools"])
    cache = tm.PagedCache(kc, vc)
    out = tm.rope_append(cache, c["q"], c["k"], c["v"], c["pos"], c["tables"], c["cos"], c["sin"], seq=c["seq"], starts=c["starts"],
                         interleaved=c["interleaved"], bias=c["bias"])
    no_error()
    ct, dim = kc.dtype, kc.shape[3]
    h, hk = c["q"].shape[1], c["k"].shape[1]
    x = torch.cat([c["q"], c["k"], c["v"]], 1).double()
    if c["bias"] is not None:
        x = x + c["bias"].double().view(1, -1, dim)
    pos = c["pos"].long()
    y, size = plain_rope(x[:, :h + hk], c["cos"], c["sin"], pos, c["interleaved"])
    y, size = torch.cat([y, x[:, h + hk:]], 1), torch.cat([size, x[:, h + hk:].abs()], 1)
    if c["bias"] is not None:
        size = size + c["bias"].double().abs().view(1, -1, dim)
    tol = U[ct] * y.abs() + 4 * 2.0 ** -24 * size + TINY[ct]
    assert out.dtype == ct and ((out.double() - y[:, :h]).abs() <= tol[:, :h]).all()
    own = pos - c["starts"].long()[c["seq"].long()]
    page = kc.shape[2]
    at = c["tables"].long()[c["seq"].long(), own // page]
    for pool, old, a, b in ((kc, c["pools"][0], h, h + hk), (vc, c["pools"][1], h + hk, h + 2 * hk)):
        assert ((pool[at, :, own % page].double() - y[:, a:b]).abs() <= tol[:, a:b]).all()
        back = pool.clone()
        back[at, :, own % page] = old[at, :, own % page]
        assert torch.equal(back, old)  # nothing else was touched


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("ctype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_append_types(dtype, ctype, interleaved):
    check_append(append_case(dtype, ctype, 14, 2, 64, 64, 16, 37, interleaved))


@pytest.mark.parametrize("heads,kv_heads,dim,rot,page", [(1, 1, 2, 2, 1), (3, 1, 6, 4, 2), (4, 4, 80, 32, 8), (16, 4, 128, 96, 64),
                                                         (5, 5, 128, 128, 256), (6, 2, 64, 0, 16), (2, 2, 72, 24, 4), (8, 1, 64, 20, 32)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_layouts(heads, kv_heads, dim, rot, page, interleaved, dtype):
    check_append(append_case(dtype, dtype, heads, kv_heads, dim, rot, page, 29, interleaved, bias=rot != 96))


@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (64, 4), (1, 7)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_strides_and_alignment(pad, offset, dtype):
    for interleaved in (True, False):
        check_append(append_case(dtype, BF16, 14, 2, 64, 64, 16, 11, interleaved, pad=pad, offset=offset))


@pytest.mark.parametrize("tokens", [1, 2, 3, 500, 6001])
def test_append_lengths(tokens):
    check_append(append_case(BF16, BF16, 14, 2, 64, 64, 32, tokens, n_seq=min(tokens, 7)))


# more places in a token than a CTA has threads, and few; several tokens a CTA, ragged at the end
@pytest.mark.parametrize("heads,kv_heads,dim", [(48, 8, 128), (70, 2, 128), (1, 1, 16), (2, 1, 64)])
@pytest.mark.parametrize("tokens", [1, 1999, 9500])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_append_many_and_few_heads(heads, kv_heads, dim, tokens, interleaved, dtype):
    if heads * tokens > 200000:
        tokens = 3001
    check_append(append_case(dtype, F16, heads, kv_heads, dim, dim if dim == 16 else dim // 2, 32, tokens, interleaved, n_seq=min(tokens, 5)))


def test_append_padding_and_bounds():
    c = append_case(F32, F32, 2, 1, 64, 64, 8, 6, n_seq=6)
    kc, vc = (p.clone() for p in c["pools"])
    cache = tm.PagedCache(kc, vc)

    def call(**kw):
        d = {**c, **kw}
        return tm.rope_append(cache, d["q"], d["k"], d["v"], d["pos"], d["tables"], d["cos"], d["sin"], seq=d["seq"], starts=d["starts"])

    out = call(seq=ints([-1] * 6))
    no_error()  # padding is no error
    assert not out.any() and torch.equal(kc, c["pools"][0]) and torch.equal(vc, c["pools"][1])
    good = call()
    no_error()
    kc.copy_(c["pools"][0]), vc.copy_(c["pools"][1])
    for kw, zero in ((dict(seq=ints([6] * 6)), True), (dict(pos=c["pos"] + 10 ** 6), True), (dict(pos=c["pos"] - 10 ** 6), True),
                     (dict(starts=c["pos"] + 1), False), (dict(starts=c["pos"] - 10 ** 6), False),
                     (dict(tables=torch.full_like(c["tables"], -1)), False), (dict(tables=c["tables"] + 10 ** 6), False)):
        out = call(**kw)
        bounds_error()
        assert torch.equal(kc, c["pools"][0]) and torch.equal(vc, c["pools"][1])
        assert not out.any() if zero else (out.shape == good.shape and out.any())


def test_append_one_token_per_sequence_without_seq():
    c = append_case(BF16, BF16, 14, 2, 64, 64, 16, 5, n_seq=5)
    k1, v1, k2, v2 = (p.clone() for p in c["pools"] * 2)
    args = c["q"], c["k"], c["v"], c["pos"], c["tables"], c["cos"], c["sin"]
    a = tm.rope_append(tm.PagedCache(k1, v1), *args, seq=c["seq"], starts=c["starts"])
    b = tm.rope_append(tm.PagedCache(k2, v2), *args, starts=c["starts"])
    assert torch.equal(a, b) and torch.equal(k1, k2) and torch.equal(v1, v2)


def test_append_past_32_bit_offsets():
    # 2^31 elements lie before the last page of this pool (4.3 GB of f16 each)
    page, hk, dim = 256, 2, 64
    n = 2 ** 31 // (page * hk * dim) + 3
    k, v = (torch.zeros((n, hk, page, dim), dtype=F16, device="cuda") for _ in range(2))
    c = append_case(F16, F16, 2, hk, dim, dim, page, 2, n_seq=2)
    tables = ints([[n - 1], [n - 2]])
    tm.rope_append(tm.PagedCache(k, v), c["q"], c["k"], c["v"], c["pos"], tables, c["cos"], c["sin"], starts=c["starts"])
    no_error()
    assert torch.equal(v[n - 1, :, 2], c["v"][0]) and torch.equal(v[n - 2, :, 2], c["v"][1])
    out = tm.prefix_attention(torch.zeros((2, 2, dim), dtype=F16, device="cuda"), tm.PagedCache(k, v), tables, ints([3, 3]))
    no_error()
    want = torch.stack([c["v"][0], c["v"][1]]).double() / 3  # equal weights over two zero rows and this one
    assert ((out.double() - want).abs() <= (2 * U[F16] + 2.0 ** -20) * want.abs() + TINY[F16]).all()
    assert v.count_nonzero() <= 2 * hk * dim


# -------------------------------------------------------- prefix_attention --

def attention_case(dtype, heads, kv_heads, dim, page, prefix, own, queries=None, prefix_lens=None, seed=0, poison=True, spread=2.0,
                   pad=0):
    """A pool whose every place that no sequence owns holds NaN, and the plain result with its tolerance."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch = len(own)
    n_q = queries or [1] * batch
    shared = -(-prefix // page)
    width = max(1, -(-max(own) // page))
    total = shared + batch * width + 1
    order = torch.randperm(total, generator=g, device="cuda").int()
    tables = order[shared:shared + batch * width].view(batch, width).clone()
    k, v = (torch.full((total, kv_heads, page, dim), NAN if poison else 0.0, device="cuda", dtype=dtype) for _ in range(2))
    pages = order[:shared].clone()

    def fill(pages, n):
        rows = [torch.randn((n, kv_heads, dim), generator=g, device="cuda").to(dtype) for _ in range(2)]
        at = torch.arange(n, device="cuda")
        for pool, r in zip((k, v), rows):
            pool[pages.long()[at // page], :, at % page] = r
        return [r.double() for r in rows]

    pk, pv = fill(pages, prefix)
    tokens = sum(n_q)
    wide = torch.randn((tokens, heads * dim + pad), generator=g, device="cuda").mul_(spread).to(dtype)
    q = wide[:, :heads * dim].unflatten(1, (heads, dim))
    want, tol = torch.zeros((tokens, heads, dim), dtype=torch.float64, device="cuda"), None
    tol = torch.zeros_like(want)
    t, scale = 0, dim ** -0.5
    for b in range(batch):
        ok, ov = fill(tables[b], own[b])
        for p in range(-(-own[b] // page), width):
            tables[b, p] = -1
        seen_p = prefix if prefix_lens is None else prefix_lens[b]
        for i in range(n_q[b]):
            n = max(0, own[b] - n_q[b] + 1 + i)
            keys = torch.cat([pk[:seen_p], ok[:n]]).repeat_interleave(heads // kv_heads, 1)
            vals = torch.cat([pv[:seen_p], ov[:n]]).repeat_interleave(heads // kv_heads, 1)
            if len(keys):
                terms = q[t].double() * keys * scale  # [keys, heads, dim]
                p = torch.softmax(terms.sum(2), 0)
                want[t] = torch.einsum("kh,khd->hd", p, vals)
                size = torch.einsum("kh,khd->hd", p, vals.abs())
                off = 2 * (dim + 4) * 2.0 ** -24 * terms.abs().sum(2).amax(0)[:, None] + (len(keys) + 16) * 2.0 ** -24
                tol[t] = U[dtype] * want[t].abs() + (off + (U[dtype] if dtype != F32 else 0)) * size + TINY[dtype]
            t += 1
    start = [sum(n_q[:b]) for b in range(batch + 1)]
    kw = dict(prefix_pages=pages if prefix else None, prefix_len=prefix, prefix_lens=None if prefix_lens is None else ints(prefix_lens))
    if queries:
        kw.update(q_start=ints(start), max_q=max(n_q))
    return dict(q=q, k=k, v=v, tables=tables, lens=ints(own), kw=kw, want=want, tol=tol)


def attend(c, **kw):
    return tm.prefix_attention(c["q"], tm.PagedCache(c["k"], c["v"]), c["tables"], c["lens"], **{**c["kw"], **kw})


def check_attention(c, **kw):
    out = attend(c, **kw)
    no_error()
    assert out.dtype == c["q"].dtype
    off = (out.double() - c["want"]).abs() - c["tol"]
    assert (off <= 0).all(), f"worst {off.max().item():.3g} past the tolerance"
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (16, 4, 128), (8, 8, 64), (12, 1, 128), (9, 3, 64), (40, 1, 64), (1, 1, 128)])
@pytest.mark.parametrize("prefix,own", [(75, [1, 40, 17]), (0, [5, 64, 65]), (300, [0, 3, 130])])
def test_attention_heads_and_types(dtype, heads, kv_heads, dim, prefix, own):
    check_attention(attention_case(dtype, heads, kv_heads, dim, 16, prefix, own))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 64, 128, 256])
def test_attention_page_sizes(dtype, page):
    check_attention(attention_case(dtype, 14, 2, 64, page, 133, [1, 66, 31, 9]))
    check_attention(attention_case(dtype, 4, 2, 128, page, 257, [128, 2]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4099])
def test_attention_lengths(dtype, n):
    check_attention(attention_case(dtype, 14, 2, 64, 16, n, [1, 2]))       # a prefix of that length
    check_attention(attention_case(dtype, 14, 2, 64, 16, 0, [n, 1]))       # an own part of that length
    check_attention(attention_case(dtype, 4, 2, 128, 32, n, [n // 2 + 1]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch", [1, 9, 10, 19, 64, 150])
def test_attention_row_tiles(dtype, batch):
    own = [b * 13 % 40 for b in range(batch)]
    check_attention(attention_case(dtype, 14, 2, 64, 16, 200, own))
    check_attention(attention_case(dtype, 4, 1, 128, 16, 333, own))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_many_rows_over_a_long_prefix(dtype):
    check_attention(attention_case(dtype, 14, 2, 64, 64, 5003, [b % 7 for b in range(75)]))
    check_attention(attention_case(dtype, 16, 4, 128, 16, 3001, [b % 50 for b in range(70)]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (8, 4, 128)])
def test_attention_several_query_tokens(dtype, heads, kv_heads, dim):
    queries = [1, 5, 0, 3, 40, 2]
    check_attention(attention_case(dtype, heads, kv_heads, dim, 16, 100, [4, 5, 9, 200, 77, 2], queries))
    # fewer own keys than queries: the first ones see the prefix alone, or nothing
    check_attention(attention_case(dtype, heads, kv_heads, dim, 16, 50, [0, 2, 0, 1, 39, 2], queries))
    check_attention(attention_case(dtype, heads, kv_heads, dim, 16, 0, [0, 2, 0, 1, 39, 2], queries))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_sequences_that_leave_the_prefix(dtype):
    for prefix, lens in ((210, [0, 210, 1, 100, 64, 128, 209]), (3000, [3000, 0, 5, 1500, 2999, 64, 2048])):
        check_attention(attention_case(dtype, 14, 2, 64, 16, prefix, [0, 0, 3, 70, 1, 2, 9], prefix_lens=lens))
        check_attention(attention_case(dtype, 14, 2, 64, 16, prefix, [0, 0, 3, 70, 1, 2, 9], [3, 0, 4, 1, 2, 1, 30], prefix_lens=lens))
        many = lens * 9
        check_attention(attention_case(dtype, 14, 2, 64, 64, prefix, [b % 5 for b in range(63)], prefix_lens=many))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_peaked_and_large_scores(dtype):
    check_attention(attention_case(dtype, 14, 2, 64, 16, 500, [3, 90], spread=30.0))
    check_attention(attention_case(dtype, 14, 2, 64, 16, 500, [b % 20 for b in range(40)], spread=30.0))
    check_attention(attention_case(dtype, 14, 2, 64, 16, 500, [3, 90], spread=0.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("batch", [2, 60])
def test_attention_unseen_values_do_not_reach_a_row(dtype, bad, batch):
    """The second half of the sequences shares the prefix past position 150; only those may notice what lies there."""
    lens = [150 if b < batch // 2 else 200 for b in range(batch)]
    c = attention_case(dtype, 14, 2, 64, 16, 200, [b % 4 for b in range(batch)], prefix_lens=lens)
    p = c["kw"]["prefix_pages"].long()
    for pool in (c["k"], c["v"]):
        pool[p[170 // 16], :, 170 % 16] = bad
    out = attend(c)
    no_error()
    first = batch // 2
    assert ((out[:first].double() - c["want"][:first]).abs() <= c["tol"][:first]).all()
    assert not torch.isfinite(out[first:]).any() or bad == -INF  # a key of -inf may weigh nothing


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_strided_rows(dtype):
    for pad in (8, 3, 1):
        c = attention_case(dtype, 14, 2, 64, 16, 70, [9, 30], pad=pad)
        plain = check_attention(c)
        wide = torch.zeros((2, 14 * 64 + pad), dtype=dtype, device="cuda")
        out = wide[:, pad:].unflatten(1, (14, 64))
        assert attend(c, out=out) is out
        assert torch.equal(out, plain) and not wide[:, :pad].any()
        one = tm.prefix_attention(c["q"][:1], tm.PagedCache(c["k"], c["v"]), c["tables"][:1], c["lens"][:1], **c["kw"])
        assert ((one.double() - c["want"][:1]).abs() <= c["tol"][:1]).all()


def test_attention_scale_and_bound_on_lengths():
    c = attention_case(F32, 14, 2, 64, 16, 90, [30, 12])
    a = attend(c, scale=0.125, max_own=30)
    b = check_attention(c)
    assert ((a.double() - c["want"]).abs() <= c["tol"]).all() and ((a - b).abs() <= 2 * c["tol"]).all()
    doubled = attend({**c, "q": c["q"] * 2}, scale=0.0625)
    assert ((doubled.double() - c["want"]).abs() <= c["tol"]).all()


def test_attention_of_nothing_is_zero():
    for dtype in (F32, BF16):
        c = attention_case(dtype, 14, 2, 64, 16, 0, [0, 0, 0])
        assert not check_attention(c).any()
        assert not attend(c, max_own=0).any()
    empty = tm.prefix_attention(c["q"][:0], tm.PagedCache(c["k"], c["v"]), c["tables"][:0], c["lens"][:0])
    assert empty.shape == (0, 14, 64)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_bounds_are_errors_not_accesses(dtype):
    c = attention_case(dtype, 14, 2, 64, 16, 64, [20, 40], poison=False)
    good = check_attention(c)
    for what, kw in (("lens", dict(lens=c["lens"] + 10 ** 6)), ("tables", dict(tables=c["tables"] + 10 ** 6)),
                     ("tables", dict(tables=torch.full_like(c["tables"], -7)))):
        attend({**c, **kw})
        bounds_error()
    attend(c, prefix_pages=c["kw"]["prefix_pages"] + 10 ** 6)
    bounds_error()
    out = attend(c, prefix_lens=ints([10 ** 6, 64]))
    bounds_error()
    assert torch.equal(out, good)  # counts as all of it
    attend(c, q_start=ints([0, 2, 2]), max_q=1)
    bounds_error()
    attend({**c, "lens": ints([-5, 40])})
    no_error()  # a negative length is none
    # a page outside the pool counts as zeros: here one of the prefix's
    pages = c["kw"]["prefix_pages"].clone()
    c["k"][pages[1].long()], c["v"][pages[1].long()] = 0, 0
    want = attend(c)
    no_error()
    pages[1] = 10 ** 6
    out = attend(c, prefix_pages=pages)
    bounds_error()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_is_the_same_every_time(dtype):
    c = attention_case(dtype, 14, 2, 64, 16, 2000, [b * 37 % 300 for b in range(40)])
    a = attend(c)
    assert all(torch.equal(a, attend(c)) for _ in range(5))


def test_attention_python_refusals():
    c = attention_case(F32, 14, 2, 64, 16, 64, [20, 40])
    for kw in (dict(prefix_len=65), dict(out=torch.empty(1, device="cuda")), dict(prefix_lens=torch.zeros(2, device="cuda")),
               dict(q_start=ints([0, 2]), max_q=2), dict(prefix_pages=c["kw"]["prefix_pages"].cpu()), dict(max_own=49)):
        with pytest.raises(tm.TmacError):
            attend(c, **kw)
    for kw in (dict(q=c["q"].half()), dict(q=c["q"].cpu()), dict(q=c["q"][:, :, :32]), dict(q=c["q"][:, ::2]),
               dict(lens=c["lens"].long()), dict(tables=c["tables"].t())):
        with pytest.raises(tm.TmacError):
            attend({**c, **kw})


# ------------------------------------------------------------------ sample --

def order_of(row, temperature):
    """(indexes in order, their d, their 64-bit weights) of one row, or None when it is empty."""
    x = row.float()
    if temperature > 0:
        x = x * (1.0 / torch.tensor(temperature, dtype=F32, device=row.device))
    x = torch.where(torch.isnan(x), -INF, x)
    top = x.max()
    if top == -INF:
        return None
    d = torch.where(x == top, 0.0, top - x)
    at = torch.sort(d, stable=True).indices
    return at, d[at], torch.floor(2.0 ** 32 * torch.exp(-d[at].double()))


def kept_count(d, w, k=0, p=1.0, m=0.0):
    """How many of the order are kept.  p is moved midway between two running sums; the p to use is returned too."""
    n = k if 0 < k < len(d) else len(d)
    if p < 1:
        sums = w[:n].cumsum(0)
        total = float(sums[-1])
        j = int((sums < p * total).sum())
        low = float(sums[j - 1]) if j else 0.0
        p = (low + float(sums[j])) / 2 / total
        n = j + 1
    if m > 0:
        n = min(n, int((torch.exp(-d.double()) >= m).sum()))
    return n, p


def sample_one(logits, **kw):
    """One call for many rows; kw: lists per row."""
    def vec(name, dtype):
        return torch.tensor(kw[name], dtype=dtype, device="cuda") if name in kw else None
    tokens, probs = tm.sample(logits, vec("u", F32), temperature=vec("temperature", F32), top_k=vec("top_k", torch.int32),
                              top_p=vec("top_p", F32), min_p=vec("min_p", F32))
    no_error()
    return tokens.tolist(), probs.tolist()


def check_sample(logits, temperature=1.0, k=0, p=1.0, m=0.0, draws=12, seed=0):
    """Rows of one setting: the first and last kept token, and draws placed in the middle of a kept token's weight."""
    g = torch.Generator().manual_seed(seed)
    rows, kw, want = [], dict(u=[], temperature=[], top_k=[], top_p=[], min_p=[]), []
    for row in logits:
        at, d, w = order_of(row, temperature)
        n, p_used = kept_count(d, w, k, p, m)
        kept, back = torch.sort(at[:n])
        weights = w[:n][back]
        sums = weights.cumsum(0)
        total = float(sums[-1])
        picks = [int(torch.searchsorted(sums, torch.tensor(float(r) * total, dtype=torch.float64, device="cuda"), right=True))
                 for r in torch.rand(draws, generator=g)]
        picks += [int(torch.nonzero(weights)[0]), int(torch.nonzero(weights)[-1])]
        for j in picks:
            j = min(j, n - 1)
            share = float(weights[j]) / total
            u = (float(sums[j]) - float(weights[j]) / 2) / total
            # u and the running sums are told apart from 2^-23 on: 32-bit u, weights within a few 2^-24 of theirs
            if share < 2.0 ** -21:
                continue
            rows.append(row)
            want.append((int(kept[j]), share))
            for name, value in (("u", min(u, 1 - 2.0 ** -24)), ("temperature", temperature), ("top_k", k), ("top_p", p_used), ("min_p", m)):
                kw[name].append(value)
    tokens, probs = sample_one(torch.stack(rows), **kw)
    assert len(want) >= len(logits)
    for (t, share), got, prob in zip(want, tokens, probs):
        assert got == t
        assert abs(prob - share) <= 16 * 2.0 ** -24 * share + 2.0 ** -30


def random_logits(n, vocab, dtype=F32, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + vocab)
    return (torch.randn((n, vocab), generator=g, device="cuda") * scale).to(dtype)


FILTERS = [dict(), dict(k=1), dict(k=3), dict(k=40), dict(k=10 ** 6), dict(p=0.3), dict(p=0.95), dict(p=0.0), dict(m=0.05), dict(m=1.0),
           dict(k=50, p=0.8), dict(k=500, p=0.5, m=0.02), dict(p=0.9, temperature=0.5), dict(k=20, temperature=2.5), dict(temperature=0.0),
           dict(temperature=1e-40)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 4096, 4097, 32003, 151936, 260001])
@pytest.mark.parametrize("f", FILTERS, ids=str)
def test_sample_filters(vocab, f):
    if f.get("p") == 0.0:  # one token, whatever u is
        logits = random_logits(4, vocab)
        tokens, probs = sample_one(logits, u=[0.0, 0.3, 0.7, 0.99], top_p=[0.0] * 4)
        assert tokens == logits.argmax(1).tolist() and probs == [1.0] * 4
    elif f.get("temperature", 1.0) <= 1e-40:
        logits = random_logits(4, vocab)
        tokens, probs = sample_one(logits, u=[0.0, 0.3, 0.7, 0.99], temperature=[f["temperature"]] * 4)
        assert tokens == logits.argmax(1).tolist() and probs == [1.0] * 4
    else:
        check_sample(random_logits(2, vocab), draws=6, **f)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("vocab", [5, 1001, 32003, 151936])
def test_sample_16_bit_logits_and_their_ties(dtype, vocab):
    logits = random_logits(2, vocab, dtype)
    for f in (dict(), dict(k=7), dict(k=300), dict(p=0.4), dict(k=300, p=0.9), dict(m=0.1)):
        check_sample(logits, draws=6, **f)


@pytest.mark.parametrize("vocab", [3, 1024, 5000, 151936])
def test_sample_all_equal_logits(vocab):
    """Every token ties: top-k keeps the lowest indexes, and the draw is uniform over them."""
    logits = torch.full((1, vocab), -2.5, device="cuda")
    for f in (dict(), dict(k=2), dict(k=vocab - 1), dict(k=min(vocab, 777), p=0.5), dict(p=0.25), dict(m=0.9)):
        check_sample(logits, **f)


@pytest.mark.parametrize("vocab", [100, 40000, 151936])
def test_sample_ties_at_the_cut(vocab):
    logits = torch.full((1, vocab), -4.0, device="cuda")
    logits[0, vocab // 2:vocab // 2 + 40] = 1.0
    logits[0, 3] = 2.0
    for k in (1, 2, 20, 41, 45):
        check_sample(logits, k=k)
    check_sample(logits, p=0.5)


def shaped_logits(shape, vocab):
    """A row whose likely tokens lie as `shape` says: any bound taken from a part of the row can then be far off."""
    row = random_logits(1, vocab, seed=3)[0]
    if shape == "falling":
        row = row.sort(descending=True).values
    elif shape == "rising":
        row = row.sort().values
    elif shape == "early":  # the first quarter above all others
        row[: vocab // 4] += 20.0
    elif shape == "late":
        row[-9:] += 20.0
    elif shape == "ties":
        row = (row / 2).round() * 2
    elif shape == "masked":
        row[: vocab // 2] = -INF
        row[vocab // 2 :: 3] = NAN
    elif shape == "equal":
        row[:] = -2.5
    elif shape == "wide":
        row *= 8
    return row[None].contiguous()


# more rows than the SMs hold: logits are read again, by one to four CTAs a row
@pytest.mark.parametrize("draws", [60, 300])
@pytest.mark.parametrize("vocab", [4099, 32003])
@pytest.mark.parametrize("shape", ["random", "falling", "rising", "early", "late", "ties", "masked", "equal", "wide"])
@pytest.mark.parametrize("f", [dict(k=2), dict(k=40), dict(k=199, p=0.9), dict(k=700), dict(p=0.8), dict(m=0.05), dict()], ids=str)
def test_sample_of_many_rows(f, shape, vocab, draws):
    check_sample(shaped_logits(shape, vocab), draws=draws, **f)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("k", [2, 40, 199])
def test_sample_of_many_16_bit_rows(dtype, k):
    check_sample(random_logits(1, 32003, dtype), draws=100, k=k)


def test_sample_of_many_rows_with_infinite_ones():
    logits = random_logits(200, 5000)
    logits[:100, 4000] = INF       # past the first quarter
    logits[50:100, 10] = INF       # and in it
    logits[100:150] = -INF
    tokens, probs = sample_one(logits, u=[0.6] * 200, top_k=[30] * 200)
    assert tokens[:50] == [4000] * 50 and probs[:50] == [1.0] * 50
    assert tokens[50:100] == [4000] * 50 and probs[50:100] == [0.5] * 50
    assert tokens[100:150] == [-1] * 50 and probs[100:150] == [0.0] * 50
    for row, token in zip(logits[150:], tokens[150:]):
        assert token in row.topk(30).indices.tolist()


def test_sample_masked_rows():
    v = 5000
    logits = random_logits(7, v)
    logits[0] = -INF
    logits[1] = NAN
    logits[2, :] = -INF
    logits[2, 4321] = -1e30
    logits[3, 100:] = -INF
    logits[4, 7] = INF
    logits[4, 77] = INF
    logits[5, ::2] = NAN
    logits[6] = torch.finfo(F32).min  # the type's lowest value is a value: a uniform row
    for f in (dict(), dict(top_k=[30] * 7), dict(top_p=[0.7] * 7), dict(min_p=[0.1] * 7), dict(top_k=[30] * 7, top_p=[0.5] * 7), dict(temperature=[0.0] * 7)):
        tokens, probs = sample_one(logits, u=[0.6] * 7, **f)
        assert tokens[:3] == [-1, -1, 4321] and probs[:3] == [0.0, 0.0, 1.0]
        assert 0 <= tokens[3] < 100 and tokens[5] % 2 == 1
        # two equal ones share row 4; top_p 0.5 is reached by the first of them alone
        one = "temperature" in f or 0.5 in f.get("top_p", [])
        assert (tokens[4], probs[4]) == ((7, 1.0) if one else (77, 0.5))
        assert 0 <= tokens[6] < v
    check_sample(logits[3:4], k=60)
    check_sample(logits[5:6], p=0.8)


def test_sample_rows_have_their_own_settings():
    logits = random_logits(6, 9000)
    at = [order_of(r, 1.0)[0] for r in logits]
    last = 1 - 2.0 ** -24
    tokens, probs = sample_one(logits, u=[last] * 6, temperature=[1.0, 0.0, -1.0, NAN, 1.0, 1.0], top_k=[2, 0, 5, 5, -3, 1],
                               top_p=[1.0, 0.5, 0.5, 0.5, 0.0, 0.9], min_p=[0.0, 0.0, 0.0, 0.0, 0.5, 0.0])
    assert tokens[0] == max(at[0][:2].tolist())
    assert tokens[1:] == [int(a[0]) for a in at[1:]] and probs[1:] == [1.0] * 5


def test_sample_u_outside_its_range_stays_inside_the_row():
    logits = random_logits(4, 3000)
    tokens, _ = sample_one(logits, u=[1.0, 5.0, -1.0, NAN], top_k=[4] * 4)
    for t, row in zip(tokens, logits):
        assert t in order_of(row, 1.0)[0][:4].tolist()


def test_sample_strided_rows():
    wide = random_logits(5, 4999 + 13)
    for part in (wide[:, 1:5000], wide[:, 13:], wide[::2, 4:300]):
        a = tm.sample(part, torch.full((len(part),), 0.4, device="cuda"))
        b = tm.sample(part.contiguous(), torch.full((len(part),), 0.4, device="cuda"))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_sample_of_one_row_for_many_draws():
    row = random_logits(1, 6000)
    u = torch.rand(50, device="cuda")
    k = torch.full((50,), 12, dtype=torch.int32, device="cuda")
    a, b = tm.sample(row.expand(50, -1), u, top_k=k), tm.sample(row.repeat(50, 1), u, top_k=k)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_sample_is_uniform_in_u():
    """Evenly spread u gives every kept token its weight's share of the draws."""
    logits = random_logits(1, 50, scale=1.0)
    n = 4096
    tokens, probs = tm.sample(logits.expand(n, -1).contiguous(), (torch.arange(n, device="cuda") + 0.5) / n,
                              top_k=torch.full((n,), 9, dtype=torch.int32, device="cuda"))
    at, d, w = order_of(logits[0], 1.0)
    for i in range(9):
        share = float(w[i] / w[:9].sum())
        assert abs(int((tokens == at[i]).sum()) - n * share) <= 1.01  # both ends of its interval


# ----------------------------------------------------------------- streams --

def test_operators_on_another_stream():
    """Inputs made, and results read, on a side stream; also given by address."""
    c = append_case(BF16, BF16, 14, 2, 64, 64, 16, 6, n_seq=6)
    cache = tm.PagedCache(*c["pools"])
    args = c["q"], c["k"], c["v"], c["pos"], c["tables"], c["cos"], c["sin"]
    lens = c["pos"] - c["starts"] + 1
    q = tm.rope_append(cache, *args, starts=c["starts"])
    want = tm.prefix_attention(q, cache, c["tables"], lens)
    logits = random_logits(6, 2000)
    u = torch.rand(6, device="cuda")
    tokens, _ = tm.sample(logits, u)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        q2 = tm.rope_append(cache, *args, starts=c["starts"], stream=stream)
        out = tm.prefix_attention(q2, cache, c["tables"], lens, stream=stream)
        t2, _ = tm.sample(logits, u, stream=stream)
        side.synchronize()
        assert torch.equal(q2, q) and torch.equal(out, want) and torch.equal(t2, tokens)
    with torch.cuda.stream(side):
        out = tm.prefix_attention(tm.rope_append(cache, *args, starts=c["starts"]), cache, c["tables"], lens)
    side.synchronize()
    assert torch.equal(out, want)


def test_operators_in_a_graph():
    """A captured step replays on new lengths, positions and random numbers."""
    c = append_case(BF16, BF16, 14, 2, 64, 64, 16, 4, n_seq=4)
    cache = tm.PagedCache(*c["pools"])
    pos, lens, u = c["pos"].clone(), c["pos"] - c["starts"] + 1, torch.rand(4, device="cuda")
    logits = random_logits(4, 3000)

    def step():
        q = tm.rope_append(cache, c["q"], c["k"], c["v"], pos, c["tables"], c["cos"], c["sin"], starts=c["starts"])
        return tm.prefix_attention(q, cache, c["tables"], lens), *tm.sample(logits, u)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    pos.sub_(1)
    lens.sub_(1)
    u.copy_(torch.rand(4, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in captured]
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    no_error()
