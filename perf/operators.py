"""The operators of a batched decode step: what is measured of them, and their plain forms.

* rope_append: the position rotation of q and k, with k and v appended to a paged cache.
* prefix_attention: attention of a batch whose sequences share a prefix, over that cache.
* sample: the next token of every sequence from its logits and a given random number.

`own` chooses between the plain forms written here (elementary torch operations in 32
bits, rounded once at the end) and the package's operators.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------- cases --

def listed():
    """The decode and prefill shapes of the 24-layer model that this package runs (14 query and 2 key/value heads of 64,
    151936 tokens), and generic ones beside them."""
    return [
        # the first step of two conversations after a short common instruction: latency
        _attention("attention first step", "bf16", 14, 2, 64, 16, batch=2, prefix=96, own=17),
        # the engine's own cache type, a 448-token prompt that 16 answers share, up to 64 steps into them
        _attention("attention 448 + 64 f32", "f32", 14, 2, 64, 16, batch=16, prefix=448, own=64),
        # an ordinary serving batch: a 2051-token instruction, answers of up to 509 tokens
        _attention("attention serving f16", "f16", 14, 2, 64, 32, batch=48, prefix=2051, own=509),
        # several proposed tokens checked at once, sequences that leave the prefix at different places, wider heads
        _attention("attention proposals bf16", "bf16", 16, 4, 128, 16, batch=24, prefix=1500, own=300, queries=7, branch=True),
        # many readers of one long document
        _attention("attention long bf16", "bf16", 14, 2, 64, 64, batch=128, prefix=32768, own=1024),
        # one decode step's q, k and v of two sequences: latency
        _append("append step", "f32", "f32", 14, 2, 64, 64, 16, tokens=2, bias=True, interleaved=True),
        # a prompt of 512 tokens in the engine's 32-bit activations, into a 16-bit cache
        _append("append prompt", "f32", "bf16", 14, 2, 64, 64, 16, tokens=512, bias=True, interleaved=True),
        # the prefill benchmark's 64 x 512 tokens, wider heads of which three quarters are rotated, halves paired
        _append("append prefill", "bf16", "bf16", 16, 4, 128, 96, 64, tokens=32768, bias=False, interleaved=False),
        # one conversation: top-k 40 of the whole vocabulary
        _sample("sample one", "f32", 1, 151936, filters="k"),
        # a batch with another choice of filters in every row, some tokens forbidden
        _sample("sample mixed", "f32", 32, 151936, filters="mixed", banned=True),
        # a smaller odd vocabulary in 16 bits, top-p
        _sample("sample odd bf16", "bf16", 77, 32003, filters="p"),
        # a large batch, top-k and top-p together
        _sample("sample large", "f32", 256, 151936, filters="kp"),
    ]


def _attention(name, dtype, heads, kv_heads, dim, page, batch, prefix, own, queries=1, branch=False):
    c = dict(op="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, batch=batch, prefix=prefix,
             own=own, queries=queries, branch=branch)
    return dict(c, name=name) if name else c


def _append(name, dtype, cache, heads, kv_heads, dim, rot, page, tokens, bias, interleaved):
    c = dict(op="append", dtype=dtype, cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, page=page,
             tokens=tokens, bias=bias, interleaved=interleaved)
    return dict(c, name=name) if name else c


def _sample(name, dtype, batch, vocab, filters, banned=False):
    c = dict(op="sample", dtype=dtype, batch=batch, vocab=vocab, filters=filters, banned=banned)
    return dict(c, name=name) if name else c


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "attention":
        heads, kv_heads, dim = rng.choice([(14, 2, 64), (16, 4, 128), (8, 8, 64), (12, 1, 128), (32, 8, 128), (9, 3, 64)])
        batch, prefix, queries = _spread(rng, 1, 128), _spread(rng, 1, 32768), rng.choice([1, 1, 1, 2, 5])
        # no costlier than the longest listed one
        while heads * dim * batch * queries * prefix > 14 * 64 * 128 * 32768 // 2:
            prefix //= 2
        return _attention(None, dtype, heads, kv_heads, dim, rng.choice([16, 32, 64, 128]), batch, prefix,
                          _spread(rng, 1, min(1024, 32768 // batch)), queries, rng.random() < 0.3)
    if op == "append":
        heads, kv_heads, dim, rot = rng.choice([(14, 2, 64, 64), (16, 4, 128, 96), (8, 8, 64, 32), (12, 1, 128, 128)])
        return _append(None, dtype, rng.choice(["f32", "bf16", "f16"]), heads, kv_heads, dim, rot,
                       rng.choice([16, 32, 64, 128]), _spread(rng, 1, 16000), rng.random() < 0.5, rng.random() < 0.5)
    vocab = _spread(rng, 1000, 260000)
    return _sample(None, dtype, _spread(rng, 1, max(1, min(256, 256 * 151936 // vocab))), vocab,
                   rng.choice(["", "k", "p", "kp", "m", "mixed"]), rng.random() < 0.5)


# ---------------------------------------------------------- sizes of a case --

def _own_lens(c):
    """Keys of each sequence's own, its queries' among them: ragged, from 1 (or its queries) to `own`."""
    return [max(min(c["own"], q), (b * 7919 + 13) % c["own"] + 1) for b, q in enumerate(_query_lens(c))]


def _query_lens(c):
    return [b * 5 % c["queries"] + 1 for b in range(c["batch"])]


def _prefix_lens(c):
    """How much of the prefix each sequence shares: all of it, or up to where it left it (some share none)."""
    if not c["branch"]:
        return [c["prefix"]] * c["batch"]
    return [b * 37 % 5 * c["prefix"] // 4 for b in range(c["batch"])]


def work(case):
    c = case
    if c["op"] == "attention":
        e, pairs, own = BYTES[c["dtype"]], 0, _own_lens(c)
        for n, ln, p in zip(_query_lens(c), own, _prefix_lens(c)):
            pairs += n * p + sum(max(0, ln - n + 1 + i) for i in range(n))
        keys = max(_prefix_lens(c)) + sum(own)
        return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * e + 2 * sum(_query_lens(c)) * c["heads"] * c["dim"] * e,
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    if c["op"] == "append":
        n = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": n * (BYTES[c["dtype"]] + BYTES[c["cache"]]) + c["tokens"] * (c["rot"] * 4 + 12),
                "flops": c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rot"] * 3 + (n if c["bias"] else 0)}
    n = c["batch"] * c["vocab"]
    return {"bytes": n * BYTES[c["dtype"]] + c["batch"] * 28, "flops": 4 * n}


# ------------------------------------------------------------------ inputs --

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": _inputs_attention, "append": _inputs_append, "sample": _inputs_sample}[case["op"]](dict(case), g)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs_attention(c, g):
    dt, ps = TYPES[c["dtype"]], c["page"]
    lens, qlens = _own_lens(c), _query_lens(c)
    width, shared = -(-c["own"] // ps), -(-c["prefix"] // ps)
    pages = [-(-n // ps) for n in lens]
    total = shared + sum(pages)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)  # pages lie anywhere in the pool
    tables = torch.full((c["batch"], width), -1, dtype=torch.int32, device="cuda")
    at = shared
    for b, n in enumerate(pages):
        tables[b, :n] = order[at:at + n]
        at += n
    pool = (total, c["kv_heads"], ps, c["dim"])
    tokens = sum(qlens)
    return {
        "case": c, "q": _normal(g, (tokens, c["heads"], c["dim"]), dt, 2.0), "k": _normal(g, pool, dt), "v": _normal(g, pool, dt),
        "tables": tables, "lens": _ints(lens), "prefix_pages": order[:shared].contiguous(), "scale": c["dim"] ** -0.5,
        "prefix_lens": _ints(_prefix_lens(c)) if c["branch"] else None,
        "q_start": _ints([sum(qlens[:b]) for b in range(c["batch"] + 1)]) if c["queries"] > 1 else None,
    }


def _inputs_append(c, g):
    dt, ct, ps, d, t = TYPES[c["dtype"]], TYPES[c["cache"]], c["page"], c["dim"], c["tokens"]
    # one sequence for every 512 tokens of a prompt, or for every token of a step; each starts after its past
    n_seq = t if t <= 64 else -(-t // 512)
    per = -(-t // n_seq)
    seq = torch.arange(t, device="cuda", dtype=torch.int32) // per
    first = torch.randint(0, 100, (n_seq,), generator=g, device="cuda", dtype=torch.int32)
    pos = first[seq.long()] + torch.arange(t, device="cuda", dtype=torch.int32) % per
    width = -(-(per + 100) // ps)
    tables = torch.randperm(n_seq * width, generator=g, device="cuda").to(torch.int32).view(n_seq, width)
    rows = _normal(g, (t, (c["heads"] + 2 * c["kv_heads"]) * d), dt)  # the projection's output: q | k | v
    nq, nk = c["heads"] * d, c["kv_heads"] * d
    half = c["rot"] // 2
    angle = torch.arange(per + 100, device="cuda", dtype=torch.float64)[:, None] * (
        1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
    pool = (n_seq * width, c["kv_heads"], ps, d)
    return {
        "case": c, "q": rows[:, :nq].unflatten(1, (-1, d)), "k": rows[:, nq:nq + nk].unflatten(1, (-1, d)),
        "v": rows[:, nq + nk:].unflatten(1, (-1, d)), "pos": pos, "seq": seq, "tables": tables,
        "cos": angle.cos().float(), "sin": angle.sin().float(),
        "bias": _normal(g, (nq + 2 * nk,), torch.float32, 0.02) if c["bias"] else None,
        "k_pages": _normal(g, pool, ct), "v_pages": _normal(g, pool, ct),
    }


def _inputs_sample(c, g):
    b, v = c["batch"], c["vocab"]
    logits = torch.randn((b, v), generator=g, device="cuda") * 2.0
    # a few likely tokens above the rest
    likely = torch.randint(0, v, (b, 64), generator=g, device="cuda")
    logits.scatter_add_(1, likely, torch.rand((b, 64), generator=g, device="cuda") * 9.0)
    if c["banned"]:
        logits[torch.rand((b, v), generator=g, device="cuda") < 0.02] = -math.inf
    u = lambda lo, hi: lo + (hi - lo) * torch.rand((b,), generator=g, device="cuda")  # noqa: E731
    kinds = torch.arange(b, device="cuda") % 6  # of a mixed batch: none, k, p, m, all three, greedy
    f, temperature = c["filters"], u(0.6, 1.3)
    k = torch.randint(1, 200, (b,), generator=g, device="cuda", dtype=torch.int32) if b > 1 else _ints([40])
    p, m = u(0.5, 0.99), u(0.01, 0.2)
    if f == "mixed":
        k = torch.where((kinds == 1) | (kinds == 4), k, 0)
        p = torch.where((kinds == 2) | (kinds == 4), p, 1.0)
        m = torch.where((kinds == 3) | (kinds == 4), m, 0.0)
        temperature = torch.where(kinds == 5, 0.0, temperature)
    mixed = f == "mixed"
    return {"case": c, "logits": logits.to(TYPES[c["dtype"]]), "u": u(0.0, 1.0).clamp_(max=1 - 2.0 ** -24), "temperature": temperature,
            "top_k": k if mixed or "k" in f else None, "top_p": p if mixed or "p" in f else None,
            "min_p": m if mixed or "m" in f else None}


# -------------------------------------------------------------------- runs --

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"attention": _plain_attention, "append": _plain_append, "sample": _plain_sample}[op](state)


def _own(op, s):
    import tmac_zynq_fpga_b200 as tm

    if op == "attention":
        return tm.prefix_attention(s["q"], tm.PagedCache(s["k"], s["v"]), s["tables"], s["lens"],
                                   prefix_pages=s["prefix_pages"], prefix_len=s["case"]["prefix"], prefix_lens=s["prefix_lens"],
                                   q_start=s["q_start"], max_q=s["case"]["queries"], scale=s["scale"])
    if op == "append":
        q = tm.rope_append(tm.PagedCache(s["k_pages"], s["v_pages"]), s["q"], s["k"], s["v"], s["pos"], s["tables"], s["cos"], s["sin"],
                           seq=s["seq"], interleaved=s["case"]["interleaved"], bias=s["bias"])
        return q, s["k_pages"], s["v_pages"]
    return tm.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _plain_attention(s):
    """Softmax over the prefix's keys and the sequence's own, the prefix's products made once for all rows."""
    c, q, dev = s["case"], s["q"], s["q"].device
    t, h, d = q.shape
    hk, b, ps = c["kv_heads"], c["batch"], c["page"]
    g, n, p_len = h // hk, c["queries"], c["prefix"]
    qf = (q.float() * s["scale"]).view(t, hk, g, d)
    if s["q_start"] is None:
        tok_seq, tok_i, n_q = torch.arange(t, device=dev), torch.zeros(t, dtype=torch.int64, device=dev), torch.ones(b, dtype=torch.int64, device=dev)
    else:
        start = s["q_start"].long()
        n_q = start[1:] - start[:-1]
        tok_seq = torch.repeat_interleave(torch.arange(b, device=dev), n_q, output_size=t)
        tok_i = torch.arange(t, device=dev) - start[tok_seq]
    lim_p = torch.full((t,), p_len, device=dev) if s["prefix_lens"] is None else s["prefix_lens"].long()[tok_seq]
    lim_o = s["lens"].long()[tok_seq] - n_q[tok_seq] + 1 + tok_i

    pages = s["prefix_pages"].long()
    kp, vp = (x[pages].transpose(0, 1).reshape(hk, -1, d)[:, :p_len].float() for x in (s["k"], s["v"]))
    tables = s["tables"].long().clamp(min=0)
    ko, vo = (x[tables].transpose(1, 2).reshape(b, hk, -1, d).float() for x in (s["k"], s["v"]))
    length = ko.shape[2]

    sp = (qf.transpose(0, 1).reshape(hk, t * g, d) @ kp.transpose(1, 2)).view(hk, t, g, p_len).transpose(0, 1)
    sp = sp.masked_fill((torch.arange(p_len, device=dev) >= lim_p[:, None])[:, None, None], -math.inf)
    padded = torch.zeros((b, n, hk, g, d), device=dev)
    padded[tok_seq, tok_i] = qf
    so = (padded.transpose(1, 2).reshape(b, hk, n * g, d) @ ko.transpose(2, 3)).view(b, hk, n, g, length)[tok_seq, :, tok_i]
    so = so.masked_fill((torch.arange(length, device=dev) >= lim_o[:, None])[:, None, None], -math.inf)

    top = torch.maximum(sp.amax(3, keepdim=True), so.amax(3, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    ep, eo = torch.exp(sp - top), torch.exp(so - top)
    total = ep.sum(3, keepdim=True) + eo.sum(3, keepdim=True)
    op = (ep.transpose(0, 1).reshape(hk, t * g, p_len) @ vp).view(hk, t, g, d).transpose(0, 1)
    wide = torch.zeros((b, n, hk, g, length), device=dev)
    wide[tok_seq, tok_i] = eo
    oo = (wide.transpose(1, 2).reshape(b, hk, n * g, length) @ vo).view(b, hk, n, g, d)[tok_seq, :, tok_i]
    return ((op + oo) / torch.where(total > 0, total, 1.0)).to(q.dtype).reshape(t, h, d)


def _plain_append(s):
    """Bias, rotation of the first 2 * half values of each head, and the rows stored where the tables say."""
    c, pos = s["case"], s["pos"].long()
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["bias"] is not None:
        bias = s["bias"].view(-1, c["dim"])
        q, k, v = q + bias[:c["heads"]], k + bias[c["heads"]:c["heads"] + c["kv_heads"]], v + bias[c["heads"] + c["kv_heads"]:]
    cos, sin, rot = s["cos"][pos][:, None], s["sin"][pos][:, None], c["rot"]

    def rotate(x):
        y = x.clone()
        if c["interleaved"]:
            a, z = x[..., 0:rot:2], x[..., 1:rot:2]
            y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - z * sin, a * sin + z * cos
        else:
            a, z = x[..., :rot // 2], x[..., rot // 2:rot]
            y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - z * sin, a * sin + z * cos
        return y

    ct = s["k_pages"].dtype
    page, slot = s["tables"].long()[s["seq"].long(), pos // c["page"]], pos % c["page"]
    s["k_pages"][page, :, slot] = rotate(k).to(ct)
    s["v_pages"][page, :, slot] = v.to(ct)
    return rotate(q).to(ct), s["k_pages"], s["v_pages"]


def _plain_sample(s):
    """Weights 2^32 exp(-(max x - x)) as whole numbers, so that every sum is the same in any order; the filters each keep
    a first part of the tokens in order (smaller max x - x first, then lower index); the token is drawn over the kept
    ones in the order of their indexes."""
    logits, temperature = s["logits"].float(), s["temperature"]
    b, v = logits.shape
    inv = 1.0 / temperature
    greedy = ~(temperature > 0) | (inv == math.inf)
    x = logits * torch.where(greedy, 1.0, inv)[:, None]
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(1, keepdim=True)
    below = torch.where(x == top, 0.0, top - x)
    e = torch.where(x == -math.inf, 0.0, torch.exp(-below))
    w = (e * 2.0 ** 32).long()
    order = torch.sort(below, dim=1, stable=True).indices
    sorted_w, sorted_e = w.gather(1, order), e.gather(1, order)
    before = sorted_w.cumsum(1) - sorted_w
    rank = torch.arange(v, device=x.device)
    keep = torch.ones_like(order, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep &= (k <= 0) | (rank < k)
    if s["top_p"] is not None:
        p = s["top_p"][:, None]
        within = (sorted_w * keep).sum(1, keepdim=True).double() * p.double()
        keep &= ~(p < 1) | (before.double() < within) | (rank == 0)
    if s["min_p"] is not None:
        keep &= sorted_e >= s["min_p"][:, None].clamp(max=1.0)
    keep &= ~greedy[:, None] | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, order, sorted_w * keep)
    sums = w.cumsum(1)
    total = sums[:, -1:]
    r = (s["u"][:, None].double() * total.double()).long().clamp(min=0)
    r = torch.minimum(r, total - 1)
    tokens = torch.searchsorted(sums, r, right=True).clamp(max=v - 1)
    chosen = w.gather(1, tokens)
    empty = total == 0
    probs = torch.where(empty, 0.0, chosen.double() / torch.where(empty, 1, total).double()).float()
    return torch.where(empty, -1, tokens).int()[:, 0], probs[:, 0]


# ----------------------------------------------------------- in 64 bits -----

def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "sample": _exact_sample}[case["op"]](s, case)


def _exact_attention(s, c):
    group, ps = c["heads"] // c["kv_heads"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    rows = lambda pool, pages, n: pool[pages.long()].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :n]  # noqa: E731
    kp, vp = rows(s["k"], s["prefix_pages"], c["prefix"]), rows(s["v"], s["prefix_pages"], c["prefix"])
    t = 0
    for b, (n, ln, p) in enumerate(zip(_query_lens(c), _own_lens(c), _prefix_lens(c))):
        mine = s["tables"][b, :-(-ln // ps)]
        keys = torch.cat([kp[:, :p], rows(s["k"], mine, ln)], 1).repeat_interleave(group, 0)
        vals = torch.cat([vp[:, :p], rows(s["v"], mine, ln)], 1).repeat_interleave(group, 0)
        for i in range(n):
            seen = p + max(0, ln - n + 1 + i)
            if seen:
                score = torch.einsum("hd,hkd->hk", s["q"][t].double(), keys[:, :seen]) * s["scale"]
                out[t] = torch.einsum("hk,hkd->hd", torch.softmax(score, 1), vals[:, :seen])
            t += 1
    return out


def _exact_append(s, c):
    h, hk, d, half = c["heads"], c["kv_heads"], c["dim"], c["rot"] // 2
    x = torch.cat([s["q"], s["k"], s["v"]], 1).double()
    if s["bias"] is not None:
        x = x + s["bias"].double().view(1, -1, d)
    first = torch.arange(half, device="cuda") * 2 if c["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if c["interleaved"] else half)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    z = torch.complex(x[:, :h + hk, first], x[:, :h + hk, second]) * turn
    x[:, :h + hk, first], x[:, :h + hk, second] = z.real, z.imag
    kc, vc = s["k_pages"].double(), s["v_pages"].double()
    flat = s["tables"].long()[s["seq"].long(), s["pos"].long() // c["page"]] * c["page"] + s["pos"].long() % c["page"]
    for pool, new in ((kc, x[:, h:h + hk]), (vc, x[:, h + hk:])):
        by_slot = pool.transpose(1, 2).flatten(0, 1).clone()
        by_slot[flat] = new
        pool.copy_(by_slot.view(pool.shape[0], c["page"], hk, d).transpose(1, 2))
    return x[:, :h].contiguous(), kc, vc


def _exact_sample(s, c):
    tokens, probs = [], []
    for b in range(c["batch"]):
        t = float(s["temperature"][b])
        x = s["logits"][b].float()
        if t > 0:
            x = x * (1.0 / s["temperature"][b])  # the scaled logit and its distance from the largest are 32-bit numbers
        x = torch.where(torch.isnan(x), -math.inf, x)
        if float(x.max()) == -math.inf:
            tokens.append(-1)
            probs.append(0.0)
            continue
        if not t > 0:
            tokens.append(int(torch.nonzero(x == x.max())[0, 0]))
            probs.append(1.0)
            continue
        below = torch.where(x == x.max(), 0.0, x.max() - x)
        e = (-below.double()).exp()
        at = torch.sort(below, stable=True).indices
        w = torch.floor(e[at] * 2.0 ** 32)
        n = c["vocab"]
        k = int(s["top_k"][b]) if s["top_k"] is not None else 0
        n = min(n, k) if k > 0 else n
        p = float(s["top_p"][b]) if s["top_p"] is not None else 1.0
        if p < 1:
            n = min(n, max(1, int((w[:n].cumsum(0) < p * w[:n].sum()).sum()) + 1))
        m = float(s["min_p"][b]) if s["min_p"] is not None else 0.0
        n = min(n, int((e[at] >= min(m, 1.0)).sum()))
        at, back = torch.sort(at[:n])
        w = w[back]
        sums = w.cumsum(0)
        r = math.floor(float(s["u"][b]) * float(sums[-1]))
        i = min(int((sums <= r).sum()), n - 1)
        tokens.append(int(at[i]))
        probs.append(float(w[i] / sums[-1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)
