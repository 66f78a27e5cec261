"""The batched decode step over a paged cache (include/tmac_cuda.h, "The batched
decode step"): several sequences, which may share a prefix, advance together.

* ``PagedCache``        -- the k and v pools [n_pages, kv_heads, page_size, head_dim]
* ``rope_table``        -- cos and sin of every position, scaled for long contexts
* ``rope_append``       -- bias, position rotation, k and v stored into the cache
* ``prefix_attention``  -- attention over the shared prefix and the sequences' own keys
* ``sample``            -- temperature, top-k, top-p, min-p and a draw

Tensors are torch CUDA tensors; results are allocated on the stream that is used: the
one given (a torch stream or a raw address), else torch's current stream.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import numpy as np

BF16 = 30  # TMAC_TYPE_BF16

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_INT = ctypes.c_int


class _CacheStruct(ctypes.Structure):
    """tmac_paged_cache"""
    _fields_ = [("k", _P), ("v", _P), ("n_pages", _I64), ("type", _INT), ("kv_heads", _INT), ("page_size", _INT),
                ("head_dim", _INT), ("device", _INT)]


SIGNATURES = {
    "tmac_rope_append": (_INT, [_P, _INT, _P, _I64, _P, _I64, _P, _I64, _INT, _INT, _P, _P, _P, _P, _P, _INT, _INT,
                                _P, _P, _INT, _INT, _INT, _P, _P]),
    "tmac_prefix_attention": (_INT, [_P, _P, _I64, _INT, _INT, _INT, _P, _INT, _P, _INT, _P, _P, _INT, _P, _INT,
                                     ctypes.c_float, _P, _I64, _P, ctypes.c_size_t, _P]),
    "tmac_prefix_attention_workspace": (_INT, [_P, _INT, _INT, _INT, _INT, _INT, _INT, _P]),
    "tmac_sample": (_INT, [_P, _INT, _I64, _INT, _INT, _P, _P, _P, _P, _P, _P, _P, _INT, _P]),
}

_types = None


def _type_of(dtype):
    global _types
    if _types is None:
        import torch
        _types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: BF16}
    return _types.get(dtype, -1)


def _lib():
    import tmac_zynq_fpga_b200 as tm
    return tm.lib()


def _check(rc):
    if rc:
        import tmac_zynq_fpga_b200 as tm
        tm.check(rc)


def _refuse(code, msg):
    import tmac_zynq_fpga_b200 as tm
    raise tm.TmacError(code, msg)


def _stream(stream, device):
    """(context that makes the stream torch's current one, its address)."""
    import torch
    if stream is None:
        return None, torch.cuda.current_stream(device).cuda_stream
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    return torch.cuda.stream(stream), stream.cuda_stream


def _vector(name, t, dtype, shape, device):
    """The address of a contiguous tensor of that type and shape, or of None."""
    if t is None:
        return None
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        _refuse(-1, f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}, "
                    f"not {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _heads(name, t, dim, device):
    """Checks [tokens, heads, head_dim] with adjoining heads; the token stride."""
    if t.dim() != 3 or t.shape[2] != dim:
        _refuse(-3, f"{name} must be [tokens, heads, {dim}], not {tuple(t.shape)}")
    s = t.stride()
    if t.device != device or (s[2] != 1 and dim > 1) or (s[1] != dim and t.shape[1] > 1):
        _refuse(-1, f"{name} must lie on {device} with the heads of a token adjoining")
    return s[0] if t.shape[0] > 1 else t.shape[1] * dim


class PagedCache:
    """The pools of keys and values: two contiguous CUDA tensors [n_pages, kv_heads,
    page_size, head_dim] of one type (float32, float16 or bfloat16); page_size is a
    power of two up to 256.  The tensors stay the caller's: which pages belong to which
    sequence is in the tables given to each call."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape:
            _refuse(-3, f"k and v must both be [n_pages, kv_heads, page_size, head_dim], not {tuple(k.shape)} and {tuple(v.shape)}")
        code = _type_of(k.dtype)
        if code < 0 or v.dtype != k.dtype:
            _refuse(-2, f"k and v must both be float32, float16 or bfloat16, not {k.dtype} and {v.dtype}")
        if not k.is_cuda or v.device != k.device or not k.is_contiguous() or not v.is_contiguous():
            _refuse(-1, "k and v must be contiguous tensors on one CUDA device")
        self.k, self.v, self.dtype, self.device = k, v, k.dtype, k.device
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self._struct = _CacheStruct(k.data_ptr(), v.data_ptr(), self.n_pages, code, self.kv_heads, self.page_size,
                                    self.head_dim, k.device.index)
        self._ref = ctypes.addressof(self._struct)


def rope_table(max_pos, rot_dim, theta=1e6, factor=1.0, original=None, low=1.0, high=32.0, scale=1.0, device="cuda"):
    """cos and sin, float32 [max_pos, rot_dim / 2], of pos * f_i with f_i = theta^(-2i / rot_dim),
    formed in 64 bits (theta 1e6: the reference's, sim/tmac_gguf.cpp:1528-1554).

    For contexts `factor` times longer than the model was trained on: without `original`
    every f_i is divided by `factor` (positions are interpolated); with `original`, the
    trained length, f_i is divided only where a whole turn takes longer than the trained
    length allows: not at all from `high` turns within `original` on, fully below `low`
    turns, linearly in between.  `scale` multiplies cos and sin (an attention temperature
    is its square)."""
    if max_pos <= 0 or rot_dim <= 0 or rot_dim % 2 or not factor > 0 or not theta > 0 or (original is not None and not low < high):
        _refuse(-3, "need max_pos > 0, an even rot_dim > 0, theta and factor > 0 and low < high")
    import torch
    f = theta ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    if original is None:
        f = f / factor
    else:
        whole = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)  # 1: as it was
        f = f * (whole + (1 - whole) / factor)
    angle = np.arange(max_pos, dtype=np.float64)[:, None] * f
    return tuple(torch.from_numpy((fn(angle) * scale).astype(np.float32)).to(device) for fn in (np.cos, np.sin))


def rope_append(cache, q, k, v, pos, tables, cos, sin, *, seq=None, starts=None, interleaved=True, bias=None, q_out=None,
                stream=None):
    """Adds the bias, turns q and k by their positions, stores k and v into the cache's pages
    and returns q in the cache's type, [tokens, heads, head_dim].

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], of one type, with any
    distance between tokens; pos, seq int32 [tokens]; tables int32 [n_seq, width]; starts
    int32 [n_seq]; cos, sin float32 [max_pos, rot_dim / 2] (`rope_table`); bias float32
    [(heads + 2 kv_heads) * head_dim].  See tmac_rope_append for the places they name."""
    import torch
    dev, dim = cache.device, cache.head_dim
    code = _type_of(q.dtype)
    if code < 0 or k.dtype != q.dtype or v.dtype != q.dtype:
        _refuse(-2, "q, k and v must be of one type: float32, float16 or bfloat16")
    qs, ks, vs = _heads("q", q, dim, dev), _heads("k", k, dim, dev), _heads("v", v, dim, dev)
    n, heads = q.shape[0], q.shape[1]
    if k.shape != v.shape or k.shape[0] != n or k.shape[1] != cache.kv_heads:
        _refuse(-3, f"k and v must be [{n}, {cache.kv_heads}, {dim}], not {tuple(k.shape)} and {tuple(v.shape)}")
    if tables.dim() != 2 or cos.dim() != 2:
        _refuse(-3, "tables must be [n_seq, width] and cos [max_pos, rot_dim / 2]")
    i32, f32 = torch.int32, torch.float32
    n_seq, width = tables.shape
    args = (_vector("bias", bias, f32, ((heads + 2 * cache.kv_heads) * dim,), dev), _vector("seq", seq, i32, (n,), dev),
            _vector("pos", pos, i32, (n,), dev), _vector("starts", starts, i32, (n_seq,), dev),
            _vector("tables", tables, i32, tables.shape, dev), n_seq, width, _vector("cos", cos, f32, cos.shape, dev),
            _vector("sin", sin, f32, cos.shape, dev), cos.shape[0], 2 * cos.shape[1], 1 if interleaved else 0)
    ctx, s = _stream(stream, dev)
    with ctx or contextlib.nullcontext():
        if q_out is None:
            q_out = torch.empty((n, heads, dim), dtype=cache.dtype, device=dev)
        _check(_lib().tmac_rope_append(cache._ref, code, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, heads, n,
                                       *args, _vector("q_out", q_out, cache.dtype, (n, heads, dim), dev), s))
    return q_out


def prefix_attention(q, cache, tables, own_lens, *, prefix_pages=None, prefix_len=0, prefix_lens=None, q_start=None, max_q=1,
                     max_own=None, scale=None, out=None, stream=None):
    """Attention of every query token over the shared prefix and its sequence's own keys, the
    prefix read once for the whole batch: [tokens, heads, head_dim] of q's type (the cache's).

    tables int32 [batch, width] and own_lens int32 [batch]: the pages and number of each
    sequence's own keys, the queries' among them (max_own: a bound on the lengths, by
    default what the tables hold); prefix_pages int32, prefix_len: the shared positions;
    prefix_lens int32 [batch]: how much of them each sequence sees (all).  q_start int32
    [batch + 1] with max_q: several query tokens per sequence, each seeing the keys up to
    its own; without it one per sequence.  See tmac_prefix_attention."""
    import torch
    dev, dim = cache.device, cache.head_dim
    if q.dtype != cache.dtype:
        _refuse(-2, f"q must have the cache's type {cache.dtype}, not {q.dtype}")
    qs = _heads("q", q, dim, dev)
    n, heads = q.shape[0], q.shape[1]
    if tables.dim() != 2:
        _refuse(-3, "tables must be [batch, width]")
    batch, width = tables.shape
    if max_own is None:
        max_own = width * cache.page_size
    if prefix_pages is not None and prefix_len > prefix_pages.numel() * cache.page_size:
        _refuse(-3, "prefix_pages do not cover prefix_len")
    i32 = torch.int32
    own = _vector("own_lens", own_lens, i32, (batch,), dev)
    table = _vector("tables", tables, i32, tables.shape, dev)
    pages = None if prefix_pages is None else _vector("prefix_pages", prefix_pages, i32, (prefix_pages.numel(),), dev)
    shared = _vector("prefix_lens", prefix_lens, i32, (batch,), dev)
    starts = _vector("q_start", q_start, i32, (batch + 1,), dev)
    L = _lib()
    need = ctypes.c_size_t()
    _check(L.tmac_prefix_attention_workspace(cache._ref, heads, n, batch, max_q, prefix_len, max_own, ctypes.addressof(need)))
    ctx, s = _stream(stream, dev)
    with ctx or contextlib.nullcontext():
        if out is None:
            out = torch.empty((n, heads, dim), dtype=q.dtype, device=dev)
        elif out.dtype != q.dtype or out.shape != q.shape:
            _refuse(-1, "out must have q's type and shape")
        work = torch.empty(need.value, dtype=torch.uint8, device=dev)
        _check(L.tmac_prefix_attention(cache._ref, q.data_ptr(), qs, heads, n, batch, starts, max_q, pages, prefix_len,
                                       shared, table, width, own, max_own, dim ** -0.5 if scale is None else scale,
                                       out.data_ptr(), _heads("out", out, dim, dev), work.data_ptr(), need.value, s))
    return out


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
    """The next token of each row of logits [batch, vocab] (float32, float16 or bfloat16, any
    distance between rows) and its probability among the kept tokens: int32 [batch],
    float32 [batch].  u float32 [batch] in [0, 1); temperature, top_p, min_p float32
    [batch], top_k int32 [batch], each optional.  See tmac_sample for the filters."""
    import torch
    code = _type_of(logits.dtype)
    if code < 0:
        _refuse(-2, f"logits must be float32, float16 or bfloat16, not {logits.dtype}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _refuse(-3, "logits must be [batch, vocab] with adjoining values")
    if not logits.is_cuda:
        _refuse(-1, "logits must lie on a CUDA device")
    dev, (n, vocab) = logits.device, logits.shape
    f32, shape = torch.float32, (n,)
    args = (_vector("u", u, f32, shape, dev), _vector("temperature", temperature, f32, shape, dev),
            _vector("top_k", top_k, torch.int32, shape, dev), _vector("top_p", top_p, f32, shape, dev),
            _vector("min_p", min_p, f32, shape, dev))
    ctx, s = _stream(stream, dev)
    with ctx or contextlib.nullcontext():
        tokens = torch.empty(n, dtype=torch.int32, device=dev)
        probs = torch.empty(n, dtype=f32, device=dev)
        _check(_lib().tmac_sample(logits.data_ptr(), code, logits.stride(0) if n > 1 else vocab, n, vocab, *args,
                                  tokens.data_ptr(), probs.data_ptr(), dev.index, s))
    return tokens, probs
