"""The batched decode step over a paged cache (include/tmac_cuda.h, "The batched
decode step"): several sequences, which may share a prefix, advance together.

* ``PagedCache``        -- the k and v pools [n_pages, kv_heads, page_size, head_dim]
* ``rope_table``        -- cos and sin of every position, scaled for long contexts
* ``rope_append``       -- bias, position rotation, k and v stored into the cache
* ``prefix_attention``  -- attention over the shared prefix and the sequences' own keys
* ``sample``            -- temperature, top-k, top-p, min-p and a draw

Tensors are torch CUDA tensors; results are allocated on the stream that is used: the
one given (a torch stream or a raw address), else torch's current stream.  Arguments may
be dropped once the call has returned; what was queued on another stream must be waited
for by the one that is used.  There are no gradients: a tensor that requires one is refused
where gradients are enabled.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

BF16 = 30  # TMAC_TYPE_BF16

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_INT = ctypes.c_int


class PagedCacheStruct(ctypes.Structure):
    """tmac_paged_cache"""
    _fields_ = [("k", _P), ("v", _P), ("n_pages", _I64), ("type", _INT), ("kv_heads", _INT), ("page_size", _INT),
                ("head_dim", _INT), ("device", _INT)]


SIGNATURES = {
    "tmac_rope_append": (_INT, [_P, _INT, _P, _I64, _P, _I64, _P, _I64, _INT, _INT, _P, _P, _P, _P, _P, _INT, _INT,
                                _P, _P, _INT, _INT, _INT, _P, _P]),
    "tmac_prefix_attention": (_INT, [_P, _P, _I64, _INT, _INT, _INT, _P, _INT, _P, _INT, _P, _P, _INT, _P, _INT,
                                     ctypes.c_float, _P, _I64, _P, ctypes.c_size_t, _P]),
    "tmac_prefix_attention_workspace": (_INT, [_P, _INT, _INT, _INT, _INT, _INT, _INT, _P]),
    "tmac_prefix_attention_engine": (_INT, [_P, _INT, _INT, _INT, _INT, _INT, _INT]),
    "tmac_sample": (_INT, [_P, _INT, _I64, _INT, _INT, _P, _P, _P, _P, _P, _P, _P, _INT, _P]),
}

_native = None


def _ext():
    """The module that checks tensors and calls the library (host/serving_binding.cpp)."""
    global _native
    if _native is None:
        import torch  # noqa: F401  (the module needs its libraries loaded)

        import tmac_zynq_fpga_b200 as tm
        tm.lib()
        try:
            from . import _serving
        except ImportError as e:
            raise tm.TmacError(-1, f"_serving.so, which buildlib.build() compiles against torch, is missing or of another torch: {e}") from e
        _serving.set_error_class(tm.TmacError)
        _native = _serving
    return _native


def _refuse(code, msg):
    import tmac_zynq_fpga_b200 as tm
    raise tm.TmacError(code, msg)


def _on(stream, device, *tensors):
    """The context in which `stream`, a torch stream or an address, is torch's current one.
    The memory of `tensors` (None among them) is not reused before the stream has read it."""
    import torch
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            t.record_stream(stream)
    return torch.cuda.stream(stream)


class PagedCache:
    """The pools of keys and values: two contiguous CUDA tensors [n_pages, kv_heads,
    page_size, head_dim] of one type (float32, float16 or bfloat16); page_size is a
    power of two up to 256.  The tensors stay the caller's: which pages belong to which
    sequence is in the tables given to each call."""

    __slots__ = ("k", "v")

    def __init__(self, k, v):
        (_native or _ext()).check_cache(k, v)
        self.k, self.v = k, v


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
    if stream is not None:
        with _on(stream, cache.k.device, cache.k, cache.v, q, k, v, pos, tables, cos, sin, seq, starts, bias, q_out):
            return rope_append(cache, q, k, v, pos, tables, cos, sin, seq=seq, starts=starts, interleaved=interleaved, bias=bias,
                               q_out=q_out)
    return (_native or _ext()).rope_append(cache.k, cache.v, q, k, v, pos, tables, cos, sin, seq, starts, interleaved, bias, q_out)


def prefix_attention(q, cache, tables, own_lens, *, prefix_pages=None, prefix_len=0, prefix_lens=None, q_start=None, max_q=1,
                     max_own=None, scale=None, out=None, stream=None):
    """Attention of every query token over the shared prefix and its sequence's own keys, the
    prefix read once for the whole batch: [tokens, heads, head_dim] of q's type (the cache's).

    tables int32 [batch, width] and own_lens int32 [batch]: the pages and number of each
    sequence's own keys, the queries' among them (max_own: a bound on the lengths, by
    default what the tables hold); prefix_pages int32, prefix_len: the shared positions;
    prefix_lens int32 [batch]: how much of them each sequence sees (all).  q_start int32
    [batch + 1] with max_q: several query tokens per sequence, each seeing the keys up to
    its own, and zeros for tokens of no sequence; without it one per sequence.  See
    tmac_prefix_attention."""
    if stream is not None:
        with _on(stream, cache.k.device, q, cache.k, cache.v, tables, own_lens, prefix_pages, prefix_lens, q_start, out):
            return prefix_attention(q, cache, tables, own_lens, prefix_pages=prefix_pages, prefix_len=prefix_len,
                                    prefix_lens=prefix_lens, q_start=q_start, max_q=max_q, max_own=max_own, scale=scale, out=out)
    return (_native or _ext()).prefix_attention(q, cache.k, cache.v, tables, own_lens, prefix_pages, prefix_len, prefix_lens, q_start,
                                                max_q, max_own, scale, out)


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
    """The next token of each row of logits [batch, vocab] (float32, float16 or bfloat16, any
    distance between rows) and its probability among the kept tokens: int32 [batch],
    float32 [batch].  u float32 [batch] in [0, 1); temperature, top_p, min_p float32
    [batch], top_k int32 [batch], each optional.  See tmac_sample for the filters."""
    if stream is not None:
        with _on(stream, logits.device, logits, u, temperature, top_k, top_p, min_p):
            return sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    return (_native or _ext()).sample(logits, u, temperature, top_k, top_p, min_p)
