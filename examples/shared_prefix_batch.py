"""Several answers to one prompt, decoded together.

The prompt is computed once and its keys and values stay in shared pages; every answer
then has pages of its own, and a step of the whole batch runs, per layer,

    q, k, v products -> rope_append -> prefix_attention -> output and FFN products

and ends with one draw per answer (sample).  The projections are the library's quantised
products (Weight.gemv), the weights a synthetic model in the `.tmac` format.

    python examples/shared_prefix_batch.py --answers 8 --prompt 40 --steps 16 --top-k 40
"""
import argparse
import os
import sys
import time

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import torch  # noqa: E402

import tmac_zynq_fpga_b200 as tm  # noqa: E402
from tmac_zynq_fpga_b200 import model  # noqa: E402

H, KV, D = model.HEADS, model.KV_HEADS, model.HEAD_DIM


class SharedPrefixBatch:
    """`answers` sequences over one prompt; cache_type: the elements of the paged cache."""

    def __init__(self, path, answers, max_prompt, max_steps, cache_type=torch.float32, page=16, device=0):
        dev = torch.device("cuda", device)
        tensors = model.read_tmac(path)
        vec = lambda n: torch.from_numpy(tensors[n][3].view(np.float32).copy()).to(dev)  # noqa: E731
        mat = lambda n: tm.Weight(tensors[n][2], tensors[n][0], tensors[n][1], tensors[n][3], device=device)  # noqa: E731
        self.dev, self.answers, self.page, self.prompt = dev, answers, page, 0
        self.embedding, self.out_norm = tensors["token_embd.weight"], vec("output_norm.weight")
        self.logits = mat("token_embd.weight")
        self.layers = []
        for i in range(model.LAYERS):
            p = f"blk.{i}."
            self.layers.append(dict(
                norm=vec(p + "attn_norm.weight"), ffn_norm=vec(p + "ffn_norm.weight"),
                bias=torch.cat([vec(p + f"attn_{x}.bias") for x in "qkv"]),
                **{x: mat(p + f"{x}.weight") for x in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down")}))
        # pages: the prompt's, then each answer's
        shared, each = -(-max_prompt // page), -(-max_steps // page)
        pool = (shared + answers * each, KV, page, D)
        self.caches = [tm.PagedCache(torch.zeros(pool, dtype=cache_type, device=dev), torch.zeros(pool, dtype=cache_type, device=dev))
                       for _ in self.layers]
        self.prefix_pages = torch.arange(shared, dtype=torch.int32, device=dev)
        self.tables = torch.arange(shared, pool[0], dtype=torch.int32, device=dev).view(answers, each)
        self.cos, self.sin = tm.rope_table(max_prompt + max_steps, D, device=dev)
        self.lens = torch.zeros(answers, dtype=torch.int32, device=dev)  # own keys

    def _embed(self, tokens):
        rows, cols, _, raw = self.embedding
        blocks = raw.reshape(rows, -1, 34)[np.asarray(tokens)]  # Q8_0: an fp16 factor and 32 bytes
        d = blocks[..., :2].copy().view(np.float16).astype(np.float32)
        return torch.from_numpy((d * blocks[..., 2:].view(np.int8)).reshape(len(blocks), cols)).to(self.dev)

    def _product(self, weight, x):
        y = torch.empty((len(x), weight.rows), device=self.dev)
        weight.gemv(x.contiguous(), y, batch=len(x), stream=torch.cuda.current_stream(self.dev))
        return y

    @staticmethod
    def _norm(x, w):
        return x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + 1e-6) * w

    def _forward(self, tokens, pos, tables, starts, seq, attend):
        x = self._embed(tokens)
        for layer, cache in zip(self.layers, self.caches):
            h = self._norm(x, layer["norm"])
            q, k, v = (self._product(layer[n], h).unflatten(1, (-1, D)) for n in ("attn_q", "attn_k", "attn_v"))
            q = tm.rope_append(cache, q, k, v, pos, tables, self.cos, self.sin, seq=seq, starts=starts, bias=layer["bias"])
            x = x + self._product(layer["attn_output"], attend(q, cache).flatten(1).float())
            h = self._norm(x, layer["ffn_norm"])
            gate, up = self._product(layer["ffn_gate"], h), self._product(layer["ffn_up"], h)
            x = x + self._product(layer["ffn_down"], gate * torch.sigmoid(gate) * up)
        return x

    def _logits(self, x):
        return self._product(self.logits, self._norm(x, self.out_norm))

    def start(self, prompt):
        """Computes the prompt once; the logits of its last position, for every answer."""
        n = self.prompt = len(prompt)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)  # noqa: E731
        pos, seq, table = torch.arange(n, dtype=torch.int32, device=self.dev), ints([0] * n), self.prefix_pages[None]
        lens, q_start = ints([n]), ints([0, n])
        x = self._forward(prompt, pos, table, None, seq,
                          lambda q, cache: tm.prefix_attention(q, cache, table, lens, q_start=q_start, max_q=n))
        self.lens.zero_()
        self.starts = torch.full((self.answers,), n, dtype=torch.int32, device=self.dev)
        return self._logits(x[-1:]).expand(self.answers, -1)

    def step(self, tokens):
        """One token of every answer; the logits after it."""
        pos = self.starts + self.lens
        self.lens += 1
        x = self._forward(tokens, pos, self.tables, self.starts, None,
                          lambda q, cache: tm.prefix_attention(q, cache, self.tables, self.lens, prefix_pages=self.prefix_pages,
                                                               prefix_len=self.prompt))
        return self._logits(x)


def generate(batch, prompt, steps, seed=0, **filters):
    """int tokens [steps, answers], drawn with uniform numbers of `seed` under `filters` (see sample)."""
    g = torch.Generator(device=batch.dev).manual_seed(seed)
    logits, out = batch.start(prompt), []
    for i in range(steps):
        tokens, _ = tm.sample(logits, torch.rand(batch.answers, generator=g, device=batch.dev), **filters)
        out.append(tokens.cpu().numpy())
        if i + 1 < steps:
            logits = batch.step(out[-1])
    return np.stack(out)


def main():
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--answers", type=int, default=8)
    a.add_argument("--prompt", type=int, default=40, help="tokens of the (random) prompt")
    a.add_argument("--steps", type=int, default=16)
    a.add_argument("--cache", choices=("f32", "f16", "bf16"), default="f32")
    a.add_argument("--temperature", type=float, default=0.8)
    a.add_argument("--top-k", type=int, default=40)
    a.add_argument("--top-p", type=float, default=0.95)
    a.add_argument("--min-p", type=float, default=0.0)
    a = a.parse_args()
    types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    batch = SharedPrefixBatch(model.default_model_path(0), a.answers, a.prompt, a.steps, types[a.cache])
    row = lambda v, t: torch.full((a.answers,), v, dtype=t, device=batch.dev)  # noqa: E731
    filters = dict(temperature=row(a.temperature, torch.float32), top_k=row(a.top_k, torch.int32),
                   top_p=row(a.top_p, torch.float32), min_p=row(a.min_p, torch.float32))
    prompt = model.prompt_tokens(a.prompt)
    generate(batch, prompt, 2, **filters)  # first use of every kernel
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens = generate(batch, prompt, a.steps, **filters)
    ms = (time.perf_counter() - t0) * 1e3
    assert tm.device_error(0) == 0
    for i in range(a.answers):
        print(f"answer {i}:", *tokens[:, i])
    print(f"{a.prompt} prompt tokens and {a.steps} x {a.answers} answer tokens in {ms:.1f} ms")


if __name__ == "__main__":
    main()
