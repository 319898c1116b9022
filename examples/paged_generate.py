"""Ragged batches on a 4-bit paged cache: prompts of different lengths, then
sampled tokens, a page at a time.

Every layer of a small decoder with synthetic INT4 weights runs on the per-op
front end: RMSNorm and the q/k/v projection, kv4_append (q and k normalised for
each head, rotated, k and v quantised into their pages), attention_kv4 (the same
call for prompts and for single tokens), the output projection, the SwiGLU MLP;
then the lm_head and sample. Sequences join with their whole prompt and go on with
one token a step; a sequence gets a page when it needs one, from a free list.

    python examples/paged_generate.py
"""
from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from aethermind_b200 import _lib as L  # noqa: E402
from aethermind_b200 import ops  # noqa: E402


@dataclass
class Config:
    vocab: int = 2048
    hidden: int = 1024
    layers: int = 4
    n_q: int = 8
    n_kv: int = 2
    head_dim: int = 128
    inter: int = 2816
    theta: float = 500000.0
    max_pos: int = 4096
    page_size: int = 16
    num_pages: int = 256


class Layer:
    def __init__(self, c: Config, i: int):
        rows = (c.n_q + 2 * c.n_kv) * c.head_dim
        scale = 0.02 / 4.61  # uniform codes in [-8, 7] with a standard deviation of 0.02

        def weight(tag, n, k):
            return ops.prepack(L.WFMT_INT4, *ops.synth_w4(11, 16 * i + tag, n, k, scale), n, k)

        self.wqkv = weight(0, rows, c.hidden)
        self.wo = weight(1, c.hidden, c.n_q * c.head_dim)
        gate, up = (ops.synth_w4(11, 16 * i + t, c.inter, c.hidden, scale) for t in (2, 3))
        self.wgu = ops.prepack_gate_up(L.WFMT_INT4, *gate, *up, c.inter, c.hidden)
        self.wd = weight(4, c.hidden, c.inter)
        ones = dict(dtype=torch.bfloat16, device="cuda")
        self.norm1, self.norm2 = torch.ones(c.hidden, **ones), torch.ones(c.hidden, **ones)
        self.q_norm, self.k_norm = torch.ones(c.head_dim, **ones), torch.ones(c.head_dim, **ones)
        self.cache = ops.kv4_cache(c.num_pages, c.page_size, c.n_kv, c.head_dim)


class Decoder:
    def __init__(self, c: Config):
        self.c = c
        self.layers = [Layer(c, i) for i in range(c.layers)]
        self.embed = ops.synth_uniform_bf16(11, 1001, c.vocab * c.hidden, 0.04).view(c.vocab, c.hidden)
        self.lm_head = ops.prepack(L.WFMT_INT4, *ops.synth_w4(11, 1002, c.vocab, c.hidden, 0.02 / 4.61), c.vocab,
                                   c.hidden)
        self.final_norm = torch.ones(c.hidden, dtype=torch.bfloat16, device="cuda")
        self.cos_sin = ops.rope_table(c.theta, c.head_dim, c.max_pos)

    def logits(self, tokens: torch.Tensor, page_table: torch.Tensor, row_start: torch.Tensor,
               ctx_len: torch.Tensor) -> torch.Tensor:
        """Logits of each sequence's last row. tokens [rows]; the other three as kv4_append takes them."""
        c = self.c
        nq, nkv, d = c.n_q, c.n_kv, c.head_dim
        x = ops.embedding(tokens, self.embed)
        for y in self.layers:
            qkv = ops.linear(ops.rmsnorm(x, y.norm1), y.wqkv)
            q, k, v = qkv[:, : nq * d], qkv[:, nq * d: (nq + nkv) * d], qkv[:, (nq + nkv) * d:]
            q = ops.kv4_append(q, k, v, y.cache, page_table, row_start, ctx_len, self.cos_sin, nq, nkv, d,
                               q_norm=y.q_norm, k_norm=y.k_norm)
            a = ops.attention_kv4(q, y.cache, page_table, row_start, ctx_len, nq, nkv, d)
            x = ops.linear(a, y.wo, epilogue=L.EPI_RESIDUAL_ADD, residual=x)
            h = ops.linear(ops.rmsnorm(x, y.norm2), y.wgu, epilogue=L.EPI_SILU_MUL)
            x = ops.linear(h, y.wd, epilogue=L.EPI_RESIDUAL_ADD, residual=x)
        last = x[row_start[1:].long() - 1]
        return ops.linear(ops.rmsnorm(last.contiguous(), self.final_norm), self.lm_head)


def generate(model: Decoder, prompts: list[list[int]], new_tokens: int, temperature: float = 0.8, top_k: int = 40,
             top_p: float = 0.95, seed: int = 0) -> torch.Tensor:
    """Sampled continuations [prompts, new_tokens]; temperature 0 is greedy."""
    c, n = model.c, len(prompts)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    free = list(range(c.num_pages))[::-1]
    lengths = [len(p) for p in prompts]
    pages: list[list[int]] = [[] for _ in prompts]

    def full(v, dtype):
        return torch.full((n,), v, dtype=dtype, device="cuda")

    t, k, p = full(temperature, torch.float32), full(top_k, torch.int32), full(top_p, torch.float32)

    def step(tokens: torch.Tensor, new_rows: list[int]) -> torch.Tensor:
        for have, length in zip(pages, lengths):
            while len(have) * c.page_size < length:
                have.append(free.pop())
        width = max(len(q) for q in pages)
        table = torch.tensor([q + [-1] * (width - len(q)) for q in pages], dtype=torch.int32, device="cuda")
        start = torch.tensor([0] + new_rows, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        ctx = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        logits = model.logits(tokens, table, start, ctx)
        u = torch.rand(n, generator=gen, device="cuda")
        return ops.sample(logits, u, temperature=t, top_k=k, top_p=p)

    flat = torch.tensor([x for q in prompts for x in q], dtype=torch.int64, device="cuda")
    out = [step(flat, lengths[:])]
    for _ in range(new_tokens - 1):
        lengths = [x + 1 for x in lengths]
        out.append(step(out[-1], [1] * n))
    return torch.stack(out, 1)


if __name__ == "__main__":
    torch.manual_seed(0)
    config = Config()
    decoder = Decoder(config)
    asked = [torch.randint(0, config.vocab, (m,)).tolist() for m in (5, 33, 128, 61)]
    for prompt, tokens in zip(asked, generate(decoder, asked, 16).tolist()):
        print(f"{len(prompt):4d} prompt tokens ->", tokens)
