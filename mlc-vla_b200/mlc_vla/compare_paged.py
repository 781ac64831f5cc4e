"""Text generation over the paged 8-bit cache against dense attention.

A small stack of Gemma-style attention layers (RMS norm, grouped heads, RoPE, residual; random
weights, tied embeddings) answers a batch of prompts of different lengths greedily, the way a
serving loop would: ``build_slots`` places the new tokens, ``attention_prompt`` runs the packed
prompts (a bidirectional prefix of image tokens, causal text), ``write_kv`` puts keys and values
into the pages, and then every step places, writes and attends (``attention_paged``) one token per
request. The same tokens run through dense fp32 attention on unquantised keys and values; the
hidden states must agree (cosine >= 0.9999 for the prompts, >= 0.995 for the steps, whose keys and
values are held in 8 bits).

    python -m mlc_vla.compare_paged [--dtype float16|bfloat16] [--steps N] [--requests N]
"""

from __future__ import annotations

import argparse
from typing import List, NamedTuple

import numpy as np
import torch

from mlc_vla import paged
from mlc_vla._compare import cosine
from mlc_vla.model.pi0.pi0_config import GemmaExpertConfig
from mlc_vla.runtime import embed_language
from mlc_vla.sample import make_rope_np


class Layer(NamedTuple):
    qkv: torch.Tensor  # [(heads + 2 kv heads) * head_dim, width]
    out: torch.Tensor  # [width, heads * head_dim]


class Stack:
    """Attention layers of one Gemma expert's shape, with random weights, for tokens at the first
    ``positions`` positions."""

    def __init__(self, cfg: GemmaExpertConfig, layers: int, vocab: int, dtype, seed: int, device="cuda",
                 positions: int = 4096):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(rows, cols):
            x = torch.randn((rows, cols), generator=g, device=device) / np.sqrt(cols)
            return x.to(dtype)

        self.cfg, self.dtype, self.device = cfg, dtype, device
        self.table = (0.05 * torch.randn((vocab, cfg.width), generator=g, device=device)).to(dtype)
        rows = (cfg.num_heads + 2 * cfg.num_kv_heads) * cfg.head_dim
        self.layers = [Layer(w(rows, cfg.width), w(cfg.width, cfg.num_heads * cfg.head_dim))
                       for _ in range(layers)]
        cos, sin = make_rope_np(positions, cfg.head_dim, 10_000.0)
        self.rope = [torch.as_tensor(np.asarray(x).reshape(positions, -1)).to(device) for x in (cos, sin)]

    def project(self, layer: Layer, x: torch.Tensor, positions: torch.Tensor):
        """q, k and v of tokens at these positions: views of one projection, q and k rotated."""
        c = self.cfg
        n = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)
        qkv = (n.to(self.dtype) @ layer.qkv.T).view(len(x), -1, c.head_dim)
        cos, sin = (t[positions.long()][:, None] for t in self.rope)
        turned = qkv[:, :c.num_heads + c.num_kv_heads]
        a, b = turned.float().chunk(2, -1)
        turned.copy_(torch.cat((a * cos - b * sin, b * cos + a * sin), -1))
        return qkv.split([c.num_heads, c.num_kv_heads, c.num_kv_heads], 1)

    def add(self, layer: Layer, x: torch.Tensor, attended: torch.Tensor) -> torch.Tensor:
        return x + attended.reshape(len(x), -1) @ layer.out.T

    def next_tokens(self, hidden: torch.Tensor) -> torch.Tensor:
        return (hidden.float() @ self.table.float().T).argmax(-1).int()


class PagedSession:
    """Requests that answer together: their block table, free pages and one cache per layer."""

    def __init__(self, stack: Stack, batch: int, most: int, page: int = 64):
        c = stack.cfg
        if most > len(stack.rope[0]):
            raise ValueError(f"requests of {most} tokens, a stack for {len(stack.rope[0])} positions")
        self.stack, self.page, self.most, self.longest = stack, page, most, 0
        columns = -(-most // page)
        pages = batch * columns
        ints = dict(dtype=torch.int32, device=stack.device)
        self.table = torch.full((batch, columns), -1, **ints)
        self.free, self.pos = torch.randperm(pages, device=stack.device).int(), torch.zeros(1, **ints)
        self.lens = torch.zeros(batch, **ints)
        self.caches = [paged.KVCache8.empty(pages, page, c.num_kv_heads, c.head_dim, stack.device)
                       for _ in stack.layers]

    def _place(self, new: torch.Tensor, tokens: int, longest: int) -> paged.Slots:
        """``longest``: the most new tokens of one request. Positions stay inside the stack's table."""
        if self.longest + longest > self.most:
            raise ValueError(f"a request may grow beyond the session's {self.most} tokens")
        self.longest += longest
        return paged.build_slots(self.lens, new, self.table, self.free, self.pos, self.page, tokens)

    def prompts(self, x: torch.Tensor, new: torch.Tensor, prefix: torch.Tensor, longest: int):
        """Packed prompt embeddings [tokens, width] -> hidden states."""
        s = self._place(new, len(x), longest)
        for layer, cache in zip(self.stack.layers, self.caches):
            q, k, v = self.stack.project(layer, x, s.positions)
            x = self.stack.add(layer, x, paged.attention_prompt(q, k, v, s.cu_seqlens,
                                                                prefix_lens=prefix))
            paged.write_kv(cache, k, v, s.cu_seqlens, self.lens, s.slot_mapping, max_new=longest)
        self.lens, self.pos = s.kv_lens, s.free_pos
        return x

    def step(self, x: torch.Tensor):
        """One token per request, embeddings [batch, width] -> hidden states."""
        s = self._place(torch.ones_like(self.lens), len(x), 1)
        for layer, cache in zip(self.stack.layers, self.caches):
            q, k, v = self.stack.project(layer, x, s.positions)
            paged.write_kv(cache, k, v, s.cu_seqlens, self.lens, s.slot_mapping, max_new=1)
            x = self.stack.add(layer, x, paged.attention_paged(q, cache, self.table, s.kv_lens))
        self.lens, self.pos = s.kv_lens, s.free_pos
        return x


def dense(stack: Stack, x: torch.Tensor, prefix: int) -> torch.Tensor:
    """One request from its first token on, dense fp32 attention on unquantised keys and values."""
    n, c = len(x), stack.cfg
    i = torch.arange(n, device=x.device)
    seen = (i[None] <= i[:, None]) | (i[None] < prefix)
    for layer in stack.layers:
        q, k, v = (t.float().transpose(0, 1) for t in stack.project(layer, x, i))
        k, v = (t.repeat_interleave(c.num_heads // c.num_kv_heads, 0) for t in (k, v))
        p = torch.softmax((q @ k.transpose(1, 2) * c.head_dim ** -0.5).masked_fill(~seen, -torch.inf), -1)
        x = stack.add(layer, x, (p @ v).transpose(0, 1).to(x.dtype))
    return x


def run(cfg: GemmaExpertConfig, dtype: str = "float16", lens: List[int] = (70, 33, 129, 1),
        images: int = 32, steps: int = 12, layers: int = 2, vocab: int = 1000, seed: int = 0) -> bool:
    lens = list(lens)
    stack = Stack(cfg, layers, vocab, getattr(torch, dtype), seed, positions=max(lens) + steps)
    rng = np.random.default_rng(seed)
    prefix = [min(images, n) for n in lens]
    prompt = [torch.as_tensor(rng.integers(0, vocab, n).astype(np.int32)).cuda() for n in lens]
    ints = dict(dtype=torch.int32, device="cuda")
    session = PagedSession(stack, len(lens), max(lens) + steps)
    embed = [embed_language(stack.table, t) for t in prompt]
    hidden = session.prompts(torch.cat(embed), torch.tensor(lens, **ints), torch.tensor(prefix, **ints),
                             max(lens))
    ends = np.cumsum(lens)
    outs = [[hidden[e - n:e]] for e, n in zip(ends, lens)]
    ids = stack.next_tokens(hidden[torch.as_tensor(ends - 1).cuda()])
    for _ in range(steps):
        x = embed_language(stack.table, ids)
        embed = [torch.cat((e, x[r:r + 1])) for r, e in enumerate(embed)]
        hidden = session.step(x)
        ids = stack.next_tokens(hidden)
        for r in range(len(lens)):
            outs[r].append(hidden[r:r + 1])
    paged.check()
    worst = [1.0, 1.0]
    for r, n in enumerate(lens):
        want = dense(stack, embed[r], prefix[r]).float().cpu().numpy()
        got = torch.cat(outs[r]).float().cpu().numpy()
        worst = [min(worst[0], cosine(got[:n], want[:n])),
                 min([worst[1]] + [cosine(got[i], want[i]) for i in range(n, n + steps)])]
    ok = worst[0] >= 0.9999 and worst[1] >= 0.995
    print(f"[compare_paged] prompts {lens}, {steps} steps: cosine prompts {worst[0]:.6f} "
          f"steps {worst[1]:.6f} {'PASS' if ok else 'FAIL'}")
    return ok


def main():
    ap = argparse.ArgumentParser(description="paged text generation against dense attention")
    ap.add_argument("--dtype", default="float16", choices=["float16", "bfloat16"])
    ap.add_argument("--variant", default="gemma_2b", help="expert shape (heads, widths)")
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=12)
    args = ap.parse_args()
    rng = np.random.default_rng(0)
    lens = [int(n) for n in rng.integers(700, 969, args.requests)]
    ok = run(GemmaExpertConfig.from_variant(args.variant), args.dtype, lens, images=768,
             steps=args.steps)
    raise SystemExit(0 if ok else 1)


if __name__ == "__main__":
    main()
