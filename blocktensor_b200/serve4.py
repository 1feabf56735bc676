"""A small decoder that serves sequences from paged 4-bit caches: the serving operators
(serving.py) between the int8 products and norms of the rest of the package.

Per layer and step: RMSNorm, the fused q/k/v product, head norms + rotation + cache append in one
launch, attention over the 4-bit cache (with an optional sliding window and sinks), the output
product, RMSNorm, SwiGLU; after the last layer the head product and one batched draw.  Weights are
random (seeded); there is no checkpoint.

    python -m blocktensor_b200.serve4 --steps 32 --window 64 --sinks 4
"""
from __future__ import annotations

import argparse
from dataclasses import dataclass
from typing import Sequence

import torch

import blocktensor_b200 as bt


@dataclass
class Shape:
    vocab: int = 4096
    dim: int = 512
    hidden: int = 1024
    layers: int = 4
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    theta: float = 10000.0
    eps: float = 1e-5


class Matrix:
    """A Q8_0 matrix [M, K] in the tensor-core tile layout."""

    def __init__(self, w):
        self.M, self.K = w.shape
        self.blocks = bt.quantize_q8_0(w.reshape(-1).contiguous())
        self.units = bt.pack_q8_units(self.blocks, self.M, self.K)

    def __call__(self, x):
        return bt.gemm_q8_units(self.units, x, self.M, self.K)


class Decoder4:
    """``slots`` sequences of up to ``max_seq`` positions, K/V in ``n_pages`` pages of ``page_tokens``
    positions a layer.  Every layer's cache shares the first one's page table."""

    def __init__(self, shape: Shape, slots: int, max_seq: int, page_tokens: int = 64, n_pages: int = 0, window: int = 0,
                 sinks: int = 0, seed: int = 0):
        s = self.shape = shape
        self.window, self.sinks = window, sinks
        g = torch.Generator("cuda").manual_seed(seed)

        def normal(*size, std):
            return torch.randn(*size, generator=g, device="cuda") * std

        width = (s.heads + 2 * s.kv_heads) * s.head_dim
        self.embed = normal(s.vocab, s.dim, std=1.0)
        self.layers = []
        for _ in range(s.layers):
            self.layers.append(dict(
                attn_norm=1 + normal(s.dim, std=0.1), ffn_norm=1 + normal(s.dim, std=0.1),
                q_norm=1 + normal(s.head_dim, std=0.1), k_norm=1 + normal(s.head_dim, std=0.1),
                qkv=Matrix(normal(width, s.dim, std=s.dim ** -0.5)), o=Matrix(normal(s.dim, s.heads * s.head_dim, std=s.dim ** -0.5)),
                up=Matrix(normal(2 * s.hidden, s.dim, std=s.dim ** -0.5)), down=Matrix(normal(s.dim, s.hidden, std=s.hidden ** -0.5))))
        self.out_norm = 1 + normal(s.dim, std=0.1)
        self.head = Matrix(normal(s.vocab, s.dim, std=2 * s.dim ** -0.5))
        self.rope = bt.rope_table(max_seq, s.head_dim, s.theta)
        n_pages = n_pages or slots * -(-max_seq // page_tokens)
        self.caches = [bt.KV4Cache(slots, max_seq, s.kv_heads, s.head_dim, page_tokens, n_pages)]
        for _ in range(1, s.layers):
            self.caches.append(bt.KV4Cache(slots, max_seq, s.kv_heads, s.head_dim, page_tokens, n_pages,
                                           page_table=self.caches[0].page_table))
        self.lens = [0] * slots                                     # cached positions of every slot
        self.next = torch.zeros(slots, dtype=torch.int32, device="cuda")  # each slot's next token

    def forward(self, tokens, slots: Sequence[int], counts: Sequence[int]):
        """Logits [sum(counts), vocab] of ``counts[i]`` more tokens of each slot, which enter its caches."""
        s = self.shape
        if len(set(slots)) != len(slots) or len(counts) != len(slots) or min(counts, default=0) < 1 or len(tokens) != sum(counts):
            raise ValueError("forward: expected different slots, and one token or more for each")
        for slot, c in zip(slots, counts):
            self.caches[0].reserve(slot, self.lens[slot] + c)
        positions = [self.lens[slot] + j for slot, c in zip(slots, counts) for j in range(c)]
        for slot, c in zip(slots, counts):
            self.lens[slot] += c

        def device(v):
            return torch.tensor(v, dtype=torch.int32, device="cuda")

        pos, lens, at = device(positions), device([self.lens[i] for i in slots]), device(list(slots))
        token_slots = device([slot for slot, c in zip(slots, counts) for _ in range(c)])
        starts = None
        if any(c != 1 for c in counts):
            starts = device([0] + torch.tensor(counts).cumsum(0).tolist())
        x = self.embed[tokens.long()]
        n = x.shape[0]
        for w, cache in zip(self.layers, self.caches):
            h = w["qkv"](bt.rmsnorm(x, w["attn_norm"], n, s.dim, s.eps)).view(n, -1, s.head_dim)
            q, k, v = h.split([s.heads, s.kv_heads, s.kv_heads], 1)
            q = cache.append_normed(q, k, v, w["q_norm"], w["k_norm"], token_slots, pos, self.rope, s.eps)
            a = cache.attention(q, lens, q_start=starts, slots=at, max_q=max(counts), window=self.window, sinks=self.sinks)
            x = x + w["o"](a.view(n, -1))
            gate, up = w["up"](bt.rmsnorm(x, w["ffn_norm"], n, s.dim, s.eps)).chunk(2, 1)
            x = x + w["down"](bt.silu(gate.contiguous()) * up)
        return self.head(bt.rmsnorm(x, self.out_norm, n, s.dim, s.eps))

    def prefill(self, prompts: Sequence[Sequence[int]], slots: Sequence[int], u, **sampling):
        """Starts a sequence in each slot; returns its first drawn token."""
        counts = [len(p) for p in prompts]
        tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
        logits = self.forward(tokens, slots, counts)
        last = torch.tensor(counts, device="cuda").cumsum(0) - 1
        return self._draw(logits[last], slots, u, sampling)

    def step(self, slots: Sequence[int], u, **sampling):
        """One token more for each slot."""
        return self._draw(self.forward(self.next[list(slots)], slots, [1] * len(slots)), slots, u, sampling)

    def _draw(self, logits, slots, u, sampling):
        token, _ = bt.sample_batch(logits, u, **sampling)
        self.next[list(slots)] = token
        return token

    def release(self, slot: int):
        self.caches[0].release(slot)
        self.lens[slot] = 0

    def check(self):
        for c in self.caches:
            c.check()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--slots", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=40)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    model = Decoder4(Shape(), a.slots, 1024, window=a.window, sinks=a.sinks, seed=a.seed)
    g = torch.Generator("cuda").manual_seed(a.seed + 1)
    slots = list(range(a.slots))
    prompts = [torch.randint(0, model.shape.vocab, (20 + 37 * i,), generator=g, device="cuda").tolist() for i in slots]

    def sampling():
        def f(v):
            return torch.full((a.slots,), v, device="cuda")
        return dict(u=torch.rand(a.slots, generator=g, device="cuda"), temperature=f(a.temperature),
                    top_k=torch.full((a.slots,), a.top_k, dtype=torch.int32, device="cuda"), top_p=f(a.top_p), min_p=f(a.min_p))

    out = [model.prefill(prompts, slots, **sampling())]
    for _ in range(a.steps - 1):
        out.append(model.step(slots, **sampling()))
    model.check()
    for i, row in enumerate(torch.stack(out, 1).tolist()):
        print(f"slot {i} ({len(prompts[i])} prompt tokens): {row}")


if __name__ == "__main__":
    main()
