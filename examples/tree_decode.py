"""Speculative decoding with trees of drafted tokens over a quantised cache.

A small random transformer decodes several sequences at once, greedily.  Their
common prompt goes through the model once and the other sequences get copies of
its cache rows.  A step drafts a tree behind each sequence's last token, runs all
nodes of all trees through the model together, accepts the branch that the model
itself would have taken, and closes its cache rows up.  The tokens are those that
one token at a time gives; a step yields more than one of them.

    python examples/tree_decode.py --sequences 4 --tokens 64 [--f16]
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from prana_b200 import kernels as K  # noqa: E402

CHAIN = 64  # a prompt is taken this many tokens at a time, as a tree without branches


class Transformer:
    """Random weights.  The embedding's own successors (see `drafts`) outweigh what
    attention adds, so that drafts are often right."""

    def __init__(self, vocab=512, layers=2, heads=8, kv_heads=2, head_dim=64, seed=1, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        width = heads * head_dim

        def weight(rows, cols, scale=1.0):
            return torch.randn(rows, cols, generator=g, device=device) * (scale / cols**0.5)

        self.heads, self.kv_heads, self.head_dim, self.device = heads, kv_heads, head_dim, device
        self.embed = torch.randn(vocab, width, generator=g, device=device)
        self.head = weight(vocab, width)
        self.layers = [(weight(width + 2 * kv_heads * head_dim, width), weight(width, width, 0.5)) for _ in range(layers)]
        self.waves = torch.exp(torch.arange(width // 2, device=device) * (-8.0 / width))
        self.ones = torch.ones(width, device=device)

    def norm(self, x: torch.Tensor) -> torch.Tensor:
        width = x.shape[-1]
        return K.rmsnorm(x, self.ones, x.numel() // width, width, 1e-5)

    def caches(self, positions: int, quantized: bool) -> list[K.KvRows]:
        return [K.KvRows.alloc(positions, self.kv_heads, self.head_dim, quantized, self.device) for _ in self.layers]

    def drafts(self, tokens: torch.Tensor, n: int) -> torch.Tensor:
        """The n likeliest successors of each token by the embedding alone."""
        return (self.norm(self.embed[tokens]) @ self.head.t()).topk(n, dim=-1).indices

    def forward(self, caches, tokens, places, starts, lens, offsets, max_nodes, rows, masks=None) -> torch.Tensor:
        """Logits of all nodes; their K and V go to the cache rows `rows`."""
        angle = places[:, None] * self.waves
        x = self.embed[tokens] + 0.3 * torch.cat((angle.sin(), angle.cos()), dim=1)
        q_width, kv_width = self.heads * self.head_dim, self.kv_heads * self.head_dim
        for cache, (qkv, out) in zip(caches, self.layers):
            q, k, v = (self.norm(x) @ qkv.t()).split((q_width, kv_width, kv_width), dim=1)
            K.kv_rows_write(cache, rows, k, v)
            x = x + K.attention_tree(q.contiguous(), cache, starts, lens, offsets, max_nodes, self.heads, masks) @ out.t()
        return self.norm(x) @ self.head.t()


class Decoder:
    def __init__(self, model: Transformer, sequences: int, room: int, quantized: bool):
        self.model, self.n, self.room = model, sequences, room
        self.caches = model.caches(sequences * room, quantized)
        self.starts = self._ints([b * room for b in range(sequences)])
        self.lens = [0] * sequences

    def _ints(self, x, dtype=torch.int32) -> torch.Tensor:
        return torch.tensor(x, dtype=dtype, device=self.model.device)

    def prompt(self, tokens: list[int]) -> list[int]:
        """The prompt into every sequence's rows; its first successor for each."""
        m, logits = self.model, None
        for at in range(0, len(tokens), CHAIN):
            part = tokens[at : at + CHAIN]
            n = len(part)
            logits = m.forward(self.caches, self._ints(part), self._ints(range(at, at + n)), self._ints([0]), self._ints([at]),
                               self._ints([0, n]), n, self._ints(range(at, at + n)))
        # the other sequences' rows: read back and written again, which quantises to the same integers
        rows = self._ints(range(len(tokens)))
        for cache in self.caches:
            k, v = K.kv_rows_read(cache, rows)
            for b in range(1, self.n):
                K.kv_rows_write(cache, rows + b * self.room, k, v)
        self.lens = [len(tokens)] * self.n
        return [int(K.argmax(logits[-1:]))] * self.n

    def step(self, last: list[int], branches: tuple[int, ...]) -> list[list[int]]:
        """One pass: `last` tokens are the trees' roots, branches[d] the children of each
        node of depth d.  Returns each sequence's new tokens."""
        m = self.model
        parents, depth, level = [-1], [0], [0]
        for d, width in enumerate(branches):
            level = [self._grow(parents, depth, p, d + 1) for p in level for _ in range(width)]
        nodes = len(parents)
        # all sequences' trees have one shape; their tokens level by level
        tokens = self._ints(last, torch.int64)[:, None]
        front = tokens
        for width in branches:
            front = m.drafts(front, width).flatten(1)
            tokens = torch.cat((tokens, front), dim=1)
        lens, place = self._ints(self.lens), self._ints(depth)
        rows = (self.starts + lens)[:, None] + torch.arange(nodes, dtype=torch.int32, device=m.device)
        masks = self._ints(K.tree_masks(parents) * self.n, torch.int64)
        logits = m.forward(self.caches, tokens.flatten(), (lens[:, None] + place).flatten(), self.starts, lens,
                           self._ints(range(0, (self.n + 1) * nodes, nodes)), nodes, rows.flatten(), masks)
        best, drafted = K.argmax(logits).view(self.n, nodes).tolist(), tokens.tolist()

        taken, path = [], []
        for b in range(self.n):
            at, branch = 0, [0]
            while True:
                child = [i for i in range(nodes) if parents[i] == at and drafted[b][i] == best[b][at]]
                if not child:
                    break
                at = child[0]
                branch.append(at)
            taken.append([best[b][i] for i in branch])
            path.append(branch + [0] * (len(branches) + 1 - len(branch)))
        counts = [len(t) for t in taken]
        for cache in self.caches:
            K.kv_rows_move(cache, self.starts, lens, self._ints(path), self._ints(counts))
        self.lens = [n + c for n, c in zip(self.lens, counts)]
        return taken

    @staticmethod
    def _grow(parents: list[int], depth: list[int], parent: int, d: int) -> int:
        parents.append(parent)
        depth.append(d)
        return len(parents) - 1


def generate(model: Transformer, prompt: list[int], sequences: int, tokens: int, quantized: bool = True,
             branches: tuple[int, ...] = (3, 2, 1)) -> tuple[list[list[int]], int]:
    """`tokens` tokens for each sequence, and the passes that took.  Sequence b starts
    from the prompt's successor plus b, so that the sequences differ."""
    # a sequence may be ahead of the others by a whole branch at every step
    room = len(prompt) + (tokens + 1) * (len(branches) + 1) + K.TREE_MAX_NODES
    d = Decoder(model, sequences, room, quantized)
    text = [[(t + b) % len(model.embed)] for b, t in enumerate(d.prompt(prompt))]
    steps = 0
    while min(len(t) for t in text) < tokens:
        for t, new in zip(text, d.step([t[-1] for t in text], branches)):
            t += new
        steps += 1
    torch.cuda.synchronize()
    return [t[:tokens] for t in text], steps


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--sequences", type=int, default=4)
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--prompt", type=int, default=100)
    p.add_argument("--f16", action="store_true", help="an f16 cache instead of int8")
    a = p.parse_args()
    model = Transformer()
    prompt = [(7 * i * i + 3) % len(model.embed) for i in range(a.prompt)]
    for name, branches in (("one token at a time", ()), ("trees of 16 nodes", (3, 2, 1))):
        generate(model, prompt, a.sequences, 8, not a.f16, branches)  # warm-up
        t0 = time.perf_counter()
        text, steps = generate(model, prompt, a.sequences, a.tokens, not a.f16, branches)
        ms = (time.perf_counter() - t0) * 1e3
        print(f"{name}: {a.sequences} x {a.tokens} tokens in {steps} steps, {ms:.1f} ms; the first begins {text[0][:8]}")


if __name__ == "__main__":
    main()
