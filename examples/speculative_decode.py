"""Speculative decoding over the quantised latent cache, on a one-layer toy model.

    python examples/speculative_decode.py [--steps 8] [--batch 4] [--tree 12]

Every step drafts a tree of candidate tokens per sequence, writes their latent rows behind
the cached context (``ops.cache_write``), attends from the whole tree at once
(``ops.tree_attn``), verifies the candidates against the model's probabilities
(``ops.verify_draft``) and writes the accepted path where the context continues; at the
end ``ops.cache_read`` gives the cached context as dense rows.  The
queries and latents come from ``ops.proj_rope``.  Weights are random: what it shows is how
the operators fit together, not text.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from kernelswift_b200 import ops  # noqa: E402


class ToyModel:
    """Embedding -> latent attention (16 heads of 192 columns, 64 of them rotary) -> logits,
    to which a token's own embedding adds a guess at its successor."""

    def __init__(self, vocab=512, dim=256, heads=16, latent=128, rope=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s, scale: (torch.randn(*s, device="cuda", generator=g) * scale).bfloat16()  # noqa: E731
        self.vocab, self.heads, self.latent, self.rope, self.width = vocab, heads, latent, rope, latent + rope
        self.embed = rnd(vocab, dim, scale=1.0)
        self.wq = rnd(heads * self.width, dim, scale=dim ** -0.5)
        self.wkv = rnd(self.width, dim, scale=dim ** -0.5)
        self.wo = rnd(vocab, heads * latent, scale=(heads * latent) ** -0.5)
        self.next = rnd(vocab, dim, scale=3.0 * dim ** -0.5)
        self.sink = torch.zeros(heads, device="cuda")
        self.inv = 10000.0 ** (-torch.arange(0, rope, 2, device="cuda").float() / rope)

    def freqs(self, pos: torch.Tensor) -> torch.Tensor:
        ang = pos.reshape(-1, 1).float() * self.inv
        return torch.stack([ang.cos(), ang.sin()], -1).contiguous()

    def queries_and_latents(self, tokens: torch.Tensor, pos: torch.Tensor):
        """tokens, pos [B, T] -> q [B, T, H, D], latent rows [B, T, D], both rotated at pos."""
        x, fr = self.embed[tokens].reshape(tokens.numel(), -1).contiguous(), self.freqs(pos)
        q = ops.proj_rope(x, self.wq, self.width, self.rope, fr)
        kv = ops.proj_rope(x, self.wkv, self.width, self.rope, fr)
        return q.view(*tokens.shape, self.heads, self.width), kv.view(*tokens.shape, self.width)

    def guess(self, tokens: torch.Tensor) -> torch.Tensor:
        """The logits' part that needs no context, tokens [...] -> [..., vocab]."""
        return self.embed[tokens].float() @ self.next.float().T

    def probabilities(self, attended: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
        """[B, T, H, latent], tokens [B, T] -> [B, T, vocab]."""
        return torch.softmax(attended.flatten(2).float() @ self.wo.float().T + self.guess(tokens), -1)


class Cache:
    """Paged e4m3 cache with a page table per sequence."""

    def __init__(self, model: ToyModel, batch: int, longest: int, page: int = 32):
        each = -(-longest // page)
        self.page, self.lens = page, torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.table = torch.randperm(batch * each, device="cuda").view(batch, each).int().contiguous()
        self.kv8 = torch.zeros(batch * each, page, model.latent, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        self.scale = torch.zeros(batch * each, page, device="cuda")
        self.tail = torch.zeros(batch * each, page, model.rope, dtype=torch.bfloat16, device="cuda")

    def write(self, kv: torch.Tensor, pos: torch.Tensor, keep: torch.Tensor | None = None) -> None:
        """Rows [B, T, D] at positions pos [B, T] of their sequences, where `keep`."""
        pages = self.table.long().gather(1, (pos // self.page).clamp_max(self.table.shape[1] - 1))
        slots = pages * self.page + pos % self.page
        if keep is not None:
            slots = torch.where(keep, slots, -1)
        ops.cache_write(kv, slots, self.kv8, self.scale, self.tail)

    def attend(self, q: torch.Tensor, model: ToyModel, mask: torch.Tensor | None = None) -> torch.Tensor:
        return ops.tree_attn(q, self.kv8, self.scale, self.tail, self.table, self.lens, model.width ** -0.5,
                             dv=model.latent, mask=mask, attn_sink=model.sink)

    def rows(self) -> torch.Tensor:
        """The cached rows as dense bf16 [B, longest, D], zero past a sequence's length: what
        a prefill over a shared prefix reads."""
        return ops.cache_read(self.kv8, self.scale, self.tail, self.table, self.lens, int(self.lens.max()))


def tree(parents: torch.Tensor):
    """Depth and ancestor mask (each node itself included) of parents [T] (-1: the root)."""
    t = len(parents)
    mask, depth = torch.eye(t, dtype=torch.bool), torch.zeros(t, dtype=torch.long)
    for i, p in enumerate(parents.tolist()):
        if p >= 0:
            mask[i] |= mask[p]
            depth[i] = depth[p] + 1
    return depth.cuda(), mask.cuda()


def draft(model: ToyModel, last: torch.Tensor, parents: torch.Tensor) -> torch.Tensor:
    """Candidates [B, T]: a node's children are the likeliest successors of its token by the
    model's guess without context, the best first."""
    tokens = torch.empty(len(last), len(parents), dtype=torch.int64, device="cuda")
    used: dict[int, int] = {}
    for i, p in enumerate(parents.tolist()):
        k = used[p] = used.get(p, -1) + 1
        tokens[:, i] = model.guess(last if p < 0 else tokens[:, p]).topk(k + 1, -1).indices[:, k]
    return tokens


def prefill(model: ToyModel, cache: Cache, prompt: torch.Tensor) -> torch.Tensor:
    """Caches all but the last prompt token, which the first step processes."""
    pos = torch.arange(prompt.shape[1], device="cuda").expand_as(prompt)
    cache.write(model.queries_and_latents(prompt, pos)[1][:, :-1].contiguous(), pos[:, :-1].contiguous())
    cache.lens += prompt.shape[1] - 1
    return prompt[:, -1]


def step(model: ToyModel, cache: Cache, last: torch.Tensor, parents: torch.Tensor, g: torch.Generator):
    """One speculative step.  `last` [B] is the newest token, not cached yet; `parents`
    the shape of the tree drafted after it.  Returns (new tokens [B, T + 1], -1 where none,
    how many drafts stood [B])."""
    b, t = len(last), len(parents)
    # the newest token is the root of what is processed; the drafted tree hangs below it
    depth, mask = tree(torch.cat([torch.tensor([-1]), parents + 1]))
    drafted = draft(model, last, parents)
    tokens = torch.cat([last[:, None], drafted], 1)
    lens = cache.lens.long()[:, None]
    q, kv = model.queries_and_latents(tokens, lens + depth)      # rotated at the depth's position
    cache.write(kv, lens + torch.arange(t + 1, device="cuda"))   # stored one after the other
    p = model.probabilities(cache.attend(q, model, mask.expand(b, -1, -1).contiguous()), tokens)
    u = torch.rand(b, t + 1, device="cuda", generator=g)
    noise = torch.empty(b, model.vocab, device="cuda").exponential_(generator=g).clamp_min_(1e-10)
    new, stood, path = ops.verify_draft(p, drafted, u, noise,
                                        parents=parents.int().cuda().expand(b, -1).contiguous())
    # the accepted path moves up to follow the newest token: rows are written again from kv
    at = torch.arange(t, device="cuda").expand(b, -1)
    rows = kv.gather(1, (path.long().clamp_min(0) + 1)[..., None].expand(-1, -1, kv.shape[-1]))
    cache.write(rows, lens + 1 + at, keep=path >= 0)
    cache.lens += 1 + stood
    return new, stood


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--tree", type=int, default=12)
    a = ap.parse_args()
    model, g = ToyModel(), torch.Generator(device="cuda").manual_seed(1)
    cache = Cache(model, a.batch, 64 + (a.steps + 1) * (a.tree + 2))
    prompt = torch.randint(0, model.vocab, (a.batch, 64), device="cuda", generator=g)
    last = prefill(model, cache, prompt)
    parents = torch.tensor([(i - 1) // 2 for i in range(a.tree)])  # a heap: two children each
    parents[: min(2, a.tree)] = -1
    for i in range(a.steps):
        new, stood = step(model, cache, last, parents, g)
        last = new.gather(1, stood.long()[:, None])[:, 0]
        print(f"step {i}: accepted {stood.tolist()} of {a.tree} drafted, newest tokens {last.tolist()}")
    dense = cache.rows()
    print(f"cached {cache.lens.tolist()} tokens: {tuple(dense.shape)} rows, largest {dense.abs().max().item():.2f}")
    ops.device_status()


if __name__ == "__main__":
    main()
