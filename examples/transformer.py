"""A small causal transformer over token numbers, trained with AdamW and asked one
token at a time over a cache of keys and values.

    python examples/transformer.py --steps 300

Each block is a norm, attention, a norm and a two-layer network; the norms add the
residual.  The text is synthetic: a sequence of random tokens, then the same again,
so that the second half can be told from the first by attention alone.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import nanotorch_amd as nt  # noqa: E402
from nanotorch_amd import nn  # noqa: E402

IGNORED = -100  # what nothing is to be learnt of


class Block(nn.Module):
    def __init__(self, dim: int, heads: int, kv_heads: int, hidden: int) -> None:
        self.norms = [nn.RMSNorm(dim), nn.RMSNorm(dim)]
        self.attention = nn.Attention(dim, heads, kv_heads)
        self.net = nn.Sequential(nn.Linear(dim, hidden), nn.ReLU(), nn.Linear(hidden, dim))

    def parameters(self):
        return [p for m in (*self.norms, self.attention, self.net) for p in m.parameters()]

    def forward(self, x, residual, lengths=None, cache=None):
        """The block's output and the residual that the next norm adds to it."""
        y, residual = self.norms[0](x, residual)
        y, residual = self.norms[1](self.attention(y, lengths, cache), residual)
        B, T, dim = y.shape
        return self.net(y.reshape(B * T, dim)).reshape(B, T, dim), residual


class Transformer(nn.Module):
    """Logits [B, T, vocabulary] of the tokens after those of [B, T]."""

    def __init__(self, vocabulary: int, dim: int, heads: int, kv_heads: int, hidden: int,
                 blocks: int, max_tokens: int) -> None:
        self.tokens = nn.Embedding(vocabulary, dim)
        self.places = nn.Embedding(max_tokens, dim)
        self.blocks = [Block(dim, heads, kv_heads, hidden) for _ in range(blocks)]
        self.norm = nn.RMSNorm(dim)
        self.head = nn.Linear(dim, vocabulary)

    def parameters(self):
        modules = (self.tokens, self.places, *self.blocks, self.norm, self.head)
        return [p for m in modules for p in m.parameters()]

    def caches(self, sequences: int, max_tokens: int):
        return [b.attention.cache(sequences, max_tokens) for b in self.blocks]

    def forward(self, tokens: nt.Tensor, lengths=None, caches=None) -> nt.Tensor:
        B, T = tokens.shape
        first = caches[0].tokens if caches else 0
        places = np.broadcast_to(np.arange(first, first + T), (B, T))
        x, residual = self.tokens(tokens), self.places(nt.Tensor(places, device="cuda"))
        for i, block in enumerate(self.blocks):
            x, residual = block(x, residual, lengths, caches[i] if caches else None)
        y, _ = self.norm(x, residual)
        dim = y.shape[2]
        return self.head(y.reshape(B * T, dim)).reshape(B, T, self.head.parameters()[0].shape[1])


def texts(rng: np.random.Generator, batch: int, half: int, vocabulary: int):
    """Tokens [batch, 2 half] of which the second half repeats the first, cut at
    lengths of their own (padded with 0), the tokens that follow, and the lengths."""
    first = rng.integers(0, vocabulary, (batch, half))
    tokens = np.concatenate([first, first], 1)
    following = np.full_like(tokens, IGNORED)
    following[:, half - 1:-1] = tokens[:, half:]
    lengths = rng.integers(half + 1, 2 * half + 1, batch)
    for b, n in enumerate(lengths):
        tokens[b, n:], following[b, n - 1:] = 0, IGNORED
    return tokens, following, lengths


def loss_of(model: Transformer, tokens, following, lengths) -> nt.Tensor:
    """The mean -log p of the tokens that follow."""
    kept = max(1, int((following != IGNORED).sum()))
    out = nt.token_logprobs(model(nt.Tensor(tokens, device="cuda"),
                                  nt.Tensor(lengths, device="cuda")),
                            nt.Tensor(following, device="cuda"), ignore_index=IGNORED)
    return out.logprob.sum() * (-1.0 / kept)


def train(model: Transformer, steps: int, batch: int, half: int, vocabulary: int, lr: float,
          rng: np.random.Generator) -> list[float]:
    optimizer = nn.AdamW(model.parameters(), lr)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad()
        loss = loss_of(model, *texts(rng, batch, half, vocabulary))
        loss.backward()
        optimizer.step()
        losses.append(float(loss.cpu().item()))
    return losses


def answer(model: Transformer, prompts: np.ndarray, count: int) -> np.ndarray:
    """The most likely `count` tokens after each of the prompts [B, T], one by one."""
    caches = model.caches(len(prompts), prompts.shape[1] + count)
    told, tokens = [], prompts
    with nt.no_grad():
        for _ in range(count):
            logits = model(nt.Tensor(tokens, device="cuda"), caches=caches)[:, -1]
            tokens = nt.token_logprobs(logits, top=1).top_tokens.numpy()
            told.append(tokens)
    return np.concatenate(told, 1)


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=600)
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--half", type=int, default=12)
    ap.add_argument("--vocabulary", type=int, default=16)
    ap.add_argument("--dim", type=int, default=64)
    ap.add_argument("--heads", type=int, default=4)
    ap.add_argument("--kv-heads", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=128)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(a.seed)
    nt.manual_seed(a.seed)
    model = Transformer(a.vocabulary, a.dim, a.heads, a.kv_heads, a.hidden, a.blocks, 2 * a.half)
    losses = train(model, a.steps, a.batch, a.half, a.vocabulary, a.lr, rng)
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {i}: loss {losses[i]:.4f}", flush=True)
    print(f"last step: loss {losses[-1]:.4f}")
    first = rng.integers(0, a.vocabulary, (2, a.half))
    for prompt, told in zip(first, answer(model, np.concatenate([first, first[:, :2]], 1),
                                          a.half - 2)):
        print(f"after {prompt.tolist()} and its first two: {told.tolist()}")
    return losses


if __name__ == "__main__":
    main()
