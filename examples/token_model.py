"""A small token model, trained and asked: the embedding of the last tokens,
dropout, a two-layer network and the log probability of the next token.

    python examples/token_model.py --steps 200

The text is synthetic: each token follows from the two before it, except that
one in ten is drawn at random, so the loss falls towards the entropy of that
rule and the most likely alternative is the rule's token.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import nanotorch_amd as nt  # noqa: E402
from nanotorch_amd import nn  # noqa: E402

PADDING = 0  # the token before a text begins: no row of its own is trained


def rule(a, b, vocabulary: int):
    return 1 + (3 * a + 5 * b + 7) % (vocabulary - 1)


def text(rng: np.random.Generator, length: int, vocabulary: int) -> np.ndarray:
    out = np.zeros(length + 2, np.int64)  # two PADDING tokens first
    for i in range(2, length + 2):
        noise = rng.random() < 0.1
        out[i] = rng.integers(1, vocabulary) if noise else rule(out[i - 2], out[i - 1],
                                                                vocabulary)
    return out


class TokenModel(nn.Module):
    """Logits [batch, vocabulary] of the token after two given ones."""

    def __init__(self, vocabulary: int, dim: int, hidden: int, dropout: float) -> None:
        self.tokens = nn.Embedding(vocabulary, dim, padding_idx=PADDING)
        self.head = nn.Sequential(nn.Dropout(dropout), nn.Linear(2 * dim, hidden), nn.Tanh(),
                                  nn.Linear(hidden, vocabulary))

    def parameters(self):
        return [*self.tokens.parameters(), *self.head.parameters()]

    def forward(self, context: nt.Tensor) -> nt.Tensor:
        x = self.tokens(context)  # [batch, 2, dim]
        return self.head(x.reshape(x.shape[0], x.shape[1] * x.shape[2]))


def train(model: TokenModel, words: np.ndarray, steps: int, batch: int, lr: float,
          rng: np.random.Generator, entropy_bonus: float = 0.01) -> list[float]:
    """The mean loss -log p of each step's next tokens."""
    optimizer = nn.GradientDescent(model.parameters(), lr)
    model.train()
    losses = []
    for _ in range(steps):
        at = rng.integers(0, len(words) - 2, batch)
        context = nt.Tensor(np.stack([words[at], words[at + 1]], 1), device="cuda")
        following = nt.Tensor(words[at + 2], device="cuda")
        optimizer.zero_grad()
        out = nt.token_logprobs(model(context), following, entropy=True)
        nll = out.logprob.mean() * -1.0
        (nll - out.entropy.mean() * entropy_bonus).backward()
        optimizer.step()
        losses.append(float(nll.cpu().item()))
    return losses


def ask(model: TokenModel, contexts: list[list[int]], top: int = 3):
    """(entropy, [(token, log probability), ...]) for each context."""
    model.eval()
    with nt.no_grad():
        out = nt.token_logprobs(model(nt.Tensor(np.array(contexts), device="cuda")),
                                entropy=True, top=top)
    return [(float(h), [(int(t), float(p)) for t, p in zip(ts, ps)])
            for h, ts, ps in zip(out.entropy.numpy(), out.top_tokens.numpy(),
                                 out.top_logprobs.numpy())]


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=1000)
    ap.add_argument("--batch", type=int, default=512)
    ap.add_argument("--vocabulary", type=int, default=32)
    ap.add_argument("--dim", type=int, default=64)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--dropout", type=float, default=0.1)
    ap.add_argument("--lr", type=float, default=0.5)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    rng = np.random.default_rng(a.seed)
    nt.manual_seed(a.seed)
    words = text(rng, 20000, a.vocabulary)
    model = TokenModel(a.vocabulary, a.dim, a.hidden, a.dropout)
    losses = train(model, words, a.steps, a.batch, a.lr, rng)
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {i}: loss {losses[i]:.4f}", flush=True)
    print(f"last step: loss {losses[-1]:.4f}")
    for at in (100, 200, 300):
        context = [int(w) for w in words[at:at + 2]]
        entropy, best = ask(model, [context])[0]
        told = ", ".join(f"{t} ({p:.2f})" for t, p in best)
        print(f"after {context}, where the rule gives {rule(*context, a.vocabulary)}: "
              f"{told}; entropy {entropy:.2f}")
    return losses


if __name__ == "__main__":
    main()
