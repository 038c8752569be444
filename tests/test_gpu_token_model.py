"""The token operators together: the example's model learns its rule, and one
of its steps agrees with the same step in plain numpy."""

from __future__ import annotations

import os
import sys

import numpy as np
import pytest
from conftest import ROOT
from helpers import dev, host

sys.path.insert(0, os.path.join(ROOT, "examples"))
import token_model as E  # noqa: E402

import nanotorch_amd as nt  # noqa: E402

pytestmark = pytest.mark.gpu


def test_example_learns(gpu, capsys):
    losses = E.main(["--steps", "300", "--vocabulary", "32", "--seed", "3"])
    # from about log 32 = 3.47 towards the rule's entropy, below 0.7
    assert losses[0] > 3.0
    assert np.mean(losses[-20:]) < 1.2
    assert "where the rule gives" in capsys.readouterr().out


def test_answers_repeat_and_dropout_rests(gpu):
    nt.manual_seed(1)
    model = E.TokenModel(16, 8, 32, 0.5)
    assert E.ask(model, [[1, 2], [3, 4]]) == E.ask(model, [[1, 2], [3, 4]])


def test_a_step_against_numpy(gpu):
    """Without dropout; sums of at most 64 terms of size about 1 in float32:
    each gradient within 64 x 2^-24 x 16 of its own largest value."""
    nt.manual_seed(2)
    r = np.random.default_rng(2)
    V, D, H, B = 13, 6, 10, 40
    model = E.TokenModel(V, D, H, 0.0)
    W, W1, b1, W2, b2 = [host(p).astype(np.float64) for p in model.parameters()]
    c, t = r.integers(0, V, (B, 2)), r.integers(0, V, B)
    out = nt.token_logprobs(model(dev(c)), dev(t), entropy=True)
    (out.logprob.mean() * -1.0 - out.entropy.mean() * 0.5).backward()

    e = W[c] * (c != E.PADDING)[:, :, None]
    x = e.reshape(B, 2 * D)
    h = np.tanh(x @ W1 + b1)
    z = h @ W2 + b2
    logp = z - z.max(1, keepdims=True)
    logp -= np.log(np.exp(logp).sum(1, keepdims=True))
    p = np.exp(logp)
    ent = -(p * logp).sum(1)
    assert np.abs(host(out.logprob) - logp[np.arange(B), t]).max() < 64 * 2.0 ** -24 * 16
    dz = p.copy()
    dz[np.arange(B), t] -= 1
    dz = (dz + 0.5 * p * (logp + ent[:, None])) / B
    dh = dz @ W2.T * (1 - h * h)
    dx = (dh @ W1.T).reshape(B, 2, D) * (c != E.PADDING)[:, :, None]
    dW = np.zeros_like(W)
    np.add.at(dW, c, dx)
    for got, want in zip(model.parameters(), (dW, x.T @ dh, dh.sum(0), h.T @ dz, dz.sum(0))):
        err = np.abs(host(got.grad) - want).max()
        assert err < 64 * 2.0 ** -24 * 16 * max(np.abs(want).max(), 2.0 ** -6), err
    assert (host(model.parameters()[0].grad)[E.PADDING] == 0).all()
