"""The transformer's operators together: the example runs, its gradients are those
of differences, answers over a cache are those without one, and one step of all of
them agrees with the same step in plain numpy."""

from __future__ import annotations

import os
import sys

import numpy as np
import pytest
from conftest import ROOT
from helpers import dev, host

sys.path.insert(0, os.path.join(ROOT, "examples"))
import transformer as E  # noqa: E402

import nanotorch_amd as nt  # noqa: E402
from nanotorch_amd import nn  # noqa: E402

pytestmark = pytest.mark.gpu


def small(seed=0, **kw):
    nt.manual_seed(seed)
    return E.Transformer(**{**dict(vocabulary=11, dim=24, heads=4, kv_heads=2, hidden=20,
                                   blocks=2, max_tokens=16), **kw})


def test_example_runs(gpu, capsys):
    losses = E.main(["--steps", "5", "--batch", "8"])
    assert len(losses) == 5 and np.isfinite(losses).all()
    assert "and its first two" in capsys.readouterr().out


def test_gradients_against_differences(gpu):
    """In float64 (Linear takes the product and the sum apart there): a central
    difference over 2 h of a loss near 2.4, evaluated to 2^-50 of itself, is off
    by 2.4 2^-50 / h = 2e-9 and by h^2 times a third derivative of at most 1e3."""
    model = small()
    for m in (model.tokens, model.places, model.norm, model.head,
              *[x for b in model.blocks for x in (*b.norms, *b.net._modules[::2],
                                                  b.attention._q, b.attention._k,
                                                  b.attention._v, b.attention._out)]):
        for name in ("_W", "_w", "_b"):
            if getattr(m, name, None) is not None:
                p = getattr(m, name).to(nt.float64)
                p.enable_grad()
                setattr(m, name, p)
    rng = np.random.default_rng(1)
    batch = E.texts(rng, 3, 5, 11)
    E.loss_of(model, *batch).backward()
    h = 1e-6
    for p in model.parameters():
        g = host(p.grad).reshape(-1)
        value = host(p)
        for at in (int(np.abs(g).argmax()), int(rng.integers(g.size))):
            losses = []
            for sign in (1, -1):
                moved = value.copy().reshape(-1)
                moved[at] += sign * h
                with nt.no_grad():
                    p[...] = dev(moved.reshape(value.shape))
                    losses.append(float(E.loss_of(model, *batch).cpu().item()))
                    p[...] = dev(value)
            slope = (losses[0] - losses[1]) / (2 * h)
            assert abs(slope - g[at]) < 2e-9 + 1e3 * h * h + 1e-7 * abs(g[at]), (
                p.shape, at, slope, g[at])


def test_answers_over_a_cache(gpu):
    """Token by token and prompt at once give the logits of the whole text.  Both
    sum the same terms (at most 24 in a product) in other orders: 24 x 2^-24 of
    values below 8, through two blocks that amplify it less than 64 times."""
    model = small(3, max_tokens=17)
    tokens = np.random.default_rng(2).integers(0, 11, (3, 14))
    with nt.no_grad():
        whole = host(model(dev(tokens)))
        caches, parts = model.caches(3, 16), []
        for beg, end in ((0, 6), (6, 7), (7, 8), (8, 13), (13, 14)):
            parts.append(host(model(dev(tokens[:, beg:end]), caches=caches)))
    assert caches[0].tokens == 14
    tol = 24 * 2.0 ** -24 * 8 * 64
    assert np.abs(np.concatenate(parts, 1) - whole).max() < tol
    with nt.no_grad(), pytest.raises(ValueError):
        model(dev(tokens[:, :3]), caches=caches)  # 16 tokens cannot hold 17
    with pytest.raises(RuntimeError):
        model(dev(tokens[:, :1]), caches=caches)  # no gradients through a cache


def test_padding_does_not_matter(gpu):
    model = small(4)
    rng = np.random.default_rng(5)
    tokens, following, lengths = E.texts(rng, 4, 6, 11)
    E.loss_of(model, tokens, following, lengths).backward()
    first = [host(p.grad) for p in model.parameters()]
    for p in model.parameters():
        p.zero_grad()
    for b, n in enumerate(lengths):
        tokens[b, n:] = rng.integers(0, 11, 12 - n)
    E.loss_of(model, tokens, following, lengths).backward()
    # (the tables' rows of the padding's tokens get zeros: sums of the same terms)
    for a, p in zip(first, model.parameters()):
        assert np.abs(a - host(p.grad)).max() <= 64 * 2.0 ** -24 * max(np.abs(a).max(), 1e-3)


def test_a_block_and_a_step_against_numpy(gpu):
    """Norm with residual, attention over grouped heads, their gradients and one
    AdamW step.  Sums of at most 40 terms in float32, values about 1: gradients
    within 40 x 2^-24 x 64 of their largest, parameters within that of the step."""
    rng = np.random.default_rng(7)
    B, T, dim, H, Hk = 2, 10, 16, 4, 2
    D = dim // H
    nt.manual_seed(7)
    norm, att = nn.RMSNorm(dim), nn.Attention(dim, H, Hk)
    x, res, G = [rng.standard_normal((B, T, dim)).astype(np.float32) for _ in range(3)]
    ps = norm.parameters() + att.parameters()
    w, Wq, Wk, Wv, Wo = [host(p).astype(np.float64) for p in ps]
    X = dev(x, True)
    y, s = norm(X, dev(res))
    out = att(y) + s
    opt = nn.AdamW(ps, 0.01, weight_decay=0.1)
    (out * dev(G)).sum().backward()

    S = x.astype(np.float64) + res
    r = 1 / np.sqrt((S * S).mean(-1, keepdims=True) + 1e-6)
    n = S * r
    Y = n * w
    q, k, v = [(Y @ W).reshape(B, T, -1, D) for W in (Wq, Wk, Wv)]
    k, v = np.repeat(k, H // Hk, 2), np.repeat(v, H // Hk, 2)
    z = np.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
    z[..., np.triu(np.ones((T, T), bool), 1)] = -np.inf
    p = np.exp(z - z.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    a = np.einsum("bhij,bjhd->bihd", p, v).reshape(B, T, dim)
    want = a @ Wo + S
    tol = 40 * 2.0 ** -24 * 64
    assert np.abs(host(out) - want).max() < tol * np.abs(want).max()
    g = G.astype(np.float64)
    dWo = a.reshape(-1, dim).T @ g.reshape(-1, dim)
    da = (g @ Wo.T).reshape(B, T, H, D)
    dv = np.einsum("bhij,bihd->bjhd", p, da)
    dp = np.einsum("bihd,bjhd->bhij", da, v)
    dz = p * (dp - (p * dp).sum(-1, keepdims=True)) * D ** -0.5
    dq, dk = np.einsum("bhij,bjhd->bihd", dz, k), np.einsum("bhij,bihd->bjhd", dz, q)
    dk, dv = [t.reshape(B, T, Hk, H // Hk, D).sum(3).reshape(B * T, -1) for t in (dk, dv)]
    dq, y2 = dq.reshape(B * T, -1), Y.reshape(-1, dim)
    dY = (dq @ Wq.T + dk @ Wk.T + dv @ Wv.T).reshape(B, T, dim)
    dw = (dY * n).sum((0, 1))
    gw = dY * w
    dX = g + r * (gw - n * (gw * n).mean(-1, keepdims=True))
    grads = (dw, y2.T @ dq, y2.T @ dk, y2.T @ dv, dWo)
    for got, exact in zip([X.grad] + [t.grad for t in ps], (dX,) + grads):
        assert np.abs(host(got) - exact).max() < tol * np.abs(exact).max()
    opt.step()
    for par, old, gr in zip(ps, (w, Wq, Wk, Wv, Wo), [host(t.grad) for t in ps]):
        gr = gr.astype(np.float64)  # m / sqrt(v) of the first step is the sign, but for eps
        new = old - 0.01 * 0.1 * old - 0.01 * gr / (np.abs(gr) + 1e-8)
        assert np.abs(host(par) - new).max() < 2.0 ** -24 * 16 * max(1, np.abs(new).max())


def test_sharing_heads_and_long_texts(gpu):
    """The module on a text as long as the half-precision planes are used for:
    finite, and its gradients repeat."""
    nt.manual_seed(9)
    att = nn.Attention(256, 4, 1)
    x = dev(np.random.default_rng(1).standard_normal((1, 1500, 256)).astype(np.float32), True)
    grads = []
    for _ in range(2):
        x.zero_grad()
        (att(x) ** 2).mean().backward()
        grads.append(host(x.grad))
    assert np.isfinite(grads[0]).all() and (grads[0] == grads[1]).all()
