"""Gradients of the token operators where they can go wrong: gradients that
share memory with the results, nearly uniform rows, results changed in place,
left-out tokens in the radix sort, logits that outgrow the Infinity Cache.

Tolerances are those of test_gpu_tokens; sums of small integers, which are
exact in any order, are compared bit for bit."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import assert_bitexact, dev, host, rng, seed_of
from test_gpu_tokens import FLOATS, U, Rows, draw_rows, within

import nanotorch_amd as nt
from nanotorch_amd.autograd.function import Function

pytestmark = pytest.mark.gpu


# ------------------------------------------- gradients that share memory


class HandsOn(Function):
    """sum(x * y), whose backward hands its saved tensors on as they are."""

    def forward(self, x, y):
        self.save_for_backward(x, y)
        with nt.no_grad():
            return (x * y).sum()

    def backward(self, grad_out):
        x, y = self.saved_tensors
        return y, x


@pytest.mark.parametrize("swapped", [False, True])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,V", [(1, 5), (7, 40), (3, 9000)])
def test_results_as_gradients(gpu, dtype, rows, V, swapped):
    """The gradient of logprob is the entropy's own tensor and the other way
    round: sum(logprob * entropy)."""
    z, t = draw_rows(rng(seed_of("hands", rows, V)), rows, V, dtype)
    Z = dev(z, True)
    out = nt.token_logprobs(Z, dev(t), entropy=True)
    a, b = host(out.entropy), host(out.logprob)
    pair = (out.entropy, out.logprob) if swapped else (out.logprob, out.entropy)
    HandsOn.apply(*pair).backward()
    Rows(z, dtype).check_grad(host(Z.grad), t, a, b)
    assert_bitexact(host(out.entropy), a)
    assert_bitexact(host(out.logprob), b)


@pytest.mark.parametrize("wanted", ["logprob", "entropy"])
@pytest.mark.parametrize("rows,V", [(1, 1), (9, 100), (3, 9000)])
def test_one_result_of_two_in_the_loss(gpu, rows, V, wanted):
    z, t = draw_rows(rng(seed_of("one", rows, V)), rows, V, np.float32)
    w = rng(1).standard_normal(rows).astype(np.float32)
    Z = dev(z, True)
    for times in (1, 2):  # a new gradient, then added to it
        (getattr(nt.token_logprobs(Z, dev(t), entropy=True), wanted) * dev(w)).sum().backward()
        a, b = (times * w, None) if wanted == "logprob" else (None, times * w)
        Rows(z, np.float32).check_grad(host(Z.grad), t, a, b)


# ------------------------------------------------------ nearly uniform rows


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("base", [0.0, 1.0])
@pytest.mark.parametrize("rows,V", [(5, 10), (4, 200), (6, 1000), (4, 3001), (2, 32000)])
def test_entropy_gradient_of_nearly_uniform_rows(gpu, dtype, rows, V, base):
    """-p_j (log p_j + H) = p_j (E d - d_j), d = z - max z: it vanishes with
    the logits' spread, and so does its bound, which holds no log s (u the unit
    roundoff, r a sum's relative error as in test_gpu_tokens): p_j is off by
    r + u (8 + |d_j|) of itself, E d = u / s by 2 r + 2u, d_j by u."""
    u = U[dtype]
    r = rng(seed_of("uniform", rows, V))
    z = (base + r.standard_normal((rows, V)) * 2.0 ** -13).astype(dtype)
    b = r.standard_normal(rows).astype(dtype)
    Z = dev(z, True)
    (nt.token_logprobs(Z, entropy=True).entropy * dev(b)).sum().backward()
    z = z.astype(np.longdouble)
    d = z - z.max(1, keepdims=True)
    e = np.exp(d)
    p = e / e.sum(1, keepdims=True)
    ed = (p * d).sum(1, keepdims=True)
    b = b[:, None].astype(np.longdouble)
    want = b * p * (ed - d)
    rel = u * (8 + np.abs(ed) + V / 64 + 32)
    size = np.abs(b) * p
    tol = (size * (np.abs(ed) + np.abs(d)) * (rel + u * (16 + np.abs(d)))
           + size * ((2 * rel + 2 * u) * np.abs(ed) + u * np.abs(d)) + 2 * u * np.abs(want))
    within(host(Z.grad), want, tol, "dz")


# ------------------------------------------------- results changed in place


@pytest.mark.parametrize("saved,changed", [
    ("entropy", "logprob"), ("logprob", "entropy"), ("logprob", "top_logprobs"),
    ("entropy", "top_logprobs"), ("logprob", "top_tokens")])
def test_a_result_changed_in_place_leaves_the_others(gpu, saved, changed):
    z, t = draw_rows(rng(3), 6, 30, np.float32)
    w = dev(rng(4).standard_normal(6).astype(np.float32), True)
    Z = dev(z, True)
    out = nt.token_logprobs(Z, dev(t), entropy=True, top=4)
    before = host(getattr(out, saved))
    loss = (getattr(out, saved) * w).sum()  # keeps the result for w's gradient
    with nt.no_grad():
        other = getattr(out, changed)
        other += 1
    loss.backward()
    assert_bitexact(host(w.grad), before)
    a, b = (host(w), None) if saved == "logprob" else (None, host(w))
    Rows(z, np.float32).check_grad(host(Z.grad), t, a, b)


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("name", ["logprob", "entropy"])
def test_a_saved_result_changed_in_place_is_refused(gpu, name, top):
    z, t = draw_rows(rng(5), 6, 30, np.float32)
    w = dev(np.ones(6, np.float32), True)
    out = nt.token_logprobs(dev(z, True), dev(t), entropy=True, top=top)
    loss = (getattr(out, name) * w).sum()
    with nt.no_grad():
        x = getattr(out, name)
        x += 1
    with pytest.raises(RuntimeError):
        loss.backward()


def test_results_outlive_each_other(gpu):
    """The results share one allocation: it stays while any of them is used."""
    z, t = draw_rows(rng(6), 300, 40, np.float32)
    ref = Rows(z, np.float32)
    out = nt.token_logprobs(dev(z, True), dev(t), entropy=True, top=4)
    top = out.top_logprobs
    del out
    others = [nt.full(2700, value=7.0, device="cuda") for _ in range(8)]
    order = np.argsort(-z, 1, kind="stable")[:, :4]
    within(host(top), np.take_along_axis(ref.logp, order, 1),
           np.take_along_axis(ref.tol_lp, order, 1))
    assert all((host(x) == 7).all() for x in others)


# ------------------------------------------------------------------- types


@pytest.mark.parametrize("flag", [1, 2, "yes"])
def test_logits_that_require_grad_by_their_truth(gpu, flag):
    z, t = draw_rows(rng(7), 5, 300, np.float32)
    a, b = rng(8).standard_normal((2, 5)).astype(np.float32)
    Z = nt.Tensor(z, requires_grad=flag, device="cuda")
    out = nt.token_logprobs(Z, dev(t), entropy=True, top=2)
    (out.logprob * dev(a) + out.entropy * dev(b)).sum().backward()
    Rows(z, np.float32).check_grad(host(Z.grad), t, a, b)


@pytest.mark.parametrize("flag", [1, 2, np.True_])
def test_entropy_is_asked_for_by_its_truth(gpu, flag):
    z, t = draw_rows(rng(9), 700, 20, np.float32)
    a, b = rng(10).standard_normal((2, 700)).astype(np.float32)
    for grad in (False, True):
        Z = dev(z, grad)
        out = nt.token_logprobs(Z, dev(t), entropy=flag, top=3)
        Rows(z, np.float32).check(out, t, True, 3)
    (out.logprob * dev(a) + out.entropy * dev(b)).sum().backward()
    Rows(z, np.float32).check_grad(host(Z.grad), t, a, b)


@pytest.mark.parametrize("op", ["embedding", "dropout", "logprob"])
@pytest.mark.parametrize("strided", [False, True])
def test_added_to_a_gradient_of_another_type(gpu, op, strided):
    """Float32 operators whose input already has a float64 gradient, as one
    that is also multiplied by float64 weights gets: added to it as they are.
    The start is a quarter of small integers, the sums exact."""
    r = rng(seed_of("into", op))
    x = r.standard_normal((20, 12)).astype(np.float32)
    t = r.integers(0, 12, 20)
    start = r.integers(-40, 40, (12, 20) if strided else (20, 12)) / 4.0
    g = r.integers(-4, 5, (20,) if op == "logprob" else (20, 12)).astype(np.float32)
    X = dev(x, True)
    y = {"embedding": lambda: nt.embedding(X, dev(t)),
         "dropout": lambda: nt.dropout(X, 0.5, seed=3),
         "logprob": lambda: nt.token_logprobs(X, dev(t)).logprob}[op]()
    alone = host(y.grad_fn.backward(dev(g))[0])
    assert alone.dtype == np.float32
    target = dev(start).T if strided else dev(start)
    y.grad_fn._backward_into(dev(g), [True, False], [target, None])
    assert_bitexact(host(target), alone + (start.T if strided else start))


# ---------------------------------------------------- radix-sorted gradient


@pytest.mark.parametrize("left_out", ["some", "most", "all"])
@pytest.mark.parametrize("N", [17001, 70001, (1 << 21) + 5001])
@pytest.mark.parametrize("V", [700, 511, 512, 1 << 18])
def test_radix_sorted_gradient_of_left_out_tokens(gpu, V, N, left_out):
    """Many tokens, of which some, most or all are padding or lie outside the
    table; V + 1 sort keys in one, two and three digits, some with a digit bit
    only for the left-out key; new gradients and added ones, contiguous and
    with longer rows."""
    D = 5
    r = rng(seed_of("radix", V, N, left_out))
    t = r.integers(0, V, N)
    hit = r.random(N) < {"some": 0.2, "most": 0.98, "all": 2.0}[left_out]
    padding = V // 3
    t[hit] = padding
    g = r.integers(-8, 9, (N, D)).astype(np.float32)
    G = dev(g)
    kept = t != padding
    want = np.stack([np.bincount(t[kept], g[kept, c], V) for c in range(D)], 1)
    want = want.astype(np.float32)
    w = dev(np.zeros((V, D), np.float32), True)
    y = nt.embedding(w, dev(t), padding_idx=padding)
    assert_bitexact(host(y.grad_fn.backward(G)[0]), want, "padding")
    start = r.integers(-8, 9, (V, D + 3)).astype(np.float32)
    for wide in (False, True):
        S = dev(start if wide else start[:, :D])
        into = S[:, 2:D + 2] if wide else S
        y.grad_fn._backward_into(G, [True, False], [into, None])
        expect = start.copy() if wide else start[:, :D].copy()
        (expect[:, 2:D + 2] if wide else expect)[...] += want
        assert_bitexact(host(S), expect, "added")
    bad = t.copy()
    bad[hit] = np.where(np.arange(hit.sum()) % 2, -1, V)
    kept = (bad >= 0) & (bad < V)
    want = np.stack([np.bincount(t[kept], g[kept, c], V) for c in range(D)], 1)
    want = want.astype(np.float32)
    y = nt.embedding(w, dev(bad))
    with pytest.raises(IndexError):
        nt.sync()
    dw = y.grad_fn.backward(G)[0]
    with pytest.raises(IndexError):
        nt.sync()
    assert_bitexact(host(dw), want, "outside")
    S = dev(start[:, :D])
    y.grad_fn._backward_into(G, [True, False], [S, None])
    with pytest.raises(IndexError):
        nt.sync()
    assert_bitexact(host(S), start[:, :D] + want, "outside, added")


# --------------------------------------- logits that outgrow the Infinity Cache


@pytest.mark.parametrize("dtype,rows,V,top", [
    (np.float32, 2100000, 33, 0), (np.float32, 700000, 100, 2), (np.float32, 270000, 260, 0),
    (np.float32, 20000, 4001, 3), (np.float32, 16500, 4101, 0), (np.float32, 16500, 4101, 5),
    (np.float64, 8300, 4101, 2), (np.float64, 1100000, 31, 0), (np.float64, 270000, 127, 0)])
def test_logits_larger_than_the_cache(gpu, dtype, rows, V, top):
    """More than 256 MB: read past the cache, the gradient's last rows first.
    Rows that differ in logits, tokens and upstream weights, some left out;
    blocks of rows from the first to the last, new gradients and added ones."""
    assert rows * V * np.dtype(dtype).itemsize > 256 << 20
    r = rng(seed_of("cache", rows, V))
    z = r.standard_normal((rows, V), dtype=dtype)
    t = r.integers(0, V, rows)
    t[r.random(rows) < 0.2] = -100
    a, b = r.standard_normal((2, rows)).astype(dtype)
    Z = dev(z, True)
    out = nt.token_logprobs(Z, dev(t), entropy=True, top=top)
    start = r.standard_normal((16, V)).astype(dtype)
    added = dev(np.resize(start, (rows, V)))  # row i: start[i % 16]
    A, B = dev(a), dev(b)
    (out.logprob * A + out.entropy * B).sum().backward()
    only = nt.token_logprobs(Z, dev(t)).logprob
    only.grad_fn._backward_into(A, [True, False], [added, None])
    blocks = {0, 1, rows // 3, rows // 2, rows - 41, rows - 20} | {
        int(k) for k in r.integers(0, rows - 20, 6)}
    for k in sorted(blocks):
        part = slice(k, k + 20)
        live = t[part] != -100
        ref = Rows(z[part], dtype, live)
        cut = nt.TokenLogProbs(*(None if x is None else x[part] for x in out))
        ref.check(cut, np.where(live, t[part], 0), True, top)
        tokens = np.where(live, t[part], 0)
        ref.check_grad(host(Z.grad[part]), tokens, a[part], b[part])
        ref.check_grad(host(added[part]), tokens, a[part], None,
                       extra=start[np.arange(k, min(k + 20, rows)) % 16])
