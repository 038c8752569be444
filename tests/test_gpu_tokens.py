"""The token operators (embedding lookup and gradient, dropout, token log
probabilities) against plain numpy in 64 bits, or in the host's long double
where the operator itself works in 64 bits and the reference's own rounding
would count.

Tolerances.  u is the unit roundoff (2^-24, 2^-53).  A lookup is one product
and dropout one product with a rounded factor: compared bit for bit.  A row of
the table's gradient sums n terms in some fixed order and is scaled once:
(n + 1) u sum|terms|.  For the log probabilities, d_j = z_j - max z is rounded
to u |d_j|, exp adds under 8u, and a lane adds up to V/64 + 32 terms (its own,
then the lanes, waves and parts), so s = sum exp(d) is off by at most
r = u (8 + E|d| + V/64 + 32) of itself, with E the mean under p;
    log p = (z_t - max) - log s:  r + 4u (1 + |d_t| + log s)
    H = log s - (sum d exp d)/s:  (2 r + 4u (1 + log s)) (1 + E|d|)
    p_j: r_j = r + u (8 + |d_j|) of itself.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

from helpers import assert_bitexact, dev, host, rng, seed_of

import nanotorch_amd as nt
from nanotorch_amd import nn

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
FLOATS = [np.float32, np.float64]


def within(got, want, tol, what=""):
    got = got.astype(np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    special = ~np.isfinite(want)
    inf = special & ~np.isnan(want)
    assert (got[inf] == want[inf]).all(), what
    assert (np.isnan(got) == np.isnan(want)).all(), what
    tol = np.broadcast_to(tol, want.shape)
    err = np.abs(got[~special] - want[~special])
    bad = err > tol[~special]
    assert not bad.any(), (what, int(bad.sum()), float((err / np.maximum(tol[~special],
                                                                         1e-300)).max()))


# ---------------------------------------------------------------- embedding


def lookup(W, t, scale, padding=None):
    y = W[t] * W.dtype.type(scale)
    if padding is not None:
        y[t == padding] = 0
    return y


def table_grad(g, t, V, scale, padding=None):
    """(gradient, sum of |terms|, terms per row)"""
    g = g.astype(np.longdouble).reshape(t.size, g.shape[-1])
    t = t.reshape(-1)
    if padding is not None:
        g, t = g[t != padding], t[t != padding]
    dw, mag = np.zeros((2, V, g.shape[1]), np.longdouble)
    np.add.at(dw, t, g)
    np.add.at(mag, t, np.abs(g))
    return dw * scale, mag * abs(scale), np.bincount(t, minlength=V)[:, None]


def check_table_grad(got, g, t, V, scale, dtype, padding=None, parts=1):
    want, mag, n = table_grad(g, t, V, scale, padding)
    within(got, want, (n + parts) * U[dtype] * mag, "dW")
    assert (got[(n == 0)[:, 0]] == 0).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("V,D,N,kind", [
    (1, 1, 1, "one"), (7, 3, 5, "any"), (1000, 64, 64, "any"), (50, 255, 300, "any"),
    (300, 257, 2048, "zipf"), (300, 260, 2049, "zipf"), (4000, 33, 9000, "zipf"),
    (70000, 20, 17000, "any"), (129, 512, 5000, "one"), (5, 1023, 4097, "few"),
    (131072, 8, 40000, "zipf"), (300000, 4, 20001, "any"), (2, 16, 70001, "any"),
    (3, 300, 4000, "one"), (511, 8, 17000, "any"), (512, 8, 17000, "any"),
    (600, 3, 1100000, "zipf"),
])
def test_embedding(gpu, dtype, V, D, N, kind):
    r = rng(seed_of(dtype.__name__, V, D, N))
    W = r.standard_normal((V, D)).astype(dtype)
    t = {"any": lambda: r.integers(0, V, N),
         "zipf": lambda: np.clip(np.exp(r.random(N) * math.log(V + 1)).astype(np.int64) - 1,
                                 0, V - 1),
         "one": lambda: np.full(N, V - 1),
         "few": lambda: r.integers(V - 3, V, N)}[kind]().astype(np.int64)
    g = r.standard_normal((N, D)).astype(dtype)
    w, G = dev(W, True), dev(g)
    for tokens in (t, t.astype(np.int32)):
        y = nt.embedding(w, dev(tokens), 3.0)
        assert_bitexact(host(y), lookup(W, t, 3.0))
        dw = y.grad_fn.backward(G)[0]
        check_table_grad(host(dw), g, t, V, 3.0, dtype)
        again = y.grad_fn.backward(G)[0]
        assert_bitexact(host(again), host(dw), "a second run")


@pytest.mark.parametrize("V", [700, 100000])
def test_embedding_gradient_of_very_many_tokens(gpu, V):
    """Sorted by more workgroups than add up each other's counts.  Small
    integers, whose sums are exact in any order."""
    N, D = (1 << 21) + 5001, 5
    r = rng(seed_of("many", V))
    t = np.where(r.random(N) < 0.2, 3, r.integers(0, V, N))
    g = r.integers(-8, 9, (N, D)).astype(np.float32)
    y = nt.embedding(dev(np.zeros((V, D), np.float32), True), dev(t))
    want = np.stack([np.bincount(t, g[:, c], V) for c in range(D)], 1)
    assert_bitexact(host(y.grad_fn.backward(dev(g))[0]), want.astype(np.float32))


@pytest.mark.parametrize("shape", [(), (0,), (4, 0), (3, 1, 5), (2, 3, 4, 5)])
def test_embedding_token_shapes(gpu, shape):
    r = rng(seed_of(shape))
    W = r.standard_normal((11, 6)).astype(np.float32)
    t = np.asarray(r.integers(0, 11, shape))
    w = dev(W, True)
    y = nt.embedding(w, nt.Tensor(t, device="cuda"))
    assert y.shape == shape + (6,)
    assert_bitexact(host(y), W[t])
    y.sum().backward()  # a broadcast gradient
    check_table_grad(host(w.grad), np.ones(shape + (6,)), t, 11, 1.0, np.float32)


@pytest.mark.parametrize("N", [100, 6000])
@pytest.mark.parametrize("dtype", FLOATS)
def test_embedding_padding(gpu, dtype, N):
    r = rng(seed_of("padding", N))
    W = r.standard_normal((9, 70)).astype(dtype)
    t = r.integers(0, 9, N)
    g = r.standard_normal((N, 70)).astype(dtype)
    y = nt.embedding(dev(W, True), dev(t), 0.5, padding_idx=4)
    assert_bitexact(host(y), lookup(W, t, 0.5, 4))
    check_table_grad(host(y.grad_fn.backward(dev(g))[0]), g, t, 9, 0.5, dtype, 4)


@pytest.mark.parametrize("N", [37, 4000])
@pytest.mark.parametrize("dtype", FLOATS)
def test_embedding_views(gpu, dtype, N):
    """Tables and tokens that are views: a layer's weight transposed, rows
    and columns taken from a larger table, every other token, one token for
    all positions."""
    r = rng(seed_of("views", N))
    base = r.standard_normal((40, 90)).astype(dtype)
    t = r.integers(0, 20, 2 * N)
    g = r.standard_normal((N, 21)).astype(dtype)
    b, T, G = dev(base), dev(t), dev(g)
    for view, ref in ((lambda x: x.T[:40, 3:24], base.T[:40, 3:24]),
                      (lambda x: x[5:31, 7:28], base[5:31, 7:28]),
                      (lambda x: x[::2, ::4][:, :21], base[::2, ::4][:, :21])):
        w = view(b)
        w.enable_grad()
        y = nt.embedding(w, T[1::2], 2.0)
        assert_bitexact(host(y), lookup(ref, t[1::2], 2.0))
        check_table_grad(host(y.grad_fn.backward(G)[0]), g, t[1::2], ref.shape[0], 2.0, dtype)
    same = T[3:4].expand(N)
    w = dev(base[:, :21].copy(), True)
    y = nt.embedding(w, same)
    assert_bitexact(host(y), np.repeat(base[t[3]][None, :21], N, 0))
    check_table_grad(host(y.grad_fn.backward(G)[0]), g, np.full(N, t[3]), 40, 1.0, dtype)


@pytest.mark.parametrize("N", [50, 5000])
@pytest.mark.parametrize("tied", [False, True])
def test_embedding_gradient_is_added(gpu, tied, N):
    """A table used twice, the second gradient added in place; tied to a
    layer's weight, through its transposed view."""
    r = rng(seed_of("added", tied, N))
    W = r.standard_normal((30, 17)).astype(np.float32)
    t1, t2 = r.integers(0, 30, N), r.integers(0, 5, 77)
    g1 = r.standard_normal((N, 17)).astype(np.float32)
    g2 = r.standard_normal((77, 17)).astype(np.float32)
    p = dev(np.ascontiguousarray(W.T) if tied else W, True)
    w = p.T if tied else p
    loss = ((nt.embedding(w, dev(t1)) * dev(g1)).sum()
            + (nt.embedding(w, dev(t2), 2.0) * dev(g2)).sum())
    loss.backward()
    got = host(p.grad).T if tied else host(p.grad)
    a, ma, na = table_grad(g1, t1, 30, 1.0)
    b, mb, nb = table_grad(g2, t2, 30, 2.0)
    within(got, a + b, (na + nb + 3) * U[np.float32] * (ma + mb))


def test_embedding_adds_into_a_strided_gradient(gpu):
    r = rng(11)
    t = r.integers(0, 12, 40)
    g = r.standard_normal((40, 8)).astype(np.float32)
    start = r.standard_normal((8, 12)).astype(np.float32)
    w = dev(r.standard_normal((12, 8)).astype(np.float32), True)
    y = nt.embedding(w, dev(t))
    target = dev(start).T
    y.grad_fn._backward_into(dev(g), [True, False], [target, None])
    want, mag, n = table_grad(g, t, 12, 1.0)
    within(host(target), want + start.T, (n + 2) * U[np.float32] * (mag + np.abs(start.T)))


@pytest.mark.parametrize("N", [10, 3000])
@pytest.mark.parametrize("bad", [-1, -5, 6, 2 ** 31 - 1])
def test_embedding_token_outside_the_table(gpu, bad, N):
    r = rng(5)
    W = r.standard_normal((6, 5)).astype(np.float32)
    t = r.integers(0, 6, N).astype(np.int32)
    t[N // 2] = bad
    g = r.standard_normal((N, 5)).astype(np.float32)
    y = nt.embedding(dev(W, True), dev(t))
    with pytest.raises(IndexError):
        nt.sync()
    kept = t != bad
    want = np.where(kept[:, None], W[np.where(kept, t, 0)], 0)
    assert_bitexact(host(y), want)
    dw = y.grad_fn.backward(dev(g))[0]
    with pytest.raises(IndexError):
        nt.sync()
    check_table_grad(host(dw), g[kept], t[kept].astype(np.int64), 6, 1.0, np.float32)


def test_embedding_gradient_by_differences(gpu):
    """float64: (f(W + h e) - f(W - h e)) / 2h is exact for a linear map but
    for rounding: 27 terms of about 1, 27 u each, times 1 / h."""
    r = rng(8)
    W, c = r.standard_normal((5, 3)), r.standard_normal((9, 3))
    t = r.integers(0, 5, 9)

    def f(a):
        return (nt.embedding(a, dev(t), 1.5) * dev(c)).sum()

    w = dev(W, True)
    f(w).backward()
    for i in np.ndindex(5, 3):
        e = np.zeros((5, 3))
        e[i] = 2.0 ** -10
        diff = (host(f(dev(W + e))) - host(f(dev(W - e)))) * 2.0 ** 9
        assert abs(diff - host(w.grad)[i]) < 2.0 ** -53 * 2.0 ** 20


def test_embedding_refusals(gpu):
    w, t = dev(np.ones((4, 3), np.float32)), dev(np.zeros(2, np.int64))
    for bad in (lambda: nt.embedding(dev(np.ones(4, np.float32)), t),
                lambda: nt.embedding(dev(np.ones((4, 3), np.int64)), t),
                lambda: nt.embedding(w, dev(np.zeros(2, np.float32))),
                lambda: nt.embedding(w, dev(np.zeros(2, np.bool_))),
                lambda: nt.embedding(w, t, padding_idx=4),
                lambda: nt.embedding(w, t, padding_idx=-1),
                lambda: nn.Embedding(0, 3), lambda: nn.Embedding(3, 3, padding_idx=3)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        nt.embedding(nt.ones(4, 3), t)
    with pytest.raises(RuntimeError):
        nt.embedding(w, nt.zeros(2, dtype=nt.int64))
    w.enable_grad()
    y = nt.embedding(w, t)
    t += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


# ------------------------------------------------------------------ dropout


def words(n, seed, offset):
    """The first n words of Philox4x32-10 over the counters (i, offset)."""
    return words_of(np.arange((n + 3) // 4, dtype=np.uint64), seed, offset)[:n]


def words_of(i, seed, offset):
    low, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [i & low, i >> s32, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & low,
             (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)


def dropped(x, p, seed, offset):
    keep = words(x.size, seed, offset).reshape(x.shape) >= np.uint64(round(p * 2 ** 32))
    return np.where(keep, x * x.dtype.type(1 / (1 - p) if p < 1 else 0), x.dtype.type(0))


def test_philox_published_words():
    # the generator's published known answers for ten rounds: counter and key
    # zero; all ones
    assert [int(v) for v in words(4, 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(), (0,), (1,), (3,), (4,), (5,), (1023,), (64, 256),
                                   (3, 0, 2), (7, 5, 3), (1000, 77), (1 << 20,)])
def test_dropout(gpu, dtype, shape):
    r = rng(seed_of(shape))
    x = np.asarray(r.standard_normal(shape)).astype(dtype)
    g = np.asarray(r.standard_normal(shape)).astype(dtype)
    for p, seed, offset in ((0.5, 0, 0), (0.1, 2 ** 64 - 3, 2 ** 33 + 5), (0.999, 77, 1),
                            (1.0, 1, 2)):
        X = nt.Tensor(x, device="cuda")
        X.enable_grad()
        y = nt.dropout(X, p, seed=seed, offset=offset)
        assert_bitexact(host(y), dropped(x, p, seed, offset))
        dx = y.grad_fn.backward(nt.Tensor(g, device="cuda"))[0]
        assert_bitexact(host(dx), dropped(g, p, seed, offset))


@pytest.mark.parametrize("dtype", FLOATS)
def test_dropout_views(gpu, dtype):
    """The mask belongs to the logical index: a view loses what its copy does."""
    a = rng(3).standard_normal((70, 90, 6)).astype(dtype)
    A = dev(a)
    for f in (lambda x: x[:, :, 2], lambda x: x.transpose(0, 2) if isinstance(x, nt.Tensor)
              else x.swapaxes(0, 2), lambda x: x[3:50, 1:88:3], lambda x: x[5], lambda x: x[1:2]):
        assert_bitexact(host(nt.dropout(f(A), 0.3, seed=9)), dropped(f(a), 0.3, 9, 0))
    row = A[0, 0:1].expand(50, 6)
    assert_bitexact(host(nt.dropout(row, 0.3, seed=9)),
                    dropped(np.repeat(a[0, 0:1], 50, 0), 0.3, 9, 0))
    flat = dev(a.reshape(-1))[1:]  # not aligned to 16 bytes
    assert_bitexact(host(nt.dropout(flat, 0.3, seed=9)), dropped(a.reshape(-1)[1:], 0.3, 9, 0))


@pytest.mark.parametrize("shape", [(67, 129), (128, 64), (1, 300), (1537, 1023)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_dropout_transposed(gpu, dtype, shape):
    a = rng(seed_of(shape)).standard_normal(shape).astype(dtype)
    x = dev(a).T
    x.enable_grad()
    y = nt.dropout(x, 0.25, seed=4, offset=6)
    assert_bitexact(host(y), dropped(a.T, 0.25, 4, 6))
    g = rng(1).standard_normal(shape[::-1]).astype(dtype)
    assert_bitexact(host(y.grad_fn.backward(dev(np.ascontiguousarray(g.T)).T)[0]),
                    dropped(g, 0.25, 4, 6))


@pytest.mark.parametrize("shape", [(3, 5, 1), (2, 3, 3), (5, 4, 4), (9, 17, 31), (40, 33, 64)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_dropout_rows_of_views(gpu, dtype, shape):
    """Rows of adjacent elements, of lengths below and beside a counter's
    four, in views of two to four dimensions; planes of columns; both passes,
    new and added."""
    a = rng(seed_of("rows", shape)).standard_normal((2,) + shape[:2] + (shape[2] + 3,))
    a = a.astype(dtype)
    swapped = (0, 2, 1, 3), (0, 1, 3, 2), (3, 1, 2, 0), (2, 3, 0, 1)
    for cut in (lambda x: x[..., 1:shape[2] + 1], lambda x: x[0, :, ::2, :shape[2]],
                lambda x: x[1, 1, :, :shape[2]], lambda x: x[..., ::2]):
        v, V = cut(a), cut(dev(a))
        orders = swapped if v.ndim == 4 else [tuple(range(v.ndim)), tuple(range(v.ndim))[::-1]]
        for order in orders:
            w, W = v.transpose(order), V
            left = list(range(v.ndim))
            for k, o in enumerate(order):  # one exchange of axes at a time
                j = left.index(o)
                if j != k:
                    W = W.transpose(k, j)
                    left[k], left[j] = left[j], left[k]
            assert W.shape == w.shape
            assert_bitexact(host(nt.dropout(W, 0.4, seed=8, offset=3)), dropped(w, 0.4, 8, 3))
            x = dev(np.ascontiguousarray(w), True)
            y = nt.dropout(x, 0.4, seed=8, offset=3)
            target = dev(a.copy())
            into = cut(target)
            left = list(range(v.ndim))
            for k, o in enumerate(order):
                j = left.index(o)
                if j != k:
                    into = into.transpose(k, j)
                    left[k], left[j] = left[j], left[k]
            y.grad_fn._backward_into(W, [True], [into])
            want = a.copy()
            cut(want).transpose(order)[...] += dropped(w, 0.4, 8, 3)
            assert_bitexact(host(target), want)


@pytest.mark.parametrize("strided", [False, True])
def test_dropout_gradient_is_added(gpu, strided):
    a = rng(2).standard_normal((33, 65)).astype(np.float32)
    x = dev(a, True)
    y = x.T if strided else x
    ((nt.dropout(y, 0.5, seed=1) + nt.dropout(y, 0.25, seed=2, offset=8)).sum() + x.sum()
     ).backward()
    ones = np.ones(y.shape, np.float32)
    m = (dropped(ones, 0.5, 1, 0).astype(np.float64) + dropped(ones, 0.25, 2, 8) + 1)
    got = host(x.grad).T if strided else host(x.grad)
    within(got, m, 4 * U[np.float32] * m)


def test_dropout_discards_special_values(gpu):
    x = np.full(4000, np.nan, np.float32)
    x[::3] = np.inf
    y = host(nt.dropout(dev(x), 0.5, seed=5))
    assert_bitexact(y, dropped(x, 0.5, 5, 0))
    assert (y == 0).any()


def test_dropout_generator(gpu):
    x = nt.ones(1000, device="cuda")
    nt.manual_seed(12)
    a, b = host(nt.dropout(x)), host(nt.dropout(x))
    u = host(nt.rand(5, device="cuda"))
    nt.manual_seed(12)
    assert_bitexact(host(nt.rand(5, device="cuda")), u)  # rand's own stream is untouched
    assert_bitexact(host(nt.dropout(x)), a)
    assert_bitexact(host(nt.dropout(x)), b)
    assert (a != b).any()
    assert_bitexact(a, dropped(np.ones(1000, np.float32), 0.5, 12, 0))
    assert_bitexact(b, dropped(np.ones(1000, np.float32), 0.5, 12, 1))


def test_dropout_module(gpu):
    x = dev(rng(0).standard_normal((40, 50)).astype(np.float32), True)
    net = nn.Sequential(nn.Dropout(0.5), nn.Tanh())
    y = net.eval()(x)
    assert_bitexact(host(y), host(nt.tanh(x)))
    assert (host(net.train()(x)) == 0).mean() > 0.4
    for p in (0.0, 1.0):
        y = nn.Dropout(p)(x)
        assert_bitexact(host(y), host(x) if p == 0 else np.zeros((40, 50), np.float32))
        x.zero_grad()
        y.sum().backward()
        assert (host(x.grad) == (1 - p)).all()


def test_dropout_refusals(gpu):
    x = nt.ones(4, device="cuda")
    for bad in (lambda: nt.dropout(x, -0.1), lambda: nt.dropout(x, 1.5),
                lambda: nt.dropout(x, float("nan")),
                lambda: nt.dropout(nt.ones(4, dtype=nt.int32, device="cuda")),
                lambda: nn.Dropout(2.0)):
        with pytest.raises(ValueError):
            bad()
    for p in (0.0, 0.5):
        with pytest.raises(RuntimeError):
            nt.dropout(nt.ones(4), p)


# ------------------------------------------------------- log probabilities


class Rows:
    """The definition for z [rows, V], with the tolerances."""

    def __init__(self, z, dtype, live=None):
        u = U[dtype]
        z = z.astype(np.longdouble if dtype == np.float64 else np.float64)
        rows, V = z.shape
        self.z, self.u = z, u
        with np.errstate(all="ignore"):
            m = z.max(1, keepdims=True)
            self.none = (m == -np.inf)[:, 0]
            m[self.none] = 0
            d = z - m
            e = np.exp(d)
            s = e.sum(1, keepdims=True)
            self.p = np.where(self.none[:, None], 0, e / np.where(s == 0, 1, s))
            self.logp = np.where(self.none[:, None], -np.inf, d - np.log(s))
            dd = np.where(e == 0, 0, d)
            pd = np.where(self.p == 0, 0, self.p * dd)
            self.H = np.where(self.none, 0, np.log(s)[:, 0] - pd.sum(1))
            ed = np.abs(pd).sum(1)
            logs = np.where(self.none, 0, np.abs(np.log(s))[:, 0])
        r = u * (8 + ed + V / 64 + 32)
        self.d = np.where(np.isfinite(d), np.abs(d), 0)
        self.tol_lp = r[:, None] + 4 * u * (1 + self.d + logs[:, None])
        self.tol_H = (2 * r + 4 * u * (1 + logs)) * (1 + ed)
        self.r = r
        self.live = np.ones(rows, bool) if live is None else live

    def check(self, out, t=None, entropy=False, top=0):
        i = np.arange(len(self.z))
        if t is not None:
            at = np.where(self.live, t, 0)
            within(host(out.logprob).reshape(-1), np.where(self.live, self.logp[i, at], 0),
                   self.tol_lp[i, at], "logprob")
        if entropy:
            within(host(out.entropy).reshape(-1), np.where(self.live, self.H, 0), self.tol_H,
                   "entropy")
        if top:
            key = np.where(np.isnan(self.z), np.inf, self.z)
            nan_first = np.isnan(self.z).astype(int)
            order = np.stack([np.lexsort((np.arange(key.shape[1]), -key[r], -nan_first[r]))
                              for r in i])[:, :top]
            token = np.where(self.live[:, None], order, -1)
            assert (host(out.top_tokens).reshape(len(i), top) == token).all()
            want = np.where(self.live[:, None], np.take_along_axis(self.logp, order, 1), -np.inf)
            within(host(out.top_logprobs).reshape(len(i), top), want,
                   np.take_along_axis(self.tol_lp, order, 1), "top")

    def check_grad(self, got, t, a, b, extra=0.0):
        """`extra`: what was there before the gradient was added."""
        u, p = self.u, self.p
        i = np.arange(len(self.z))
        ok = self.live & ~self.none
        a = np.zeros(len(i)) if a is None else np.where(ok, a, 0).astype(np.float64)
        b = np.zeros(len(i)) if b is None else np.where(ok, b, 0).astype(np.float64)
        a, b = a[:, None], b[:, None]
        lp = np.where(p == 0, 0, self.logp)
        with np.errstate(invalid="ignore"):
            want = -p * (a + b * (lp + self.H[:, None]))
            rj = self.r[:, None] + u * (8 + self.d)
            size = p * (np.abs(a) + np.abs(b) * (np.abs(lp) + self.H[:, None] + 1))
            tol = size * (rj + 8 * u) + p * np.abs(b) * (self.tol_lp + self.tol_H[:, None])
        if t is not None:
            at = np.where(self.live, t, 0)
            want[i, at] += a[:, 0]
            tol[i, at] += 2 * u * np.abs(a[:, 0])
        want = want + extra
        tol = tol + 2 * u * np.abs(want) + 2.0 ** -126
        within(got.reshape(want.shape), want, tol, "dz")


def draw_rows(r, rows, V, dtype, masked=0.0):
    z = (r.standard_normal((rows, V)) * 3).astype(dtype)
    t = r.integers(0, V, rows)
    if masked:
        hit = r.random((rows, V)) < masked
        hit[np.arange(rows), t] = False
        z[hit] = -np.inf
    return z, t


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 2), (3, 10), (65, 63), (5, 64), (3, 257),
                                    (9, 1000), (4, 1024), (4, 1025), (2, 2048), (3, 2049),
                                    (7, 4097), (2, 9000), (1, 50001), (300, 5003),
                                    (1030, 4100), (1, 131072), (70, 17), (3, 33), (1001, 65),
                                    (17, 129), (9, 256), (4100, 2100)])
def test_token_logprobs(gpu, dtype, rows, V):
    r = rng(seed_of("lp", dtype.__name__, rows, V))
    z, t = draw_rows(r, rows, V, dtype, 0.1 if V > 200 else 0.0)
    Z = dev(z, True)
    ref = Rows(z, dtype)
    top = min(5, V)
    for tokens in (t, t.astype(np.int32)):
        out = nt.token_logprobs(Z, dev(tokens), entropy=True, top=top)
        ref.check(out, t, True, top)
    out = nt.token_logprobs(Z, dev(t))
    assert out.entropy is None and out.top_tokens is None
    ref.check(out, t)
    a, b = r.standard_normal(rows).astype(dtype), r.standard_normal(rows).astype(dtype)
    ref.check_grad(host(out.logprob.grad_fn.backward(dev(a))[0]), t, a, None)
    out = nt.token_logprobs(Z, entropy=True)
    ref.check(out, None, True)
    ref.check_grad(host(out.entropy.grad_fn.backward(dev(b))[0]), None, None, b)
    with nt.no_grad():
        out = nt.token_logprobs(Z, top=top)
    ref.check(out, None, False, top)
    out = nt.token_logprobs(Z, dev(t), entropy=True)
    (out.logprob * dev(a) + out.entropy * dev(b)).sum().backward()
    ref.check_grad(host(Z.grad), t, a, b)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,V,top", [(3, 64, 64), (2, 700, 64), (4, 5000, 64), (1, 40000, 33),
                                        (600, 3000, 2), (2, 9, 9), (1, 1, 1)])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "rising", "falling", "zeros"])
def test_top_alternatives(gpu, dtype, rows, V, top, kind):
    r = rng(seed_of("top", rows, V, kind))
    z = {"random": lambda: r.standard_normal((rows, V)),
         "ties": lambda: r.integers(-3, 4, (rows, V)),
         "equal": lambda: np.full((rows, V), 1.25),
         "rising": lambda: np.tile(np.arange(V) / 64.0, (rows, 1)),
         "falling": lambda: np.tile(-np.arange(V) / 64.0, (rows, 1)),
         "zeros": lambda: np.where(r.random((rows, V)) < 0.5, 0.0, -0.0)}[kind]().astype(dtype)
    Rows(z, dtype).check(nt.token_logprobs(dev(z), entropy=True, top=top), None, True, top)


@pytest.mark.parametrize("kind", ["random", "tied", "rising"])
@pytest.mark.parametrize("top", [1, 15, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("rows,V", [(1, 131073), (3, 66000), (40, 20000), (1100, 4500)])
@pytest.mark.parametrize("dtype", FLOATS)
def test_top_alternatives_of_split_rows(gpu, dtype, rows, V, top, kind):
    """Lists joined by waves and by workgroups, in 16 lanes and in 64; equal
    logits in different parts; parts of a few elements; the largest last."""
    r = rng(seed_of("split", rows, V, kind))
    z = r.standard_normal((rows, V)).astype(dtype)
    if kind == "tied":
        z = np.round(z)
    elif kind == "rising":
        z.sort(1)
    out = nt.token_logprobs(dev(z), top=top)
    # the largest first, equal ones by their tokens
    found = np.argpartition(-z, top - 1, 1)[:, top - 1:top]
    least = np.take_along_axis(z, found, 1)
    want = []
    for row, low in zip(z, least):
        at = np.flatnonzero(row >= low)
        want.append(at[np.argsort(-row[at], kind="stable")][:top])
    assert_bitexact(host(out.top_tokens), np.array(want))


LOW = {np.float32: np.finfo(np.float32).min, np.float64: np.finfo(np.float64).min}


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("V", [5, 100, 300, 3001, 20000])
def test_masked_rows(gpu, dtype, V):
    """Rows that a mask empties, leaves one token of, or fills with the type's
    lowest value; scores far apart; infinities and NaN."""
    r = rng(seed_of("masked", V))
    z = r.standard_normal((10, V)).astype(dtype)
    t = r.integers(0, V, 10)
    z[0] = -np.inf
    z[1] = -np.inf
    z[1, V // 2] = 3
    t[1] = V // 2
    z[2] = -np.inf
    z[2, V - 1] = -1e30
    t[2] = 0
    z[3] = LOW[dtype]
    z[4] = LOW[dtype]
    z[4, 1] = 2
    t[4] = 1
    z[5, : V // 2] = LOW[dtype]
    z[6, :2] = (1e30, -1e30)
    z[7, V - 2] = np.nan
    z[8, 1] = np.inf
    z[9, 0] = LOW[dtype]
    z[9, 1] = -LOW[dtype]
    t[9] = 1
    ref = Rows(z, dtype)
    Z = dev(z, True)
    ref.check(nt.token_logprobs(Z, dev(t), entropy=True), t, True)
    out = nt.token_logprobs(Z, dev(t), entropy=True, top=3)
    ref.check(out, t, True, 3)
    a, b = r.standard_normal(10).astype(dtype), r.standard_normal(10).astype(dtype)
    (out.logprob * dev(a) + out.entropy * dev(b)).sum().backward()
    ref.check_grad(host(Z.grad), t, a, b)
    assert (host(Z.grad)[0] == 0).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,V", [(12, 30), (50, 200), (40, 3000), (3, 30000), (2000, 2500)])
def test_rows_left_out(gpu, dtype, rows, V):
    r = rng(seed_of("ignored", rows, V))
    z, t = draw_rows(r, rows, V, dtype)
    live = r.random(rows) < 0.6
    live[0], live[1] = False, True
    z[0] = np.nan  # never read
    t = np.where(live, t, -7)
    ref = Rows(z, dtype, live)
    ref.none[0] = False
    ref.p[0] = ref.logp[0] = ref.H[0] = ref.r[0] = 0
    ref.tol_H[0] = 0
    ref.tol_lp[0] = 0
    ref.d[0] = 0
    Z = dev(z, True)
    ref.check(nt.token_logprobs(Z, dev(t), entropy=True, ignore_index=-7), t, True)
    out = nt.token_logprobs(Z, dev(t), entropy=True, top=2, ignore_index=-7)
    ref.check(out, t, True, 2)
    a, b = r.standard_normal(rows).astype(dtype), r.standard_normal(rows).astype(dtype)
    (out.logprob * dev(a) + out.entropy * dev(b)).sum().backward()
    ref.check_grad(host(Z.grad), t, a, b)


@pytest.mark.parametrize("dtype", FLOATS)
def test_logits_views(gpu, dtype):
    """Sliced vocabularies, every other row, a transposed layer's output, one
    row for many tokens, 1-D and 4-D logits."""
    r = rng(21)
    base = (r.standard_normal((6, 50, 70)) * 2).astype(dtype)
    B = dev(base)
    for f in (lambda x: x[:, :, 3:64], lambda x: x[::2, 1::3], lambda x: x[:, :, ::2],
              lambda x: x[2], lambda x: x[1, 4], lambda x: x[:, 5:6],
              lambda x: x.transpose(1, 2) if isinstance(x, nt.Tensor) else x.swapaxes(1, 2),
              lambda x: x.reshape(2, 3, 50, 70), lambda x: x[:, :, 4:5]):
        z = f(base)
        Z = f(B)
        Z.enable_grad()
        t = np.asarray(r.integers(0, z.shape[-1], z.shape[:-1]))
        out = nt.token_logprobs(Z, nt.Tensor(t, device="cuda"), entropy=True,
                                top=min(3, z.shape[-1]))
        assert out.logprob.shape == out.entropy.shape == z.shape[:-1]
        assert out.top_tokens.shape == z.shape[:-1] + (min(3, z.shape[-1]),)
        flat = np.ascontiguousarray(z).reshape(-1, z.shape[-1])
        ref = Rows(flat, dtype)
        ref.check(out, t.reshape(-1), True, min(3, z.shape[-1]))
        (out.logprob.sum() + out.entropy.sum()).backward()
        assert Z.grad.shape == z.shape
        ref.check_grad(host(Z.grad), t.reshape(-1), np.ones(t.size), np.ones(t.size))
    one = B[0, 0:1].expand(40, 70)
    t = r.integers(0, 70, 80)
    ref = Rows(np.repeat(base[0, 0:1], 40, 0), dtype)
    ref.check(nt.token_logprobs(one, dev(t)[::2]), t[::2])


@pytest.mark.parametrize("strided", [False, True])
def test_logits_gradient_is_added(gpu, strided):
    r = rng(31)
    z, t = draw_rows(r, 20, 37, np.float32)
    start = r.standard_normal((37, 20) if strided else (20, 37)).astype(np.float32)
    a = r.standard_normal(20).astype(np.float32)
    out = nt.token_logprobs(dev(z, True), dev(t))
    target = dev(start).T if strided else dev(start)
    out.logprob.grad_fn._backward_into(dev(a), [True, False], [target, None])
    Rows(z, np.float32).check_grad(host(target), t, a, None,
                                   extra=start.T if strided else start)


def test_logits_used_twice(gpu):
    r = rng(32)
    z, t = draw_rows(r, 20, 2500, np.float32)
    Z = dev(z, True)
    (nt.token_logprobs(Z, dev(t)).logprob.sum()
     + nt.token_logprobs(Z, entropy=True).entropy.sum()).backward()
    Rows(z, np.float32).check_grad(host(Z.grad), t, np.ones(20), np.ones(20))


@pytest.mark.parametrize("entropy", [False, True])
def test_logprob_gradient_by_differences(gpu, entropy):
    """float64 central differences with h = 2^-13: truncation h^2 / 6 times a
    third derivative below 8, rounding 2 tol / h."""
    r = rng(41)
    z, t = draw_rows(r, 3, 6, np.float64)
    a, b = r.standard_normal(3), r.standard_normal(3)

    def f(x):
        out = nt.token_logprobs(x, dev(t), entropy=entropy)
        y = out.logprob * dev(a)
        return ((y + out.entropy * dev(b)) if entropy else y).sum()

    Z = dev(z, True)
    f(Z).backward()
    h = 2.0 ** -13
    scale = 3 * (np.abs(a).max() + np.abs(b).max())
    for i in np.ndindex(3, 6):
        e = np.zeros((3, 6))
        e[i] = h
        diff = (float(host(f(dev(z + e)))) - float(host(f(dev(z - e))))) / (2 * h)
        assert abs(diff - host(Z.grad)[i]) < scale * (8 * h * h + 100 * 2.0 ** -53 / h)


@pytest.mark.parametrize("rows,V", [(4, 30), (2, 9000)])
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1])
def test_given_token_outside_the_row(gpu, bad, rows, V):
    r = rng(51)
    z, t = draw_rows(r, rows, V, np.float32)
    t[1] = bad
    live = np.arange(rows) != 1
    Z = dev(z, True)
    out = nt.token_logprobs(Z, dev(t), top=1)
    with pytest.raises(IndexError):
        nt.sync()
    ref = Rows(z, np.float32, live)
    ref.check(out, t, False, 1)
    a = np.ones(rows, np.float32)
    ref.check_grad(host(out.logprob.grad_fn.backward(dev(a))[0]), np.where(live, t, 0), a, None)


def test_no_rows(gpu):
    z = nt.zeros(0, 5, device="cuda")
    z.enable_grad()
    out = nt.token_logprobs(z, nt.zeros(0, dtype=nt.int64, device="cuda"), entropy=True, top=2)
    assert out.logprob.shape == (0,) and out.top_tokens.shape == (0, 2)
    out.logprob.sum().backward()
    assert z.grad.shape == (0, 5)


def test_logprob_refusals(gpu):
    z, t = nt.zeros(2, 70, device="cuda"), nt.zeros(2, dtype=nt.int64, device="cuda")
    for bad in (lambda: nt.token_logprobs(z), lambda: nt.token_logprobs(z, t, top=65),
                lambda: nt.token_logprobs(z, t, top=-1),
                lambda: nt.token_logprobs(z[:, :3], t, top=4),
                lambda: nt.token_logprobs(z, t[:1]), lambda: nt.token_logprobs(z, z),
                lambda: nt.token_logprobs(t, t),
                lambda: nt.token_logprobs(z[0, 0], t),
                lambda: nt.token_logprobs(nt.zeros(2, 0, device="cuda"), t)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        nt.token_logprobs(nt.zeros(2, 3), t)
    with pytest.raises(RuntimeError):
        nt.token_logprobs(z, nt.zeros(2, dtype=nt.int64))
    z.enable_grad()
    lp = nt.token_logprobs(z, t).logprob
    with nt.no_grad():
        z += 1.0
    with pytest.raises(RuntimeError):
        lp.sum().backward()


@pytest.mark.parametrize("op", ["embedding", "dropout", "logprob"])
@pytest.mark.parametrize("N", [20, 700])
def test_gradient_of_another_type(gpu, op, N):
    """Float32 operators under float64 weights: the gradient that arrives is
    float64, what they give is float32, new and added.  The weights are small
    integers, so the cast is exact and the results are those of float32 ones."""
    r = rng(seed_of("type", op, N))
    x = r.standard_normal((N, 12)).astype(np.float32)
    t = r.integers(0, 12, N)
    shape = (N,) if op == "logprob" else (N, 12)
    a = r.integers(-4, 5, shape).astype(np.float32)
    f = {"embedding": lambda X: nt.embedding(X, dev(t)),
         "dropout": lambda X: nt.dropout(X, 0.5, seed=3),
         "logprob": lambda X: nt.token_logprobs(X, dev(t)).logprob}[op]
    grads = []
    for weights in (a, a.astype(np.float64)):
        X = dev(x, True)
        (f(X) * dev(weights)).sum().backward()
        once = host(X.grad).copy()
        (f(X) * dev(weights)).sum().backward()
        grads.append((once, host(X.grad)))
    for got, want in zip(grads[1], grads[0]):
        assert got.dtype == np.float32
        assert_bitexact(got, want)


def test_operators_between_elementwise_ops(gpu):
    """Kernels that may overlap (launched without the stream's barrier) and
    those that may not, each reading what the one before has written."""
    r = rng(61)
    x = r.standard_normal((300, 70)).astype(np.float32)
    t = r.integers(0, 300, 300)
    y, want = dev(x), x
    for k in range(12):
        y = nt.dropout(y, 0.25, seed=k) * 2.0
        want = dropped(want, 0.25, k, 0) * np.float32(2)
        if k % 4 == 3:
            y = nt.embedding(y, dev(t)) * 0.125
            want = want[t] * np.float32(0.125)
    assert_bitexact(host(y), want)


# -------------------------------------------------------------- large tensors


def test_dropout_past_32_bits(gpu):
    n = (1 << 32) + 13
    x = nt.ones(n, device="cuda")
    y = nt.dropout(x, 0.5, seed=3, offset=4)
    for at in (0, (1 << 32) - 8, n - 13):
        part = host(y[at:at + 13])
        i = np.arange(at // 4, at // 4 + 5, dtype=np.uint64)
        w = words_of(i, 3, 4)[at % 4:at % 4 + 13]
        assert_bitexact(part, np.where(w >= np.uint64(1 << 31), np.float32(2), np.float32(0)))


def test_dropout_of_a_view_past_32_bits(gpu):
    m = (1 << 16) + 1
    x = nt.ones(m, m + 63, device="cuda")[:, 5:m + 5]
    y = nt.dropout(x, 0.5, seed=3, offset=4)
    for row in (0, 1, 40000, m - 1):
        i = np.arange(row * m // 4, (row + 1) * m // 4 + 1, dtype=np.uint64)
        w = words_of(i, 3, 4)[row * m % 4:][:m]
        assert_bitexact(host(y[row]), np.where(w >= np.uint64(1 << 31), np.float32(2),
                                               np.float32(0)))


def test_offsets_past_32_bits(gpu):
    """A table and logits of more than 2^32 elements; the last rows."""
    V, D = (1 << 21) + 3, 2049
    w = nt.zeros(V, D, device="cuda")
    w.enable_grad()
    last = np.arange(D, dtype=np.float32)
    with nt.no_grad():
        w[V - 1] = dev(last)
    t = dev(np.array([0, V - 1, V - 1], np.int64))
    y = nt.embedding(w, t, 2.0)
    assert_bitexact(host(y), np.stack([0 * last, 2 * last, 2 * last]))
    dw = y.grad_fn.backward(nt.ones(3, D, device="cuda"))[0]
    assert (host(dw[V - 1]) == 4).all() and (host(dw[V - 2]) == 0).all()
    assert (host(dw[0]) == 2).all() and (host(dw[1]) == 0).all()
    assert float(dw.sum().cpu().item()) == 6 * D
    del w, y, dw
    rows, V = 70000, 65537
    z = nt.zeros(rows, V, device="cuda")
    z.enable_grad()
    out = nt.token_logprobs(z, nt.full(rows, value=V - 1, dtype=nt.int64, device="cuda"), top=1)
    tol = 2.0 ** -24 * (V / 64 + 60)
    assert np.abs(host(out.logprob) + math.log(V)).max() < tol
    assert (host(out.top_tokens) == 0).all()
    dz = out.logprob.grad_fn.backward(nt.ones(rows, device="cuda"))[0]
    row = host(dz[rows - 1])
    assert np.abs(row[:-1] + 1 / V).max() < tol / V and abs(row[-1] - 1 + 1 / V) < 2.0 ** -23
