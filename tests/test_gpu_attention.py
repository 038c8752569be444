"""Attention and its gradients against plain numpy in 64 bits, or in the host's
long double where the operator itself works in 64 bits.

Tolerances.  u is the unit roundoff (2^-24, 2^-53).  A dot product of D terms is
off by at most (D + 8) u of the sum of its terms' magnitudes, the scale's
roundings among them: with A_ij = |scale| sum |q| |k|, a score and the maximum that
it is compared with are off by (D + 8) u A each, and exp doubles neither, so a
probability is off by
    r_i = 2 (D + 8) u (max_j A_ij + 1) + u (n / 4 + 64)
of itself: the sum over n keys runs in 16 lanes at least, and each block of 32
keys rescales it once.  Then, with P = sum p |v|,
    y: r_i P;   dv: sum (2 r_i + (R + 8) u) p |g| over R rows
    g . v - delta: e = (D + 4) u sum |g| |v| + D u sum |g| |y| + r_i sum |g| P
    ds: f = p (2 r_i |g . v - delta| + e + 4 u |g . v - delta|)
    dq: scale sum (f + (n + 8) u |ds|) |k|;  dk: scale sum (f + (R + 8) u |ds|) |q|
and one rounding of the result each.
"""

from __future__ import annotations

import gc

import numpy as np
import pytest

from helpers import assert_bitexact, dev, host, rng, seed_of

import nanotorch_amd as nt
from nanotorch_amd import _lib

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
FLOATS = [np.float32, np.float64]


def visible(B, Tq, Tk, causal, lengths=None, starts=None):
    """[B, Tq, Tk]"""
    n = np.full(B, Tk) if lengths is None else np.clip(np.asarray(lengths), 0, Tk)
    first = n - Tq if starts is None else np.broadcast_to(np.asarray(starts), (B,))
    j = np.arange(Tk)
    see = np.broadcast_to(j < n[:, None, None], (B, Tq, Tk)).copy()
    if causal:
        see &= j <= (first[:, None] + np.arange(Tq))[:, :, None]
    return see


def reference(q, k, v, g, see, scale, u):
    """{name: (value, tolerance)} of y, dq, dk and dv; what a pair that is not
    seen holds is never touched."""
    B, Tq, H, D = q.shape
    G = H // k.shape[2]
    wide = np.longdouble if q.dtype == np.float64 else np.float64
    out = {n: (np.zeros(x.shape, wide), np.zeros(x.shape, wide))
           for n, x in (("y", q), ("dq", q), ("dk", k), ("dv", k))}
    R = Tq * G
    for b in range(B):
        if all(np.isfinite(t[b]).all() for t in ((q, k, v) if g is None else (q, k, v, g))):
            groups = [np.arange(Tq)]  # 0 times what is not seen is 0
        else:
            groups = np.arange(Tq)[:, None]
        for h in range(H):
            for rows in groups:
                on = np.nonzero(see[b, rows].any(0))[0]
                if not on.size:
                    continue
                s = see[b, rows][:, on]
                n = s.sum(1, keepdims=True)
                x, K, V = [t.astype(wide) for t in
                           (q[b, rows, h], k[b, on, h // G], v[b, on, h // G])]
                z = np.where(s, x @ K.T * scale, -np.inf)
                A = np.where(s, np.abs(x) @ np.abs(K).T * abs(scale), 0).max(1, keepdims=True)
                top = z.max(1, keepdims=True)
                p = np.exp(z - np.where(n > 0, top, 0))
                p /= np.where(n > 0, p.sum(1, keepdims=True), 1)
                r = 2 * (D + 8) * u * (A + 1) + u * (n / 4 + 64)
                P = p @ np.abs(V)
                y = p @ V
                out["y"][0][b, rows, h] = y
                out["y"][1][b, rows, h] = r * P + u * np.abs(y)
                if g is None:
                    continue
                go = g[b, rows, h].astype(wide)
                a = np.abs(go)
                d = go @ V.T - (go * y).sum(1, keepdims=True)
                e = ((D + 4) * u * (a @ np.abs(V).T)
                     + (D * u * (a * np.abs(y)).sum(1, keepdims=True)
                        + r * (a * P).sum(1, keepdims=True)))
                ds = p * d
                f = p * (2 * r * np.abs(d) + e + 4 * u * np.abs(d))
                out["dq"][0][b, rows, h] = scale * (ds @ K)
                out["dq"][1][b, rows, h] = abs(scale) * (
                    (f + (n + 8) * u * np.abs(ds)) @ np.abs(K))
                out["dk"][0][b, on, h // G] += scale * (ds.T @ x)
                out["dk"][1][b, on, h // G] += abs(scale) * (
                    (f + (R + 8) * u * np.abs(ds)).T @ np.abs(x))
                out["dv"][0][b, on, h // G] += p.T @ go
                out["dv"][1][b, on, h // G] += ((2 * r + (R + 8) * u) * p).T @ a
    for value, tol in list(out.values())[1:]:
        tol += u * np.abs(value)
    return out


def check(got, want, what):
    value, tol = want
    got = got.astype(value.dtype)
    assert got.shape == value.shape
    err = np.abs(got - value)
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.size,
                           float(np.nanmax(err / np.maximum(tol, 1e-300))))


def inputs(r, B, Tq, Tk, H, Hk, D, dtype, sharp=1.0):
    q = (r.standard_normal((B, Tq, H, D)) * sharp).astype(dtype)
    k, v = [r.standard_normal((B, Tk, Hk, D)).astype(dtype) for _ in range(2)]
    g = (r.standard_normal((B, Tq, H, D)) * 0.1).astype(dtype)
    return q, k, v, g


def run(q, k, v, g=None, **kw):
    """(y, [dq, dk, dv]) on the device."""
    track = g is not None
    q, k, v = [dev(x, track) if isinstance(x, np.ndarray) else x for x in (q, k, v)]
    for t in (q, k, v):
        if track:
            t.enable_grad()
    y = nt.attention(q, k, v, **kw)
    if not track:
        return host(y), None
    return host(y), [host(t) for t in y.grad_fn.backward(dev(g))[:3]]


def check_all(q, k, v, g, see, dtype, scale=None, **kw):
    D = q.shape[-1]
    want = reference(q, k, v, g, see, D ** -0.5 if scale is None else scale, U[dtype])
    y, grads = run(q, k, v, g, scale=scale, **kw)
    check(y, want["y"], "y")
    if grads is not None:
        for name, x in zip(("dq", "dk", "dv"), grads):
            check(x, want[name], name)


SHAPES = [  # B, Tq, Tk, H, Hk, D
    (1, 1, 1, 1, 1, 1), (2, 5, 5, 2, 1, 3), (1, 16, 16, 1, 1, 16), (1, 17, 33, 2, 2, 64),
    (2, 31, 31, 4, 2, 40), (1, 64, 64, 2, 1, 128), (1, 65, 130, 3, 3, 80), (1, 20, 20, 6, 2, 256),
    (3, 1, 70, 8, 2, 32), (1, 3, 300, 5, 1, 65), (1, 130, 7, 2, 2, 31), (1, 40, 40, 1, 1, 129),
    (2, 4, 4, 33, 3, 7), (1, 48, 200, 2, 2, 96),
]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(gpu, shape, causal, dtype):
    B, Tq, Tk, H, Hk, D = shape
    r = rng(seed_of("attn", shape, causal, dtype.__name__))
    q, k, v, g = inputs(r, *shape, dtype, sharp=3.0 if D > 30 else 1.0)
    check_all(q, k, v, g, visible(B, Tq, Tk, causal), dtype, causal=causal)


LARGE = [  # as many products as the half-precision planes are used for
    (1, 1100, 1100, 6, 3, 128), (2, 1030, 1470, 6, 3, 96), (2, 1600, 1601, 3, 3, 33),
    (3, 657, 1640, 2, 1, 80), (1, 70, 9001, 8, 1, 100), (1, 3333, 330, 4, 1, 96),
    (9, 777, 777, 2, 2, 64), (1, 1777, 1777, 4, 4, 32),
    (1, 1300, 1200, 2, 1, 160), (1, 900, 1150, 4, 2, 190), (2, 700, 700, 3, 3, 256),
    (1, 140, 5000, 6, 1, 131),
    # the backward pass alone
    (1, 20, 9049, 8, 1, 96), (1, 520, 520, 8, 4, 64), (8, 1, 4100, 40, 4, 32),
    (2, 300, 470, 6, 6, 128), (1, 1300, 1300, 2, 2, 40),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", LARGE)
def test_large(gpu, shape, causal):
    B, Tq, Tk, H, Hk, D = shape
    r = rng(seed_of("large", shape, causal))
    q, k, v, g = inputs(r, *shape, np.float32, sharp=2.0)
    check_all(q, k, v, g, visible(B, Tq, Tk, causal), np.float32, causal=causal)


@pytest.mark.parametrize("causal,starts", [(False, None), (True, None), (True, 0),
                                           (True, [5, -1700, 1000, 64, 0])])
def test_large_lengths_and_starts(gpu, causal, starts):
    B, Tq, Tk, H, Hk, D = 5, 1130, 1150, 2, 1, 64
    lengths = np.array([1150, 0, 1, 593, 1100])
    r = rng(seed_of("large len", causal, str(starts)))
    q, k, v, g = inputs(r, B, Tq, Tk, H, Hk, D, np.float32)
    for b, n in enumerate(lengths):
        k[b, n:] = np.nan
        v[b, n:] = np.inf
    see = visible(B, Tq, Tk, causal, lengths, starts)
    given = dev(np.array(starts)) if isinstance(starts, list) else starts
    check_all(q, k, v, g, see, np.float32, causal=causal, lengths=dev(lengths), starts=given)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e15])
@pytest.mark.parametrize("what", ["v", "g", "qk"])
def test_large_of_any_magnitude(gpu, what, size):
    """Values far from 1, and rows of gradients of very different sizes: nothing
    is lost to the range of half precision."""
    r = rng(seed_of("magnitude", what, size))
    q, k, v, g = inputs(r, 1, 1820, 1820, 2, 1, 64, np.float32)
    if what == "v":
        v *= np.float32(size)
    elif what == "g":
        g *= np.float32(size)
        g *= (10.0 ** r.uniform(-6, 6, (1, 1820, 1, 1))).astype(np.float32)
        g[0, ::7] = 0
    else:
        q *= np.float32(size)
        k /= np.float32(size)
    check_all(q, k, v, g, visible(1, 1820, 1820, True), np.float32, causal=True)


@pytest.mark.parametrize("what,D", [("k", 64), ("v", 64), ("q", 64), ("k", 256), ("v", 200),
                                    ("q", 132)])
def test_large_with_an_outlier(gpu, what, D):
    """One row 2^13 times and more above its neighbours, where most rows do not
    see it: the others keep their bits."""
    r = rng(seed_of("outlier", what))
    T = 1820
    q, k, v, g = inputs(r, 1, T, T, 2, 1, D, np.float32)
    see = visible(1, T, T, True)
    clean = reference(q, k, v, g, see, D ** -0.5, U[np.float32])
    x = {"q": q, "k": k, "v": v}[what]
    at = T - 20
    x[0, at] *= np.float32(1e12)
    y, (dq, dk, dv) = run(q, k, v, g, causal=True)
    if what == "q":
        keep = np.arange(T) != at
        check(y[:, keep], [t[:, keep] for t in clean["y"]], "y")
        check(dq[:, keep], [t[:, keep] for t in clean["dq"]], "dq")
    else:
        check(y[:, :at], [t[:, :at] for t in clean["y"]], "y")
        check(dq[:, :at], [t[:, :at] for t in clean["dq"]], "dq")


@pytest.mark.parametrize("T,D", [(1820, 64), (1300, 128), (1200, 160)])
@pytest.mark.parametrize("power", [10, 17, 20, 24, 28, 32, 40])
@pytest.mark.parametrize("what", ["v", "g", "q up", "k up"])
def test_large_with_a_column_apart(gpu, what, power, T, D):
    """One column far above the others, which keep their bits: the columns of a
    result are no concern of one another's.  Queries and keys are scaled against
    each other, so that scores stay as they are."""
    r = rng(seed_of("column", what, power, D))
    q, k, v, g = inputs(r, 1, T, T, 2, 1, D, np.float32)
    by = np.float32(2.0 ** power)
    if what == "v":
        v[..., 5] *= by
        g[..., 5] /= by
    elif what == "g":
        g[..., 5] *= by
        v[..., 5] /= by
    else:
        q[..., 5] *= by if what == "q up" else 1 / by
        k[..., 5] *= 1 / by if what == "q up" else by
    check_all(q, k, v, g, visible(1, T, T, True), np.float32, causal=True)


@pytest.mark.parametrize("power", [15, 25, 33])
@pytest.mark.parametrize("what", ["v", "k", "q", "g"])
def test_large_elements_in_every_row_and_column(gpu, what, power):
    """Rows are alike and columns are alike, but no row has all the large values that
    its columns have: rows that do not see a column's large ones keep their bits."""
    r = rng(seed_of("diagonal", what, power))
    T, D = 1820, 64
    q, k, v, g = inputs(r, 1, T, T, 2, 1, D, np.float32, sharp=0.5)
    x = {"q": q, "k": k, "v": v, "g": g}[what]
    other = {"q": k, "k": q}.get(what)
    at = np.arange(T)
    if other is not None:  # no score is large: the other side has zeros there
        some = r.integers(0, D // 2, T)
        other[..., :D // 2] = 0
        x[0, at, :, some] *= np.float32(2.0 ** power)
    else:
        x[0, at, :, at % D] *= np.float32(2.0 ** power)
    check_all(q, k, v, g, visible(1, T, T, True), np.float32, causal=True)


@pytest.mark.parametrize("small", [1.0, 2.0 ** -80])
def test_large_with_small_probabilities(gpu, small):
    """Keys that no query cares for, with columns of values of their own: what is e^-30
    beside the rest is all that those columns have.  With gradients so small that
    probability times gradient is next to float32's smallest number."""
    r = rng(seed_of("tail"))
    T, D = 1820, 64
    q, k, v, g = inputs(r, 1, T, T, 2, 1, D, np.float32, sharp=0.2)
    q[..., 0] = 10.0
    k[..., 0] = 12.0
    some = np.zeros(T, bool)
    some[1728:1792] = True  # behind others
    k[:, some, :, 0] = -12.0
    v[:, ~some, :, :8] = 0
    g *= np.float32(small)
    check_all(q, k, v, g, visible(1, T, T, False), np.float32)


def test_large_values_with_small_gradients(gpu):
    """Values of 2^110 and their gradients of 2^-66: nothing passes float32's range that
    the results do not pass."""
    r = rng(seed_of("range"))
    T, D = 1820, 64
    q, k, v, g = inputs(r, 1, T, T, 2, 1, D, np.float32)
    v *= np.float32(2.0 ** 110)
    g *= np.float32(2.0 ** -66)
    check_all(q, k, v, g, visible(1, T, T, True), np.float32, causal=True)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("wide", [np.int32, np.int64])
@pytest.mark.parametrize("causal,starts", [(False, None), (True, None), (True, 0), (True, -3),
                                           (True, [2, -50, 4, 40, 0, 2**40])])
def test_lengths_and_starts(gpu, causal, starts, wide, dtype):
    """Rows that see nothing, sequences of no and of one token, starts of any
    size; what lies behind a sequence is not a number."""
    B, Tq, Tk, H, Hk, D = 6, 21, 45, 4, 2, 20
    if isinstance(starts, list) and wide is np.int32:
        starts = starts[:-1] + [2**31 - 1]
    lengths = np.array([45, 0, 1, 16, 33, 20])
    r = rng(seed_of("len", causal, str(starts), dtype.__name__))
    q, k, v, g = inputs(r, B, Tq, Tk, H, Hk, D, dtype)
    for b, n in enumerate(lengths):
        k[b, n:] = np.nan
        v[b, n:] = np.inf
    see = visible(B, Tq, Tk, causal, lengths, starts)
    given = dev(np.array(starts, wide)) if isinstance(starts, list) else starts
    check_all(q, k, v, g, see, dtype, causal=causal, lengths=dev(lengths.astype(wide)),
              starts=given)
    y, (dq, dk, dv) = run(q, k, v, g, causal=causal, lengths=dev(lengths.astype(wide)),
                          starts=given)
    none = ~see.any(2)
    assert (y[none] == 0).all() and (dq[none] == 0).all()
    unseen = ~see.any(1)
    assert (dk[unseen] == 0).all() and (dv[unseen] == 0).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("T,D,dtype", [(37, 24, np.float32), (37, 24, np.float64),
                                       (150, 64, np.float32), (150, 64, np.float64),
                                       (1860, 64, np.float32), (90, 90, np.float64),
                                       (70, 201, np.float64)])
def test_what_is_not_seen_does_not_matter(gpu, dtype, bad, T, D):
    """A key, value, query or gradient that is no number reaches the rows that
    see it and no other."""
    r = rng(seed_of("hidden", str(bad), T, dtype.__name__))
    q, k, v, g = inputs(r, 1, T, T, 2, 1, D, dtype)
    see = visible(1, T, T, True)
    at = T // 2 + 3
    clean = reference(q, k, v, g, see, D ** -0.5, U[dtype])
    for what in "kv":
        x = {"k": k.copy(), "v": v.copy()}
        x[what][0, at, 0, 1] = bad
        y, (dq, _, _) = run(q, x["k"], x["v"], g, causal=True)
        check(y[:, :at], [t[:, :at] for t in clean["y"]], "y before " + what)
        check(dq[:, :at], [t[:, :at] for t in clean["dq"]], "dq before " + what)
    for what in "qg":
        x = {"q": q.copy(), "g": g.copy()}
        x[what][0, at, 1, 1] = bad
        _, (_, dk, dv) = run(x["q"], k, v, x["g"], causal=True)
        for name, got in (("dk", dk), ("dv", dv)):
            check(got[:, at + 1:], [t[:, at + 1:] for t in clean[name]], f"{name} after {what}")


@pytest.mark.parametrize("causal", [False, True])
def test_long_rows_of_few_queries(gpu, causal):
    """Keys split over workgroups, as for an answer's token over a long cache."""
    B, Tq, Tk, H, Hk, D = 2, 2, 9001, 6, 2, 64
    r = rng(seed_of("long", causal))
    q, k, v, _ = inputs(r, B, Tq, Tk, H, Hk, D, np.float32, sharp=2.0)
    lengths = np.array([9001, 5003])
    see = visible(B, Tq, Tk, causal, lengths)
    check_all(q, k, v, None, see, np.float32, causal=causal, lengths=dev(lengths))


@pytest.mark.parametrize("Tq,Tk,H,Hk,D", [(2, 2500, 6, 2, 100), (1, 3001, 4, 4, 256),
                                          (5, 1111, 33, 1, 65), (300, 290, 4, 2, 128),
                                          (150, 170, 3, 3, 250)])
@pytest.mark.parametrize("causal", [False, True])
def test_wide_rows_in_64_bits(gpu, Tq, Tk, H, Hk, D, causal):
    """Split keys, lengths that leave tiles of no row and of one, values that are
    no numbers behind them."""
    r = rng(seed_of("wide", Tq, Tk, D, causal))
    q, k, v, g = inputs(r, 3, Tq, Tk, H, Hk, D, np.float64, sharp=2.0)
    lengths = np.array([Tk, 0, Tk // 2 + 1])
    for b, n in enumerate(lengths):
        k[b, n:] = np.nan
        v[b, n:] = np.inf
    see = visible(3, Tq, Tk, causal, lengths)
    check_all(q, k, v, g, see, np.float64, causal=causal, lengths=dev(lengths))


def test_a_cache_longer_than_32_bits(gpu):
    """Keys and values whose elements pass 2^32: views of one row, repeated."""
    Tk, D = 40, 64
    r = rng(3)
    q, k, v, _ = inputs(r, 1, 1, Tk, 1, 1, D, np.float32)
    step = 2**32 // (Tk - 1) // 64 * 64 + 64
    buf = nt.zeros((Tk - 1) * step + D, device="cuda")
    for j in range(Tk):
        buf[j * step:j * step + D] = dev(k[0, j, 0])
    K = nt.Tensor._new_view(buf.storage, (1, Tk, 1, D), (0, step, D, 1), 0)
    y, _ = run(q, K, K)
    want = reference(q, k, k, None, visible(1, 1, Tk, False), D ** -0.5, U[np.float32])
    check(y, want["y"], "y")


@pytest.mark.parametrize("dtype", FLOATS)
def test_views(gpu, dtype):
    """Heads before tokens, every second token, offsets of one element, shared
    (stride 0) keys: the same values as from contiguous tensors."""
    B, Tq, Tk, H, Hk, D = 2, 19, 22, 4, 2, 36
    r = rng(seed_of("views", dtype.__name__))
    q, k, v, g = inputs(r, B, Tq, Tk, H, Hk, D, dtype)
    want, grads = run(q, k, v, g, causal=True)

    def heads_first(x):
        return dev(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).transpose(1, 2)

    def second(x):
        wide = np.zeros((x.shape[0], 2 * x.shape[1]) + x.shape[2:], dtype)
        wide[:, ::2] = x
        return dev(wide)[:, ::2]

    def shifted(x):
        flat = dev(np.concatenate([np.zeros(1, dtype), x.reshape(-1)]))
        return flat[1:].reshape(*x.shape) if False else nt.Tensor._new_view(
            flat.storage, x.shape, None, 1)

    def inner(x):  # elements of a head not adjacent: copied
        return dev(np.ascontiguousarray(np.swapaxes(x, 2, 3))).transpose(2, 3)

    ref = reference(q, k, v, g, visible(B, Tq, Tk, True), D ** -0.5, U[dtype])
    for how in (heads_first, second, shifted, inner):
        y, got = run(how(q), how(k), how(v), g, causal=True)
        check(y, ref["y"], how.__name__)
        for name, x in zip(("dq", "dk", "dv"), got):
            check(x, ref[name], how.__name__ + name)
    Q = dev(q, True)
    y = nt.attention(Q, dev(k), dev(v), causal=True)
    dq = y.grad_fn.backward(heads_first(g))[0]
    check(host(dq), ref["dq"], "g of heads first")
    assert_bitexact(want, host(nt.attention(dev(q), dev(k), dev(v), causal=True)))
    one = dev(k[:1], True).expand(B, Tk, Hk, D)
    y2, _ = run(q, one, one)
    check(y2, reference(q, np.repeat(k[:1], B, 0), np.repeat(k[:1], B, 0), None,
                        visible(B, Tq, Tk, False), D ** -0.5, U[dtype])["y"], "expanded")


def test_large_views(gpu):
    """Queries, keys and values as parts of one projection's output, a gradient with
    heads before tokens, and one head's keys for all: the half-precision planes'
    kernels read them in place."""
    B, T, H, D = 2, 1180, 3, 64
    r = rng(seed_of("large views"))
    x = (r.standard_normal((B, T, 3 * H, D)) * 1.5).astype(np.float32)
    g = (r.standard_normal((B, T, H, D)) * 0.1).astype(np.float32)
    q, k, v = [np.ascontiguousarray(x[:, :, i * H:(i + 1) * H]) for i in range(3)]
    X = dev(x)
    parts = [X[:, :, i * H:(i + 1) * H] for i in range(3)]
    for p in parts:
        p.enable_grad()
    y = nt.attention(*parts, causal=True)
    G = dev(np.ascontiguousarray(g.transpose(0, 2, 1, 3))).transpose(1, 2)
    want = reference(q, k, v, g, visible(B, T, T, True), D ** -0.5, U[np.float32])
    check(host(y), want["y"], "y")
    for name, t in zip(("dq", "dk", "dv"), y.grad_fn.backward(G)[:3]):
        check(host(t), want[name], name)
    one = dev(k[:, :, :1]).expand(B, T, H, D)
    same = np.repeat(k[:, :, :1], H, 2)
    got, _ = run(q, one, one)
    check(got, reference(q, same, same, None, visible(B, T, T, False), D ** -0.5,
                         U[np.float32])["y"], "expanded")


@pytest.mark.parametrize("scale", [-0.7, 1.0, 1e-20])
def test_large_scales(gpu, scale):
    r = rng(seed_of("large scale"))
    q, k, v, g = inputs(r, 2, 1200, 1200, 2, 2, 64, np.float32, sharp=0.5)
    check_all(q, k, v, g, visible(2, 1200, 1200, True), np.float32, scale=scale, causal=True)


@pytest.mark.parametrize("T,H", [(33, 2), (1250, 2)])  # of either kind of kernels
def test_one_tensor_as_queries_keys_and_values(gpu, T, H):
    r = rng(seed_of("one tensor", T))
    x = r.standard_normal((2, T, H, 64)).astype(np.float32)
    g = (r.standard_normal(x.shape) * 0.1).astype(np.float32)
    X = dev(x, True)
    y = nt.attention(X, X, X, causal=True)
    (y * dev(g)).sum().backward()
    want = reference(x, x, x, g, visible(2, T, T, True), 64 ** -0.5, U[np.float32])
    check(host(y), want["y"], "y")
    value, tol = [sum(want[n][i] for n in ("dq", "dk", "dv")) for i in range(2)]
    # three roundings of sums of them
    tol = tol + 3 * U[np.float32] * sum(np.abs(want[n][0]) for n in ("dq", "dk", "dv"))
    check(host(X.grad), (value, tol), "dx")


def test_results_repeat(gpu):
    r = rng(8)
    for T, D in ((50, 48), (1400, 64), (1200, 128)):
        q, k, v, g = inputs(r, 2, T, T, 4, 2, D, np.float32)
        y, grads = run(q, k, v, g, causal=True)
        y2, grads2 = run(q, k, v, g, causal=True)
        assert_bitexact(y, y2)
        for a, b in zip(grads, grads2):
            assert_bitexact(a, b)


def test_scale_and_no_batch(gpu):
    r = rng(5)
    q, k, v, g = inputs(r, 1, 12, 18, 2, 2, 8, np.float32)
    for scale in (0.0, 1.0, -0.7):
        want = reference(q, k, v, g, visible(1, 12, 18, False), 0.0, 0.0) if scale == 0 else None
        y, grads = run(q, k, v, g, scale=scale)
        flat = nt.attention(dev(q[0], True), dev(k[0]), dev(v[0]), scale=scale)
        assert flat.shape == (12, 2, 8)
        assert_bitexact(host(flat), y[0])
        assert_bitexact(host(flat.grad_fn.backward(dev(g[0]))[0]), grads[0][0])
        if scale == 0:
            assert (grads[0] == 0).all() and (grads[1] == 0).all()
            assert np.abs(y - want["y"][0]).max() < 18 * 2.0 ** -24 * 4
    check_all(q, k, v, g, visible(1, 12, 18, False), np.float32, scale=0.9)


@pytest.mark.parametrize("dtype,bad", [(nt.float32, 1e39), (nt.float32, np.nan),
                                       (nt.float64, np.inf), (nt.float64, -2.0 ** 1023)])
def test_an_abi_call_refuses_scales(gpu, dtype, bad):
    view = _lib.pack_view(0, 0, dtype, (1, 0, 1, 4), (4, 4, 4, 1))
    for name, args in (("nt_attention", (view, None)),
                       ("nt_attention_bwd", (view, view, view, None, None, None))):
        with pytest.raises(ValueError, match="scale must be finite"):
            _lib.call_packed(name, view, view, view, None, None, 0, 0, bad, *args)


@pytest.mark.parametrize("shape", [(0, 4, 4), (2, 0, 5), (2, 5, 0)])
def test_empty(gpu, shape):
    B, Tq, Tk = shape
    q, k = dev(np.ones((B, Tq, 2, 8), np.float32), True), dev(np.ones((B, Tk, 1, 8), np.float32),
                                                              True)
    y = nt.attention(q, k, k, causal=True)
    assert y.shape == q.shape
    dq, dk, dv = y.grad_fn.backward(dev(np.ones(q.shape, np.float32)))[:3]
    assert dq.shape == q.shape and dk.shape == k.shape
    for t in (y, dq, dk, dv):
        assert (host(t) == 0).all()


def test_through_the_engine(gpu):
    """Accumulation into existing gradients, one tensor as query, key and value,
    and gradients of expanded keys, against differences."""
    r = rng(11)
    x = r.standard_normal((1, 6, 2, 4))

    def loss(a):
        t = dev(a, True)
        y = nt.attention(t, t, t, causal=True)
        return t, (y * y).sum()

    t, out = loss(x)
    out.backward()
    got = host(t.grad)
    for at in ((0, 0, 0, 0), (0, 3, 1, 2), (0, 5, 0, 3)):
        d = np.zeros_like(x)
        d[at] = 1e-6
        slope = (host(loss(x + d)[1]) - host(loss(x - d)[1])) / 2e-6
        assert abs(slope - got[at]) < 1e-7 * max(1, abs(got[at])), (at, slope, got[at])
    y = nt.attention(t, t, t, causal=True)  # a second backward adds
    (y * y).sum().backward()
    np.testing.assert_allclose(host(t.grad), 2 * got, rtol=1e-12, atol=1e-12)

    k = dev(r.standard_normal((1, 5, 1, 4)), True)
    q = dev(r.standard_normal((3, 6, 2, 4)))
    wide = k.expand(3, 5, 1, 4)
    nt.attention(q, wide, wide).sum().backward()
    kk = dev(np.repeat(host(k), 3, 0), True)
    nt.attention(q, kk, kk).sum().backward()
    np.testing.assert_allclose(host(k.grad), host(kk.grad).sum(0, keepdims=True), rtol=1e-12,
                               atol=1e-13)


def test_in_place_changes_are_caught(gpu):
    q, k, v = [dev(np.ones((1, 4, 1, 4), np.float32), True) for _ in range(3)]
    y = nt.attention(q, k, v).sum()
    with nt.no_grad():
        k += 1.0
    with pytest.raises(RuntimeError, match="modified inplace"):
        y.backward()


@pytest.mark.parametrize("T", [1, 4000])  # of either kind of kernels
def test_a_length_outside_is_reported(gpu, T):
    q = dev(np.ones((2, T, 1, 4), np.float32))
    k = dev(np.ones((2, 6 * T, 1, 4), np.float32))
    for bad in ([6 * T + 1, 3], [3, -1]):
        y = nt.attention(q, k, k, lengths=dev(np.array(bad)))
        with pytest.raises(IndexError):
            nt.sync()
        got = host(y)
        assert (got[[b < 0 for b in bad]] == 0).all()
        assert (got[[b >= 0 for b in bad]] == 1).all()


def test_more_sequences_than_one_launch_holds(gpu):
    """Over 2^21 tiles of 16 rows: taken some sequences at a time, each as alone."""
    B, T, H, D = 42000, 100, 8, 4
    nt.manual_seed(4)
    q, k, v = [nt.rand(B, T, H, D, device="cuda") for _ in range(3)]
    lengths = dev(np.arange(B) % (T + 1))
    for t in (q, k, v):
        t.enable_grad()
    y = nt.attention(q, k, v, causal=True, lengths=lengths, starts=0)
    grads = y.grad_fn.backward(v)[:3]
    for beg in (0, 37000, 37440, B - 50):  # about the border and at the ends
        some = slice(beg, beg + 50)
        parts = [dev(host(t[some]), True) for t in (q, k, v)]
        y1 = nt.attention(*parts, causal=True, lengths=lengths[some], starts=0)
        assert_bitexact(host(y[some]), host(y1))
        want = reference(*[host(t) for t in parts], host(parts[2]),
                         visible(50, T, T, True, host(lengths[some]), 0), 0.5, U[np.float32])
        for name, got in zip(("dq", "dk", "dv"), grads):
            check(host(got[some]), want[name], name)


def test_no_memory_is_kept_by_a_cycle(gpu):
    q = dev(np.ones((1, 64, 4, 64), np.float32), True)
    gc.collect()
    gc.disable()
    try:
        refs = []
        for _ in range(3):
            y = nt.attention(q, q, q)
            import weakref
            refs.append(weakref.ref(y.storage))
            del y
        assert all(w() is None for w in refs)
    finally:
        gc.enable()
