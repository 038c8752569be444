"""The root-mean-square norm with a residual, and its gradients, against plain
numpy in 64 bits (long double for float64).

Tolerances, u the unit roundoff.  A lane adds at most 32 squares, then 6 + 16
partial sums, and D / 1024 more where a row outgrows the registers: the mean is
off by (60 + D / 1024) u of itself, its root's inverse by half of that and 3 u,
so y by (40 + D / 2048) u |y|, the sum x + residual's own rounding within it.
    ds: (70 + D / 512) u r (|g w| + |n| mean |g w n|) + 2 u (|gs| + |ds|)
    dw: (rows + 80 + D / 1024) u sum |g n|
"""

from __future__ import annotations

import gc
import weakref

import numpy as np
import pytest

from helpers import assert_bitexact, dev, host, rng, seed_of

import nanotorch_amd as nt
from nanotorch_amd import nn

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
FLOATS = [np.float32, np.float64]
EPS = 1e-6


def reference(x, w, residual, g, gs, u):
    wide = np.longdouble if x.dtype == np.float64 else np.float64
    s = x + residual if residual is not None else x  # in x's own type
    S, D = s.astype(wide), x.shape[-1]
    W = np.ones(D, wide) if w is None else w.astype(wide)
    r = 1 / np.sqrt((S * S).mean(-1, keepdims=True) + EPS)
    n = S * r
    y = n * W
    out = {"s": (s, 0), "y": (y, (40 + D / 2048) * u * np.abs(y))}
    if g is None:
        return out
    gw = g.astype(wide) * W
    ds = r * (gw - n * (gw * n).mean(-1, keepdims=True))
    tol = (70 + D / 512) * u * r * (np.abs(gw) + np.abs(n) * np.abs(gw * n).mean(-1,
                                                                                keepdims=True))
    if gs is not None:
        ds = ds + gs
        tol = tol + 2 * u * np.abs(gs)
    rows = x.size // D
    gn = (g.astype(wide) * n).reshape(rows, D)
    out["ds"] = (ds, tol + 2 * u * np.abs(ds))
    out["dw"] = (gn.sum(0), (rows + 80 + D / 1024) * u * np.abs(gn).sum(0))
    return out


def check(got, want, what):
    value, tol = want
    err = np.abs(got.astype(np.longdouble) - value)
    bad = ~(err <= tol)
    assert got.shape == value.shape and not bad.any(), (
        what, int(bad.sum()), float(np.nanmax(err / np.maximum(tol, 1e-300))))


def data(r, shape, dtype):
    x, res, g, gs = [(r.standard_normal(shape) * m).astype(dtype) for m in (1.0, 3.0, 1.0, 1.0)]
    return x, (1 + 0.3 * r.standard_normal(shape[-1])).astype(dtype), res, g, gs


SHAPES = [(1, 1), (3, 5), (1000, 3), (64, 256), (5, 257), (7, 511), (300, 513), (33, 1024),
          (9, 1023), (1030, 2047), (6, 2049), (12, 4096), (5, 4099), (3, 8192), (4, 8193),
          (2, 16384), (3, 16385), (2, 40001), (70, 17000)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rms_norm(gpu, shape, weighted, residual, dtype):
    r = rng(seed_of("norm", shape, dtype.__name__))
    x, w, res, g, gs = data(r, shape, dtype)
    w, res = w if weighted else None, res if residual else None
    want = reference(x, w, res, g, gs if residual else None, U[dtype])
    X = dev(x, True)
    args = (X, None if w is None else dev(w, True))
    if not residual:
        y = nt.rms_norm(*args, eps=EPS)
        grads = y.grad_fn.backward(dev(g))
    else:
        y, s = nt.rms_norm(*args, residual=dev(res, True), eps=EPS)
        assert_bitexact(host(s), want["s"][0])
        grads = y.grad_fn.inputs[0].grad_fn.backward(dev(np.stack([g, gs])))
        check(host(grads[-1]), want["ds"], "dresidual")
    check(host(y), want["y"], "y")
    check(host(grads[0]), want["ds"], "dx")
    if weighted:
        check(host(grads[1]), want["dw"], "dw")


@pytest.mark.parametrize("dtype", FLOATS)
def test_through_the_engine(gpu, dtype):
    """Both results in one loss, either alone, and a chain of blocks; added to
    what is there."""
    shape = (11, 50)
    r = rng(seed_of("engine", dtype.__name__))
    x, w, res, g, gs = data(r, shape, dtype)
    for use in ("both", "y", "s"):
        X, W, R = dev(x, True), dev(w, True), dev(res, True)
        for turn in (1, 2):
            y, s = nt.rms_norm(X, W, residual=R, eps=EPS)
            total = (y * dev(g)).sum() if use != "s" else None
            if use != "y":
                more = (s * dev(gs)).sum()
                total = more if total is None else total + more
            total.backward()
            want = reference(x, w, res, g if use != "s" else np.zeros_like(g),
                             gs if use != "y" else np.zeros_like(g), U[dtype])
            for t, name in ((X, "ds"), (R, "ds"), (W, "dw")):
                value, tol = want[name]
                check(host(t.grad), (turn * value, turn * (tol + 1e-30) + U[dtype] *
                                     np.abs(value) * turn), (use, name))
        X._grad *= 2.0  # leaves' gradients are their own
        check(host(R.grad), (2 * want["ds"][0], 2 * want["ds"][1] + 1e-30 +
                             2 * U[dtype] * np.abs(want["ds"][0])), "alone")


def test_gradients_shared_by_inner_tensors(gpu):
    """x and the residual get one gradient; what is added to one of them later
    does not reach the other."""
    r = rng(4)
    a, b = [dev(r.standard_normal((5, 8)), True) for _ in range(2)]
    x, h = a * 1.0, b * 1.0
    y, s = nt.rms_norm(x, residual=h)
    ((y * y * y).sum() + (s * s).sum() + (x * x * x).sum() * 5.0).backward()
    da, db = host(a.grad), host(b.grad)
    np.testing.assert_allclose(da - db, 15 * host(a) ** 2, rtol=1e-12, atol=1e-12)


def test_gradients_shared_beside_a_trained_weight(gpu):
    """As above, with a weight that is a leaf."""
    r = rng(14)
    a, b = [dev(r.standard_normal((5, 8)), True) for _ in range(2)]
    w = dev(1 + 0.1 * r.standard_normal(8), True)
    x, h = a * 1.0, b * 1.0
    y, s = nt.rms_norm(x, w, residual=h)
    ((y * y * y).sum() + (s * s).sum() + (x * x * x).sum() * 5.0).backward()
    da, db = host(a.grad), host(b.grad)
    np.testing.assert_allclose(da - db, 15 * host(a) ** 2, rtol=1e-12, atol=1e-12)
    X, R = host(a), host(b)
    y0 = reference(X, host(w), R, None, None, U[np.float64])["y"][0]
    want = reference(X, host(w), R, 3 * y0 ** 2, 2 * (X + R), U[np.float64])
    np.testing.assert_allclose(db, want["ds"][0].astype(np.float64), rtol=1e-11, atol=1e-12)
    np.testing.assert_allclose(host(w.grad), want["dw"][0].astype(np.float64), rtol=1e-11,
                               atol=1e-12)


def test_same_tensor_twice(gpu):
    r = rng(6)
    x = r.standard_normal((3, 9))
    X = dev(x, True)
    y, s = nt.rms_norm(X, residual=X)
    (y.sum() + s.sum() * 0.5).backward()
    want = reference(x, None, x, np.ones_like(x), np.full_like(x, 0.5), U[np.float64])["ds"]
    check(host(X.grad), (2 * want[0], 4 * want[1]), "dx")


def test_views_and_shapes(gpu):
    r = rng(7)
    x, w, res, g, _ = data(r, (4, 6, 40), np.float32)
    want = reference(x, w, res, g, np.zeros_like(g), U[np.float32])
    X = dev(np.ascontiguousarray(x.transpose(1, 0, 2)), True).transpose(0, 1)
    R = dev(np.ascontiguousarray(res.transpose(2, 0, 1)))
    R = R.transpose(0, 1).transpose(1, 2)
    y, s = nt.rms_norm(X, dev(w), residual=R, eps=EPS)
    assert y.shape == s.shape == x.shape
    check(host(y), want["y"], "y")
    wide = np.zeros((24, 100), np.float32)
    wide[:, 7:47] = x.reshape(24, 40)
    check(host(nt.rms_norm(dev(wide)[:, 7:47], dev(w), eps=EPS)),
          [t.reshape(24, 40) for t in reference(x, w, None, None, None, U[np.float32])["y"]],
          "columns")
    one = nt.rms_norm(dev(x[0, 0]), eps=EPS)
    assert one.shape == (40,)
    check(host(one), reference(x[0, 0], None, None, None, None, U[np.float32])["y"], "a vector")
    same = dev(x[0, :1]).expand(6, 40)
    check(host(nt.rms_norm(same, eps=EPS)),
          reference(np.repeat(x[0, :1], 6, 0), None, None, None, None, U[np.float32])["y"], "rows")


def test_zeros_and_not_numbers(gpu):
    x = np.zeros((3, 300), np.float32)
    x[1, 5], x[2, 7] = np.nan, np.inf
    y = host(nt.rms_norm(dev(x)))
    assert (y[0] == 0).all() and np.isnan(y[1]).all()
    assert (y[2][:7] == 0).all() and np.isnan(y[2, 7])
    for rows, D in ((0, 5), (0, 20000)):
        X, W = dev(np.zeros((rows, D), np.float32), True), dev(np.ones(D, np.float32), True)
        y = nt.rms_norm(X, W)
        dx, dw = y.grad_fn.backward(dev(np.zeros((rows, D), np.float32)))
        assert host(dx).shape == (rows, D) and (host(dw) == 0).all()


def test_results_repeat_and_changes_are_caught(gpu):
    r = rng(9)
    x, w, res, g, gs = data(r, (5000, 300), np.float32)
    X, W, G = dev(x, True), dev(w, True), dev(g)
    y = nt.rms_norm(X, W)
    first = [host(t) for t in y.grad_fn.backward(G)]
    for a, b in zip(first, y.grad_fn.backward(G)):
        assert_bitexact(host(b), a)
    with nt.no_grad():
        X += 1.0
    with pytest.raises(RuntimeError, match="modified inplace"):
        y.grad_fn.backward(G)
    y, s = nt.rms_norm(X, W, residual=dev(res))
    with nt.no_grad():
        y += 1.0  # the sum is what the gradient needs
    (s.sum() + y.sum()).backward()
    y, s = nt.rms_norm(X, W, residual=dev(res))
    with nt.no_grad():
        s += 1.0
    with pytest.raises(RuntimeError, match="modified inplace"):
        y.sum().backward()


def test_no_memory_is_kept_by_a_cycle(gpu):
    X, R = dev(np.ones((8, 64), np.float32), True), dev(np.ones((8, 64), np.float32))
    gc.collect()
    gc.disable()
    try:
        y, s = nt.rms_norm(X, residual=R)
        w = weakref.ref(y.storage)
        (y.sum() + s.sum()).backward()
        del y, s
        assert w() is None
    finally:
        gc.enable()


def test_more_rows_than_one_launch_counts(gpu):
    """2^26 rows of one wave each are 2^32 work-items, one more than a launch has.
    Rows of ones but for the last and one in the middle."""
    rows, D = 2 ** 26 + 1, 4
    x = nt.full(rows, D, value=2.0, device="cuda")
    for at in (2 ** 25 + 3, rows - 1):
        x[at] = nt.Tensor(np.array([1, 0, 0, 0], np.float32), device="cuda")
    x.enable_grad()
    y = nt.rms_norm(x, eps=0.0)
    for at, want in ((0, [1, 1, 1, 1]), (2 ** 25 + 2, [1, 1, 1, 1]), (2 ** 25 + 3, [2, 0, 0, 0]),
                     (rows - 2, [1, 1, 1, 1]), (rows - 1, [2, 0, 0, 0])):
        assert host(y[at]).tolist() == want, at
    # powers of two throughout: dx = r (g - n mean(g n)) without rounding
    dx = y.grad_fn.backward(y)[0]
    assert float(host(dx.max())) == 0.0 and float(host(dx.min())) == 0.0


def test_module(gpu):
    norm = nn.RMSNorm(32)
    x = rng(1).standard_normal((4, 3, 32)).astype(np.float32)
    check(host(norm(dev(x))), reference(x, None, None, None, None, U[np.float32])["y"], "y")
    y, s = norm(dev(x), dev(x))
    assert_bitexact(host(s), x + x)
    assert [p.shape for p in norm.parameters()] == [(32,)]
