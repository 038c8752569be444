"""What the transformer's operators refuse, and what they hand to the library,
recorded in place of it.  No device is needed."""

from __future__ import annotations

import math
import struct

import numpy as np
import pytest

from test_tokens_calls import Recorder, lib, parse, tensor  # noqa: F401

import nanotorch_amd as nt
from nanotorch_amd import _lib, nn
from nanotorch_amd._data_type import Dtype
from nanotorch_amd.core import Tensor


def heads(*shape, **kw):
    return tensor(*shape, **kw)


@pytest.mark.parametrize("q,k,v", [
    ((4, 8), (4, 8), (4, 8)),                        # no heads
    ((1, 2, 3, 4, 8), (1, 2, 3, 4, 8), (1, 2, 3, 4, 8)),
    ((2, 4, 3, 8), (2, 4, 2, 8), (2, 4, 2, 8)),      # 3 heads over 2
    ((2, 4, 2, 8), (2, 4, 0, 8), (2, 4, 0, 8)),
    ((2, 4, 0, 8), (2, 4, 1, 8), (2, 4, 1, 8)),
    ((2, 4, 2, 8), (2, 4, 2, 8), (2, 5, 2, 8)),
    ((2, 4, 2, 8), (2, 4, 2, 9), (2, 4, 2, 9)),
    ((2, 4, 2, 8), (3, 4, 2, 8), (3, 4, 2, 8)),
    ((2, 4, 2, 8), (4, 2, 8), (4, 2, 8)),
    ((2, 4, 2, 257), (2, 4, 2, 257), (2, 4, 2, 257)),
    ((2, 4, 2, 0), (2, 4, 2, 0), (2, 4, 2, 0)),
])
def test_attention_refuses_shapes(lib, q, k, v):  # noqa: F811
    with pytest.raises(ValueError):
        nt.attention(heads(*q), heads(*k), heads(*v))
    assert not [n for n, _ in lib.calls if n == "nt_attention"]


def test_attention_refuses_types_and_masks(lib):  # noqa: F811
    q = heads(2, 4, 2, 8)
    for other in (Dtype.Float64, Dtype.Int64):
        with pytest.raises(ValueError):
            nt.attention(q, heads(2, 4, 2, 8, dtype=other), q)
        with pytest.raises(ValueError):
            nt.attention(q, q, heads(2, 4, 2, 8, dtype=other))
    i = heads(2, 4, 2, 8, dtype=Dtype.Int32)
    with pytest.raises(ValueError):
        nt.attention(i, i, i)
    for bad in (tensor(3, dtype=Dtype.Int64), tensor(2), tensor(2, 1, dtype=Dtype.Int32)):
        with pytest.raises(ValueError):
            nt.attention(q, q, q, lengths=bad)
        with pytest.raises(ValueError):
            nt.attention(q, q, q, causal=True, starts=bad)
    with pytest.raises(ValueError):
        nt.attention(q, q, q, starts=0)
    with pytest.raises(ValueError):
        nt.attention(q, q, q, causal=True, starts=2**63)
    assert not [n for n, _ in lib.calls if n == "nt_attention"]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bad", [[1, 2], 2, np.array([1, 2])])
def test_attention_refuses_lengths_that_are_no_tensor(lib, bad, causal):  # noqa: F811
    q = heads(2, 4, 2, 8)
    with pytest.raises(TypeError):
        nt.attention(q, q, q, causal=causal, lengths=bad)
    assert not [n for n, _ in lib.calls if n == "nt_attention"]


@pytest.mark.parametrize("bad", [[1, 2], 2.5, np.array([1, 2]), "3"])
def test_attention_refuses_starts_that_are_no_whole_number(lib, bad):  # noqa: F811
    q = heads(2, 4, 2, 8)
    with pytest.raises(TypeError):
        nt.attention(q, q, q, causal=True, starts=bad)
    assert not [n for n, _ in lib.calls if n == "nt_attention"]
    nt.attention(q, q, q, causal=True, starts=np.int64(3))
    assert [n for n, _ in lib.calls if n == "nt_attention"]


def test_starts_without_a_causal_mask_have_no_effect(lib):  # noqa: F811
    """A program that switches the mask off keeps its other arguments."""
    q = heads(2, 4, 2, 8)
    for starts in (0, 3, tensor(2, dtype=Dtype.Int32)):
        nt.attention(q, q, q, causal=False, starts=starts)
        a = lib.args("nt_attention")
        assert a[4] is None and a[5:7] == (0, 0)
    with pytest.raises(TypeError):
        nt.attention(q, q, q, causal=False, starts=1.5)
    with pytest.raises(ValueError):
        nt.attention(q, q, q, causal=False, starts=tensor(3, dtype=Dtype.Int32))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 2.0**127, -1e39])
def test_attention_refuses_scales_that_are_not_finite(lib, bad):  # noqa: F811
    q = heads(2, 4, 2, 8)
    with pytest.raises(ValueError, match="finite scale"):
        nt.attention(q, q, q, scale=bad)
    assert not [n for n, _ in lib.calls if n == "nt_attention"]
    if math.isfinite(bad):
        q = heads(2, 4, 2, 8, dtype=Dtype.Float64)
        nt.attention(q, q, q, scale=bad)


def test_host_tensors_are_refused():
    x = nt.Tensor(np.ones((1, 3, 2, 4), np.float32))
    with pytest.raises(RuntimeError, match="GPU"):
        nt.attention(x, x, x)
    with pytest.raises(RuntimeError, match="GPU"):
        nt.rms_norm(x)
    p = nt.Tensor(np.ones(3, np.float32), requires_grad=True)
    p._grad = nt.Tensor(np.ones(3, np.float32))
    with pytest.raises(RuntimeError, match="GPU"):
        nn.AdamW([p], 0.1).step()


def test_attention_calls(lib):  # noqa: F811
    q, k = heads(2, 5, 4, 8, requires_grad=True), heads(2, 9, 2, 8)
    n = tensor(2, dtype=Dtype.Int32)
    y = nt.attention(q, k, k, causal=True, lengths=n)
    a = lib.args("nt_attention")
    assert a[0].shape == (2, 5, 4, 8) and a[3].shape == (2,) and a[4] is None
    assert a[5:8] == (0, 1, 8 ** -0.5)
    assert a[8].shape == (2, 5, 4, 8) and a[9].shape == (40,)
    lib.within(a[8]), lib.within(a[9])
    y.grad_fn._backward_into(heads(2, 5, 4, 8), [True, False, False, False], [None] * 4)
    b = lib.args("nt_attention_bwd")
    assert b[:8] == a[:8] and b[8] == a[8] and b[9] == a[9]
    assert b[11].shape == (2, 5, 4, 8) and b[12] is None and b[13] is None
    with nt.no_grad():
        nt.attention(q, k, k, causal=True, starts=3)
    a = lib.args("nt_attention")
    assert a[5:7] == (3, 2) and a[9] is None


def test_rms_norm_refuses(lib):  # noqa: F811
    x = tensor(4, 6)
    for bad in (lambda: nt.rms_norm(tensor(4, 6, dtype=Dtype.Int32)),
                lambda: nt.rms_norm(tensor()), lambda: nt.rms_norm(tensor(4, 0)),
                lambda: nt.rms_norm(x, tensor(5)), lambda: nt.rms_norm(x, tensor(4, 6)),
                lambda: nt.rms_norm(x, tensor(6, dtype=Dtype.Float64)),
                lambda: nt.rms_norm(x, residual=tensor(6)),
                lambda: nt.rms_norm(x, residual=tensor(4, 6, dtype=Dtype.Float64)),
                lambda: nt.rms_norm(x, eps=-1.0), lambda: nt.rms_norm(x, eps=math.nan)):
        with pytest.raises(ValueError):
            bad()
    assert not [n for n, _ in lib.calls if n == "nt_rms_norm"]


def test_rms_norm_calls(lib):  # noqa: F811
    x, w, res = tensor(3, 4, 6, requires_grad=True), tensor(6), tensor(3, 4, 6)
    y, s = nt.rms_norm(x, w, residual=res, eps=0.5)
    a = lib.args("nt_rms_norm")
    assert [v.shape for v in a[:3]] == [(12, 6), (12, 6), (6,)] and a[3] == 0.5
    assert not set(lib.within(a[4])) & set(lib.within(a[5]))
    assert y._storage._ptr == a[4].ptr and s._storage._ptr == a[4].ptr + 4 * 72
    assert y._shape == s._shape == (3, 4, 6) and a[6].shape == (12,)
    (s.sum()).backward()  # the norm takes no part: its gradient is absent
    b = lib.args("nt_rms_norm_bwd")
    assert b[3] is None and b[4].shape == (12, 6) and b[6] is None
    with nt.no_grad():
        nt.rms_norm(x)
    a = lib.args("nt_rms_norm")
    assert a[1] is a[2] is a[5] is a[6] is None


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("leaf", ["none", "x", "residual"])
def test_rms_norm_gradients_of_one_memory(lib, weighted, leaf):  # noqa: F811
    """x and the residual share their gradient's memory unless one of them is a
    leaf, which keeps it; whether the weight is trained does not matter."""
    x, res = [tensor(4, 6, requires_grad=True) for _ in range(2)]
    w = tensor(6, requires_grad=True) if weighted else None
    if leaf != "x":
        x = x * 2.0
    if leaf != "residual":
        res = res * 2.0
    y, _ = nt.rms_norm(x, w, residual=res)
    fn = y.grad_fn.inputs[0].grad_fn
    n = 3 if weighted else 2
    lib.calls.clear()
    got = fn._backward_into(tensor(2, 4, 6), [True] * n, [None] * n)
    assert (got[0]._storage is got[-1]._storage) == (leaf == "none")
    if leaf == "none":
        assert [name for name, _ in lib.calls] == ["nt_rms_norm_bwd"]
        assert got[0]._shared and got[-1]._shared
    # a weight that alone is wanted
    if weighted:
        got = fn._backward_into(tensor(2, 4, 6), [False, True, False], [None] * 3)
        assert got[0] is got[2] is None and got[1]._shape == (6,)


def test_adamw_refuses(lib):  # noqa: F811
    p = tensor(4, requires_grad=True)
    for kw in ({"lr": math.nan}, {"lr": math.inf}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)},
               {"eps": -1.0}, {"weight_decay": -0.1}, {"weight_decay": math.nan}):
        with pytest.raises(ValueError):
            nn.AdamW([p], **{"lr": 0.1, **kw})
    with pytest.raises(ValueError):
        nn.AdamW([p, tensor(3, dtype=Dtype.Float64)], 0.1)
    with pytest.raises(ValueError):
        nn.AdamW([tensor(3, dtype=Dtype.Int64)], 0.1)
    opt = nn.AdamW([p], 0.1)
    with pytest.raises(RuntimeError, match="Gradients not set"):
        opt.step()
    p._grad = tensor(5)
    with pytest.raises(ValueError):
        opt.step()
    with pytest.raises(ValueError):
        opt.load_moments(tensor(4), tensor(64), 1)
    with pytest.raises(ValueError):
        opt.load_moments(tensor(64), tensor(64), -1)
    assert opt.steps == 0 and not [n for n, _ in lib.calls if n == "nt_adamw_step"]


def test_adamw_calls(lib):  # noqa: F811
    ps = [tensor(3, 5, requires_grad=True), tensor(70, requires_grad=True), tensor(2)]
    ps.append(ps[0])
    for p in ps[:2]:
        p._grad = tensor(*p._shape)
    opt = nn.AdamW(ps, 0.1, betas=(0.5, 0.25), eps=1e-3, weight_decay=0.2)
    opt.step()
    args = [a for n, a in lib.calls if n == "nt_adamw_step"][-1]
    rows = np.array(struct.unpack("=8q", args[0])).reshape(2, 4)
    assert args[1] == 2 and rows[:, 2].tolist() == [15, 70] and rows[:, 3].tolist() == [0, 64]
    assert rows[:, 0].tolist() == [p._storage._ptr for p in ps[:2]]
    assert rows[:, 1].tolist() == [p._grad._storage._ptr for p in ps[:2]]
    assert parse(args[2]).shape == (256,)
    assert args[4:] == (0.1, 0.5, 0.25, 1e-3, 0.2, 1)
    assert opt.steps == 1


def test_a_refused_call_leaves_the_cache(lib):  # noqa: F811
    for dtype, heads_, dim in ((Dtype.Float64, 2, 8), (Dtype.Float32, 1, 300)):
        a = nn.Attention(dim, heads_)
        cache = a.cache(2, 10)
        with nt.no_grad():
            if dtype is Dtype.Float32:
                with pytest.raises(ValueError, match="1 to 256"):
                    a(tensor(2, 4, dim), cache=cache)
            else:
                a(tensor(2, 3, dim), cache=cache)
                with pytest.raises(ValueError, match="one dtype"):
                    a(tensor(2, 4, dim, dtype=dtype), cache=cache)
        assert cache.tokens == (0 if dtype is Dtype.Float32 else 3)


def test_modules_refuse():
    for args in ((0, 1), (8, 3), (8, 4, 3), (8, 0), (8, 4, 0)):
        with pytest.raises(ValueError):
            nn.Attention(*args)
    with pytest.raises(ValueError):
        nn.RMSNorm(0)


def test_an_abi_call_reports_and_survives():
    """Errors at the C entry points are statuses, without a device too."""
    l = _lib.load()
    rc = l.nt_attention(None, None, None, None, None, 0, 0, 1.0, None, None)
    assert rc != 0 and l.nt_last_error()
    assert l.nt_rms_norm(None, None, None, 0.0, None, None, None) != 0
    assert l.nt_adamw_step(None, 1, None, None, 0.1, 0.9, 0.9, 0.0, 0.0, 1) != 0
    assert isinstance(Tensor, type)
