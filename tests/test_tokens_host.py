"""The token operators' argument checks and switches that need no device."""

from __future__ import annotations

import numpy as np
import pytest

import nanotorch_amd as nt
from nanotorch_amd import nn
from nanotorch_amd.autograd import ops_token
from nanotorch_amd.factories import next_dropout_counter


def test_arguments_are_checked_before_the_device():
    w, t = nt.ones(4, 3), nt.zeros(2, dtype=nt.int64)
    for bad in (lambda: nt.embedding(nt.ones(4), t), lambda: nt.embedding(w, w),
                lambda: nt.embedding(w, t, padding_idx=9), lambda: nt.dropout(w, 2.0),
                lambda: nt.dropout(t, 0.5), lambda: nt.token_logprobs(w),
                lambda: nt.token_logprobs(w, t), lambda: nt.token_logprobs(w, entropy=True, top=4),
                lambda: nt.token_logprobs(t, t), lambda: nn.Dropout(-1.0),
                lambda: nn.Embedding(3, 0)):
        with pytest.raises(ValueError):
            bad()


def test_host_tensors_are_refused():
    w, t = nt.ones(4, 3), nt.zeros(4, dtype=nt.int64)
    for call in (lambda: nt.embedding(w, t), lambda: nt.dropout(w), lambda: nt.dropout(w, 0.0),
                 lambda: nt.token_logprobs(w, t), lambda: nt.token_logprobs(w, top=2)):
        with pytest.raises(RuntimeError):
            call()


def test_dropout_counter():
    nt.manual_seed(5)
    assert [next_dropout_counter() for _ in range(3)] == [(5, 0), (5, 1), (5, 2)]
    nt.manual_seed(-1)
    assert next_dropout_counter() == (2 ** 64 - 1, 0)


def test_train_and_eval_reach_nested_modules():
    a, b = nn.Dropout(0.5), nn.Dropout(0.5)
    net = nn.Sequential(a, nn.Sequential(nn.Tanh(), b), lambda x: x)
    x = nt.ones(3)
    assert net.eval() is net
    assert a(x) is x and b(x) is x
    net.train()
    with pytest.raises(RuntimeError):  # drops again: needs the device
        b(x)


@pytest.mark.parametrize("make,in_place", [
    (lambda a: a, True), (lambda a: a[1], True), (lambda a: a[:, :, 2:7], True),
    (lambda a: a[0, 0], True), (lambda a: a[:, 1:], False), (lambda a: a[:, :, ::2], False),
    (lambda a: a.transpose(0, 1), False), (lambda a: a[:, ::2, 1:2], False)])
def test_rows_in_place(make, in_place):
    """A view of rows where the strides allow one, else a copy; the same values."""
    x = make(nt.Tensor(np.arange(2 * 3 * 20, dtype=np.float32).reshape(2, 3, 20)))
    assert (ops_token._rows_in_place(x) is not None) == in_place
    rows = ops_token._as_rows(x)
    assert (rows.storage is x.storage) == in_place
    want = x.numpy().reshape(-1, x.shape[-1])
    assert rows.shape == want.shape and (rows.numpy() == want).all()


def test_dropout_offset_without_a_seed_is_refused():
    nt.manual_seed(5)
    for offset in (0, 7):
        with pytest.raises(ValueError):
            nt.dropout(nt.ones(3), 0.5, offset=offset)
    assert next_dropout_counter() == (5, 0)  # a refused call draws nothing


class Composed(nn.Module):
    """Holds its modules in every way that an attribute can."""

    def __init__(self):
        self.drop = nn.Dropout(0.5)
        self.layers = [nn.Tanh(), (nn.Dropout(0.5), [nn.Dropout(0.5)])]
        self.heads = {"a": nn.Dropout(0.5), "b": {"c": nn.Sequential(nn.Dropout(0.5))}}
        self.other = ("a text", 3, None, {"x": 1.0}, nt.ones(2), lambda x: x)

    def dropouts(self):
        return [self.drop, self.layers[1][0], self.layers[1][1][0], self.heads["a"],
                self.heads["b"]["c"]._modules[0]]


def dropping(m):
    """Whether a Dropout drops: then it needs the device."""
    x = nt.ones(3)
    try:
        return m(x) is not x
    except RuntimeError:
        return True


@pytest.mark.parametrize("wrap", [lambda m: m, lambda m: nn.Sequential(nn.Tanh(), m)])
def test_train_and_eval_reach_the_modules_of_a_composed_one(wrap):
    inner = Composed()
    net = wrap(inner)
    before = dict(vars(inner))
    assert net.eval() is net
    assert not any(map(dropping, inner.dropouts()))
    assert net.train() is net
    assert all(map(dropping, inner.dropouts()))
    assert net.train(False) is net
    assert not any(map(dropping, inner.dropouts()))
    assert vars(inner) == before


def test_train_reaches_modules_that_refer_to_each_other():
    a, b = Composed(), Composed()
    a.child, b.parent = b, a
    b.eval()
    assert not any(map(dropping, a.dropouts() + b.dropouts()))
    a.train()
    assert all(map(dropping, a.dropouts() + b.dropouts()))


def test_a_train_of_ones_own_is_called():
    class Own(nn.Module):
        def train(self, mode=True):
            self.modes = getattr(self, "modes", []) + [mode]
            return self

    own = Own()
    net = nn.Sequential(own)
    net.train()
    net.eval()
    assert own.modes == [True, False]


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    ((2 ** 32 - 1,) * 4, (2 ** 32 - 1,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     "d16cfe09 94fdcceb 5001e420 24126ea1")])
def test_philox_published_answers(counter, key, want):
    """What dropout's device results are compared with, against the known
    answers published with Philox4x32-10: zeros, all ones, digits of pi."""
    from test_gpu_tokens import words_of

    i = np.array([counter[0] | counter[1] << 32], np.uint64)
    got = words_of(i, key[0] | key[1] << 32, counter[2] | counter[3] << 32)
    assert " ".join(f"{int(w):08x}" for w in got) == want
