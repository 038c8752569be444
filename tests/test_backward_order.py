"""The order in which the engine runs the nodes of a graph: that of the reference's
walk along every path, without its length.  No device is needed."""

from __future__ import annotations

import random

import pytest

from test_tokens_calls import lib, tensor  # noqa: F401

from nanotorch_amd.core import Tensor, _backward_order


class Node:
    def __init__(self, inputs):
        self.inputs = tuple(inputs)


def leaf(requires_grad=True) -> Tensor:
    t = Tensor.__new__(Tensor)
    t._grad_fn, t._requires_grad, t._grad = None, requires_grad, None
    return t


def node(*inputs) -> Tensor:
    t = leaf(False)
    t._grad_fn = Node(inputs)
    return t


def every_path(seed) -> list[int]:
    """ids of the nodes by their last place in a breadth-first walk of all paths."""
    walk, last = [seed], {}
    for at, x in enumerate(walk):
        if x._grad_fn is None:
            continue
        last[id(x)] = at
        walk.extend(y for y in x._grad_fn.inputs
                    if isinstance(y, Tensor) and (y._requires_grad or y._grad_fn is not None))
    return sorted(last, key=last.get)


@pytest.mark.parametrize("seed", range(200))
def test_order_of_random_graphs(seed):
    r = random.Random(seed)
    made = [leaf(r.random() < 0.7) for _ in range(3)]
    for _ in range(r.randint(1, 11)):
        near = made[-r.randint(1, len(made)):]
        made.append(node(*[r.choice(near) for _ in range(r.randint(1, 3))], 5, None))
    got = _backward_order(made[-1])
    assert [id(x) for x, _, _ in got] == every_path(made[-1])
    for x, fn, inputs in got:
        assert fn is x._grad_fn and inputs == fn.inputs[:-2]


def test_long_chains_of_residuals():
    x = leaf()
    for _ in range(300):
        x = node(x, node(node(x), x))
    assert len(_backward_order(x)) == 900
    assert _backward_order(leaf()) == []


def test_a_residual_around_a_longer_path(lib):  # noqa: F811
    """The short way reaches the shared tensor before any gradient does."""
    w = tensor(4, requires_grad=True)
    x = w * 2.0
    y = (x + ((x * 3.0) * 4.0)) + ((x * 5.0) + x)
    (y.sum() + (x * y).sum()).backward()
    assert w.grad is not None and x._grad is None
