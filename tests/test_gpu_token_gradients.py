"""Gradients of the token operators where they can go wrong: gradients that
share memory with the results, nearly uniform rows, results changed in place,
left-out tokens in the radix sort, logits that outgrow the Infinity Cache.

Tolerances are those of test_gpu_tokens; sums of small integers, which are
exact in any order, are compared bit for bit."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import dev, host, rng
from test_gpu_tokens import Rows, draw_rows

import nanotorch_amd as nt

pytestmark = pytest.mark.gpu


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
