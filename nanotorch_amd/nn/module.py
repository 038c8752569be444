"""Parametrised modules (reference: src/nanotorch/nn/module.py).

``Linear`` keeps the reference's He-uniform init ``2 * U[0,1) * z - z`` with
``z = sqrt(6 / fan_in)`` and zero bias; the arithmetic runs in float32 on the
device (same three roundings as the reference's host loop), so parameters
start on ``device`` (default "cuda").  ``Sigmoid`` is added next to ReLU and
Tanh (the reference exposes sigmoid only as a function).  ``Linear.forward``
on float32 device tensors runs the product and the bias add as one kernel
(``LinearOp``): same values and gradients as the reference's two ops.
``Embedding`` and ``Dropout`` are additions too, and with ``Dropout`` the
modules' ``train`` / ``eval`` switch.
"""

from __future__ import annotations

import math
from typing import Any, Iterable, Iterator, Sequence

from ..autograd import EmbeddingOp, ReluOp, SigmoidOp, TanhOp
from ..autograd.ops_binary import LinearOp
from ..core import Tensor
from ..cuda import Device
from ..factories import rand, zeros
from ..ops import dropout


class Module:
    def __call__(self, *args: Any, **kwargs: Any) -> Any:
        return self.forward(*args, **kwargs)

    def parameters(self) -> Sequence[Tensor]:
        return []

    def to(self, device: Device | str) -> "Module":
        return self

    def train(self, mode: bool = True) -> "Module":
        """Training (True) or answering (False), for this module and those
        among its attributes, in lists, tuples and dicts too: only Dropout
        differs."""
        own = vars(self)
        if "_switching" not in own:  # once, where modules refer to each other
            modules = list(_modules_in(own.values()))
            own["_switching"] = True
            try:
                for m in modules:
                    m.train(mode)
            finally:
                del own["_switching"]
        return self

    def eval(self) -> "Module":
        return self.train(False)

    def forward(self, *args: Any, **kwargs: Any) -> Any:
        raise NotImplementedError


def _modules_in(values: Iterable[Any]) -> Iterator[Module]:
    for v in values:
        if isinstance(v, Module):
            yield v
        elif isinstance(v, dict):
            yield from _modules_in(v.values())
        elif isinstance(v, (list, tuple)):
            yield from _modules_in(v)


class Linear(Module):
    """y = x @ W + b with W [fan_in, fan_out]."""

    def __init__(self, fan_in: int, fan_out: int, bias: bool = True, *,
                 device: Device | str = "cuda") -> None:
        self._W = _kaiming_W(fan_in, fan_out, device)
        self._W.enable_grad()
        self._b = zeros(fan_out, requires_grad=True, device=device) if bias else None

    def parameters(self) -> Sequence[Tensor]:
        return [self._W] if self._b is None else [self._W, self._b]

    def to(self, device: Device | str) -> "Linear":
        self._W = self._W.to(device)
        if self._b is not None:
            self._b = self._b.to(device)
        return self

    def forward(self, x: Tensor) -> Tensor:
        if x.ndim != 2:
            raise NotImplementedError(f"Can only forward a 2D tensor for now, got {x.ndim}")
        if x.shape[1] != self._W.shape[0]:
            raise ValueError(f"Cannot align axes of size {x.shape[1]} and {self._W.shape[0]}.")
        if self._b is not None and LinearOp.usable(x, self._W, self._b):
            # the product and the bias add in one kernel, same roundings
            return LinearOp.apply(x, self._W, self._b)
        z = x @ self._W
        if self._b is not None:
            z = z + self._b
        return z


class Embedding(Module):
    """scale * W[tokens] with W [num_tokens, dim] drawn uniformly with unit
    variance; a token equal to padding_idx gives zeros and trains nothing."""

    def __init__(self, num_tokens: int, dim: int, scale: float = 1.0, *,
                 padding_idx: int | None = None, device: Device | str = "cuda") -> None:
        if num_tokens <= 0 or dim <= 0:
            raise ValueError(
                f"Cannot initialize Embedding with {num_tokens=}, {dim=} (non-positive)."
            )
        if padding_idx is not None and not 0 <= padding_idx < num_tokens:
            raise ValueError(f"padding_idx {padding_idx} is no row of a table of {num_tokens}.")
        z = math.sqrt(3.0)
        w = 2 * rand(num_tokens, dim, device="cuda") * z - z
        self._W = w.to(device)
        self._W.enable_grad()
        self._scale, self._padding_idx = scale, padding_idx

    def parameters(self) -> Sequence[Tensor]:
        return [self._W]

    def to(self, device: Device | str) -> "Embedding":
        self._W = self._W.to(device)
        return self

    def forward(self, tokens: Tensor) -> Tensor:
        return EmbeddingOp.apply(self._W, tokens, self._scale, self._padding_idx)


class Dropout(Module):
    """Drops each element with probability p while training and scales the
    others by 1 / (1 - p); passes its input on otherwise."""

    def __init__(self, p: float = 0.5) -> None:
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"Dropout needs 0 <= p <= 1, got {p}.")
        self._p = p
        self._training = True

    def train(self, mode: bool = True) -> "Dropout":
        self._training = mode
        return self

    def forward(self, x: Tensor) -> Tensor:
        return dropout(x, self._p) if self._training and self._p > 0.0 else x


class ReLU(Module):
    def forward(self, x: Tensor) -> Tensor:
        return ReluOp.apply(x)


class Tanh(Module):
    def forward(self, x: Tensor) -> Tensor:
        return TanhOp.apply(x)


class Sigmoid(Module):
    def forward(self, x: Tensor) -> Tensor:
        return SigmoidOp.apply(x)


class Sequential(Module):
    def __init__(self, *modules: Module) -> None:
        self._modules = list(modules)

    def parameters(self) -> Sequence[Tensor]:
        params: list[Tensor] = []
        for m in self._modules:
            params.extend(m.parameters())
        return params

    def to(self, device: Device | str) -> "Sequential":
        self._modules = [m.to(device) for m in self._modules]
        return self

    def forward(self, *args: Any, **kwargs: Any) -> Any:
        x = None
        for i, m in enumerate(self._modules):
            x = m(*args, **kwargs) if i == 0 else m(x)
        return x


def _kaiming_W(fan_in: int, fan_out: int, device: Device | str = "cuda") -> Tensor:
    if fan_in <= 0 or fan_out <= 0:
        raise ValueError(
            f"Cannot initialize Linear with {fan_in=}, {fan_out=} (non-positive)."
        )
    z = math.sqrt(6 / fan_in)
    u = rand(fan_in, fan_out, device="cuda")  # drawn on the device, same stream
    w = 2 * u * z - z
    return w if str(device) in ("cuda", "Device.Cuda") or device == Device.Cuda else w.to(device)
