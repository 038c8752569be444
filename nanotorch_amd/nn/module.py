"""Parametrised modules (reference: src/nanotorch/nn/module.py).

``Linear`` keeps the reference's He-uniform init ``2 * U[0,1) * z - z`` with
``z = sqrt(6 / fan_in)`` and zero bias; the arithmetic runs in float32 on the
device (same three roundings as the reference's host loop), so parameters
start on ``device`` (default "cuda").  ``Sigmoid`` is added next to ReLU and
Tanh (the reference exposes sigmoid only as a function).  ``Linear.forward``
on float32 device tensors runs the product and the bias add as one kernel
(``LinearOp``): same values and gradients as the reference's two ops.
``Embedding`` and ``Dropout`` are additions too, and with ``Dropout`` the
modules' ``train`` / ``eval`` switch; so are ``RMSNorm``, ``Attention`` and its
``KeyValueCache``.
"""

from __future__ import annotations

import math
from typing import Any, Iterable, Iterator, Sequence

from ..autograd import EmbeddingOp, ReluOp, SigmoidOp, TanhOp, is_grad_enabled
from ..autograd.ops_binary import LinearOp
from ..core import Tensor
from ..cuda import Device
from ..factories import ones, rand, zeros
from ..ops import attention, dropout, rms_norm


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


class RMSNorm(Module):
    """x (mean x^2 + eps)^-1/2 w over the last axis, w [dim] beginning with
    ones.  With a residual: (that of x + residual, x + residual)."""

    def __init__(self, dim: int, eps: float = 1e-6, *, device: Device | str = "cuda") -> None:
        if dim <= 0:
            raise ValueError(f"Cannot initialize RMSNorm with {dim=} (non-positive).")
        self._w = ones(dim, requires_grad=True, device=device)
        self._eps = eps

    def parameters(self) -> Sequence[Tensor]:
        return [self._w]

    def to(self, device: Device | str) -> "RMSNorm":
        self._w = self._w.to(device)
        return self

    def forward(self, x: Tensor, residual: Tensor | None = None):
        return rms_norm(x, self._w, residual=residual, eps=self._eps)


class KeyValueCache:
    """Keys and values of up to max_tokens tokens of some sequences, which
    Attention fills and reads: every call's tokens come behind those before."""

    def __init__(self, sequences: int, max_tokens: int, kv_heads: int, head_dim: int) -> None:
        shape = (sequences, max_tokens, kv_heads, head_dim)
        self.keys = zeros(*shape, device="cuda")
        self.values = zeros(*shape, device="cuda")
        self.tokens = 0

    def append(self, k: Tensor, v: Tensor) -> tuple[Tensor, Tensor]:
        """Stores [sequences, n, kv_heads, head_dim] and returns views of all so
        far."""
        B, most, heads, dim = self.keys.shape
        n, end = k.shape[1], self.tokens + k.shape[1]
        if k.shape != (B, n, heads, dim) or v.shape != k.shape:
            raise ValueError(f"A cache of {self.keys.shape} cannot take {k.shape}, {v.shape}.")
        if end > most:
            raise ValueError(f"A cache of {most} tokens cannot hold {end}.")
        self.keys[:, self.tokens:end] = k
        self.values[:, self.tokens:end] = v
        self.tokens = end
        return self.keys[:, :end], self.values[:, :end]


class Attention(Module):
    """Self-attention of x [B, T, dim]: projections to `heads` query heads and
    `kv_heads` key heads (as many unless given), attention, projection back.

    Causal unless told otherwise.  `lengths` [B] are the texts' own tokens where
    they are padded at their ends.  With a cache, x holds the tokens after those
    that it has; nothing is differentiated through it."""

    def __init__(self, dim: int, heads: int, kv_heads: int | None = None, *, causal: bool = True,
                 device: Device | str = "cuda") -> None:
        kv_heads = heads if kv_heads is None else kv_heads
        if min(dim, heads, kv_heads) <= 0 or dim % heads or heads % kv_heads:
            raise ValueError(f"Cannot initialize Attention with {dim=}, {heads=}, {kv_heads=}.")
        self._heads, self._kv_heads, self._head_dim = heads, kv_heads, dim // heads
        self._causal = causal
        self._q = Linear(dim, dim, False, device=device)
        self._k = Linear(dim, kv_heads * self._head_dim, False, device=device)
        self._v = Linear(dim, kv_heads * self._head_dim, False, device=device)
        self._out = Linear(dim, dim, False, device=device)

    def parameters(self) -> Sequence[Tensor]:
        return [p for m in (self._q, self._k, self._v, self._out) for p in m.parameters()]

    def to(self, device: Device | str) -> "Attention":
        for m in (self._q, self._k, self._v, self._out):
            m.to(device)
        return self

    def cache(self, sequences: int, max_tokens: int) -> KeyValueCache:
        return KeyValueCache(sequences, max_tokens, self._kv_heads, self._head_dim)

    def forward(self, x: Tensor, lengths: Tensor | None = None,
                cache: KeyValueCache | None = None) -> Tensor:
        if x.ndim != 3:
            raise ValueError(f"Attention takes [B, T, dim], got {x.shape}.")
        B, T, dim = x.shape
        flat = x.reshape(B * T, dim)
        q = self._q(flat).reshape(B, T, self._heads, self._head_dim)
        k = self._k(flat).reshape(B, T, self._kv_heads, self._head_dim)
        v = self._v(flat).reshape(B, T, self._kv_heads, self._head_dim)
        if cache is None:
            starts = 0 if self._causal else None
        else:
            if lengths is not None or not self._causal:
                raise ValueError("A cache is for causal attention without padding.")
            if is_grad_enabled() and any([t.requires_grad for t in (q, k, v)]):
                raise RuntimeError("A cache is not differentiated: use no_grad().")
            starts = cache.tokens
            k, v = cache.append(k, v)
        try:
            y = attention(q, k, v, causal=self._causal, lengths=lengths, starts=starts)
        except BaseException:
            if cache is not None:
                cache.tokens = starts  # a refused call adds nothing
            raise
        return self._out(y.reshape(B * T, dim)).reshape(B, T, dim)


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
