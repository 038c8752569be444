"""Optimizers (reference: src/nanotorch/nn/optimizers.py)."""

from __future__ import annotations

from typing import Sequence

import math
import struct

import numpy as np

from .. import _kernels as K
from .. import autograd as ag
from .._data_type import Dtype, is_float
from .._indexing import row_major_strides
from ..core import Tensor
from ..cuda import Device


class Optimizer:
    def __init__(self, parameters: Sequence[Tensor]) -> None:
        self._parameters = parameters

    @property
    def parameters(self) -> Sequence[Tensor]:
        return self._parameters

    def zero_grad(self) -> None:
        for p in self._parameters:
            p.zero_grad()

    def step(self) -> None:
        raise NotImplementedError


class GradientDescent(Optimizer):
    """p <- p - grad * float32(lr), two roundings, under no_grad."""

    def __init__(self, parameters: Sequence[Tensor], lr: float) -> None:
        super().__init__(parameters)
        self._lr = lr

    def step(self) -> None:
        # lr as the reference's 0-d scalar tensor holds it (float32).  A step
        # size beyond float32's range (an inf scalar), a NaN, or anything that
        # is not a plain real number (e.g. a Tensor) takes the composition,
        # which gives what `p -= g * lr` gives for it.
        try:
            lr32 = struct.unpack("f", struct.pack("f", self._lr))[0]
        except (OverflowError, struct.error, TypeError):
            lr32 = None
        if lr32 is not None and (math.isnan(lr32) or isinstance(self._lr, Tensor)):
            lr32 = None
        for p in self.parameters:
            if p.requires_grad:
                if p.grad is None:
                    raise RuntimeError("Gradients not set, did you call backward?")
                g = p.grad
                with ag.no_grad():
                    if (lr32 is not None and p.device == Device.Cuda and g.device == Device.Cuda
                            and p.dtype == Dtype.Float32 and g.dtype == Dtype.Float32
                            and p.shape == g.shape):
                        # one pass, same two roundings as the composition
                        K.sgd_step(p, g, lr32)
                    else:
                        p -= g * self._lr


def _memory(p: Tensor) -> np.ndarray:
    """An array of p's extent, which is never read: for np.shares_memory."""
    item = 4 if p._storage._dtype is Dtype.Float32 else 8

    class Extent:
        __array_interface__ = {
            "version": 3, "typestr": f"<f{item}", "shape": p._shape,
            "strides": tuple([s * item for s in p._strides]),
            "data": (p._storage._ptr + p._offset * item, True)}

    return np.asarray(Extent())


class AdamW(Optimizer):
    """Adam with decoupled weight decay, over all parameters in one launch for
    each 96 of them:

        m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
        p <- p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

    Parameters are device tensors of one float type, and so are the moments,
    which lie in two vectors, the parameters' parts one after the other (each
    beginning at a multiple of 64 elements).  A parameter listed twice is
    stepped once; different ones may not share memory."""

    _ALIGN = 64

    def __init__(self, parameters: Sequence[Tensor], lr: float, *,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01) -> None:
        parameters = list(parameters)
        super().__init__(parameters)
        lr, eps, weight_decay = float(lr), float(eps), float(weight_decay)
        b1, b2 = [float(b) for b in betas]
        if not (math.isfinite(lr) and 0.0 <= eps < math.inf and 0.0 <= weight_decay < math.inf
                and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW needs a finite lr, 0 <= betas < 1, eps >= 0 and "
                             f"weight_decay >= 0, got {lr=}, {betas=}, {eps=}, {weight_decay=}.")
        self.lr = lr
        self._betas, self._eps, self._decay = (b1, b2), eps, weight_decay
        self._step = 0
        unique: dict[int, Tensor] = {id(p): p for p in parameters}
        # each parameter, where its moments begin, its shape, strides and size
        self._slots: list[tuple[Tensor, int, tuple, tuple, int]] = []
        self._dtype, n = Dtype.Float32, 0
        for i, p in enumerate(unique.values()):
            dtype = p._storage._dtype
            if not is_float(dtype) or (i and dtype != self._dtype):
                raise ValueError(f"AdamW needs parameters of one float type, got "
                                 f"{dtype.name} at {i}.")
            self._dtype = dtype
            self._slots.append((p, n, p._shape, row_major_strides(p._shape), p.numel))
            n += -(-p.numel // self._ALIGN) * self._ALIGN
        self._size = n
        self._m: Tensor | None = None  # made with the first step
        self._v: Tensor | None = None

    @property
    def steps(self) -> int:
        """How many steps were taken."""
        return self._step

    def moments(self) -> tuple[Tensor, Tensor]:
        """The first and second moments of all parameters, as the two vectors
        that the steps update."""
        if self._m is None:
            self._m, self._v = [Tensor._new_contiguous(
                K.fill(self._size, 0.0, self._dtype, Device.Cuda), (self._size,))
                for _ in range(2)]
        return self._m, self._v

    def moments_of(self, i: int) -> tuple[Tensor, Tensor]:
        """The moments of parameter i, as views of its shape."""
        p = list(self._parameters)[i]
        at = next(slot[1] for slot in self._slots if slot[0] is p)
        return tuple([Tensor._new_view(t._storage, p._shape, None, at)
                      for t in self.moments()])

    def load_moments(self, m: Tensor, v: Tensor, steps: int) -> None:
        """Continues from moments() and steps of an earlier optimizer of the
        same parameters; the vectors are copied."""
        for t in (m, v):
            if t._shape != (self._size,) or t._storage._dtype != self._dtype:
                raise ValueError(f"The moments are vectors of {self._size} {self._dtype.name}, "
                                 f"got {t.dtype.name} {t.shape}.")
        if steps < 0:
            raise ValueError(f"steps cannot be negative, got {steps}.")
        self._m, self._v = [t.to(Device.Cuda)._to_contiguous(force=True) for t in (m, v)]
        self._step = int(steps)

    def _check_views(self, views: list[Tensor]) -> None:
        """Refuses memory that is stepped twice; the library sees the views' copies."""
        for p in views:
            if any([n > 1 and s == 0 for n, s in zip(p._shape, p._strides)]) or any([
                    q is not p and q._storage is p._storage
                    and np.shares_memory(_memory(p), _memory(q)) for q, *_ in self._slots]):
                raise RuntimeError("adamw: parameters that share memory with one another "
                                   "cannot be updated together")

    def step(self) -> None:
        tensors: list[int] = []
        written = []
        copies: list[tuple[Tensor, Tensor]] = []  # views: stepped as a copy
        keep = []  # temporaries live until the call
        dtype, cuda = self._dtype, Device.Cuda
        item = 4 if dtype is Dtype.Float32 else 8
        for p, at, shape, strides, n in self._slots:
            if not p._requires_grad and p._grad_fn is None:
                continue
            g = p._grad
            if g is None:
                raise RuntimeError("Gradients not set, did you call backward?")
            to, ps, gs = p, p._storage, g._storage
            if not (ps._dtype is dtype and gs._dtype is dtype and ps._device is cuda
                    and gs._device is cuda and p._strides == strides and g._strides == strides
                    and p._shape == shape and g._shape == shape):
                K.require_device(p, g)
                if ps._dtype != dtype or p._shape != shape or g._shape != shape:
                    raise ValueError(f"A parameter {dtype.name} {shape} became {p.dtype.name} "
                                     f"{p.shape}, or its gradient has another shape: {g.shape}.")
                if gs._dtype != dtype or g._strides != strides:
                    g = g.to(dtype)._to_contiguous()
                    keep.append(g)
                if p._strides != strides:
                    to = p._to_contiguous(force=True)
                    copies.append((to, p))
            tensors += (to._storage._ptr + to._offset * item, g._storage._ptr + g._offset * item,
                        n, at)
            written.append(ps)
        if copies:
            self._check_views([p for _, p in copies])
        m, v = self.moments()
        K.adamw_step(tensors, m, v, self.lr, self._betas, self._eps, self._decay, self._step + 1)
        self._step += 1
        for new, p in copies:
            K.copy_view(new, p)
        for storage in written:
            storage.version += 1
