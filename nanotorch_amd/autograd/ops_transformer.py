"""Differentiable ops of a transformer's blocks: the root-mean-square norm with
the residual's addition, and attention.  The reference has neither."""

from __future__ import annotations

import math

from .. import _kernels as K
from .._data_type import is_float, is_int, sizeof
from .._indexing import row_major_strides
from ..core import Tensor, reshape_view
from .function import Function
from .grad_mode import is_grad_enabled
from .ops_token import RowOp, _added, _as_rows, _row_of, _RowGradients, _vector


def _give(storage, shape, target: Tensor | None) -> Tensor:
    """A new gradient, or `target` with it added."""
    if target is not None:
        return _added(target, storage, shape)
    return Tensor._unchecked_view(storage, shape, row_major_strides(shape), 0)


class RmsNormOp(Function):
    """s (mean s^2 + eps)^-1/2 weight over the last axis, s = x + residual.

    With a residual the output is [2, ...]: that, and s itself, whose gradients
    one pass takes together; NormRowOp hands out the two."""

    def forward(self, x: Tensor, weight: Tensor | None = None, residual: Tensor | None = None,
                eps: float = 1e-6) -> Tensor:
        shape, dtype = x._shape, x._storage._dtype
        if not shape or shape[-1] == 0 or not is_float(dtype):
            raise ValueError(f"rms_norm() needs a float tensor with an axis of elements, got "
                             f"{x.dtype.name} {shape}.")
        if residual is not None and (residual._shape != shape
                                     or residual._storage._dtype != dtype):
            raise ValueError(f"The residual must be {x.dtype.name} {shape} as x is, got "
                             f"{residual.dtype.name} {residual.shape}.")
        if weight is not None and (weight._shape != shape[-1:]
                                   or weight._storage._dtype != dtype):
            raise ValueError(f"The weight must be {x.dtype.name} {shape[-1:]}, got "
                             f"{weight.dtype.name} {weight.shape}.")
        if not eps >= 0.0:
            raise ValueError(f"rms_norm() needs eps >= 0, got {eps}.")
        inputs = [t for t in (x, weight, residual) if t is not None]
        keep = is_grad_enabled() and any(t.requires_grad for t in inputs)
        rows = _as_rows(x)
        w = None if weight is None else weight._to_contiguous()
        out, rstd = K.rms_norm(rows, None if residual is None else _as_rows(residual), w,
                               float(eps), keep)
        strides = row_major_strides(shape)
        self._given = tuple([t is not None for t in (x, weight, residual)])
        self._shape = shape
        if residual is None:
            y, total, saved = Tensor._unchecked_view(out, shape, strides, 0), rows, x
        else:
            n = rows._shape[0] * rows._shape[1]
            total = saved = Tensor._unchecked_view(out.part(n, n), shape, strides, 0)
            y = Tensor._unchecked_view(out, (2,) + shape, (n,) + strides, 0)
            y._rows = (Tensor._unchecked_view(out, shape, strides, 0), total)
        # (none of the tensors kept here gets a graph node: no cycles)
        if keep:
            self.save_for_backward(*((saved,) if weight is None else (saved, weight)))
            self._call = (_as_rows(total), w, rstd)
        return y

    def backward(self, grad_out: Tensor) -> tuple:
        n = sum(self._given)  # x and the residual get one tensor, as those of a sum do
        return tuple(self._grad(grad_out, [True] * n, [None] * n, True))

    def fused_ok(self) -> bool:
        return True

    def _backward_into(self, g: Tensor, needs, targets):
        # of x and the residual; the weight, mostly a leaf, has a gradient of its own
        tensors = [t for t in self._inputs if isinstance(t, Tensor)]
        leaf = any([tensors[i].is_leaf for i in (0, len(needs) - 1) if needs[i]])
        return self._grad(g, needs, targets, not leaf)

    def _grad(self, g: Tensor, needs, targets, share: bool) -> list:
        self.saved_tensors  # raises if the sum or the weight was modified in place
        s, w, rstd = self._call
        _, weighted, residual = self._given
        if not residual:
            gy, gs = g, None
        elif isinstance(g, _RowGradients):
            gy, gs = g.rows.get(0), g.rows.get(1)
        else:
            gy, gs = _row_of(g, 0), _row_of(g, 1)
        dtype, shape = s._storage._dtype, self._shape
        gy, gs = [None if t is None else _as_rows(reshape_view(t.to(dtype), shape))
                  for t in (gy, gs)]
        at = [0] + [len(needs) - 1] * residual  # x and the residual among the inputs
        summed = [i for i in at if needs[i]]
        ds, dw = K.rms_norm_bwd(s, w, rstd, gy, gs, bool(summed), weighted and needs[1])
        out = [None] * len(needs)
        if weighted and needs[1]:
            out[1] = _give(dw, shape[-1:], targets[1])
        for k, i in enumerate(summed):
            if k and targets[i] is None and targets[summed[0]] is None:
                # x and the residual have one gradient: one memory for both, but
                # where a leaf keeps it
                first = out[summed[0]]
                if share:
                    out[i] = first._alias()
                    first._shared = out[i]._shared = True
                else:
                    out[i] = _give(ds.clone(), shape, None)
            else:
                out[i] = _give(ds, shape, targets[i])
        return out

    @classmethod
    def flops(cls, x: Tensor, *args) -> int:
        return 4 * x.numel

    @classmethod
    def mem_bytes(cls, x: Tensor, weight=None, residual=None, *args) -> int:
        return (2 if residual is None else 4) * x.numel * sizeof(x.dtype)


class NormRowOp(RowOp):
    """Row i of RmsNormOp's [2, ...]: the tensor that it made, with a version
    of its own."""

    def forward(self, x: Tensor, i: int) -> Tensor:
        self._i, self._x = i, x
        return x._rows[i]._alias()


class AttentionOp(Function):
    """softmax(scale q . k) v over the keys that each query sees; see
    nanotorch_amd.attention."""

    def forward(self, q: Tensor, k: Tensor, v: Tensor, causal: int, lengths: Tensor | None,
                starts: Tensor | None, start: int, scale: float) -> Tensor:
        self._shapes = (q._shape, k._shape, v._shape)
        keep = is_grad_enabled() and any([t.requires_grad for t in (q, k, v)])
        views = [_heads(t) for t in (q, k, v)]
        call = (None if lengths is None else _vector(lengths),
                None if starts is None else _vector(starts), start, causal, scale)
        out, lse = K.attention(*views, *call, keep)
        y = Tensor._unchecked_view(out, q._shape, row_major_strides(q._shape), 0)
        if keep:
            given = [t for t in (lengths, starts) if t is not None]
            self.save_for_backward(q, k, v, *given, y._alias())
            self._call = (*views, *call, out, lse)
        return y

    def backward(self, grad_out: Tensor) -> tuple:
        return tuple(self._grad(grad_out, (True,) * 3, (None,) * 3))

    def fused_ok(self) -> bool:
        return True

    def _backward_into(self, g: Tensor, needs, targets):
        return self._grad(g, needs[:3], targets[:3]) + [None] * (len(needs) - 3)

    def _grad(self, g: Tensor, needs, targets) -> list:
        self.saved_tensors  # raises if one of them was modified in place
        q = self._call[0]
        g = _heads(reshape_view(g.to(q._storage._dtype), self._shapes[0]))
        new = K.attention_bwd(*self._call, g, needs)
        return [None if st is None else _give(st, shape, target)
                for st, shape, target in zip(new, self._shapes, targets)]

    @classmethod
    def flops(cls, q: Tensor, k: Tensor, *args) -> int:
        return 4 * q.numel * k.shape[-3]

    @classmethod
    def mem_bytes(cls, q: Tensor, k: Tensor, *args) -> int:
        return (2 * q.numel + 2 * k.numel) * sizeof(q.dtype)


def _heads(x: Tensor) -> Tensor:
    """x as [B, T, heads, D] with adjacent elements in a head; copied only where
    they are not."""
    if x._shape[-1] > 1 and x._strides[-1] != 1:
        x = x._to_contiguous(force=True)
    if len(x._shape) == 4:
        return x
    return Tensor._unchecked_view(x._storage, (1,) + x._shape, (0,) + x._strides, x._offset)


def check_attention(q: Tensor, k: Tensor, v: Tensor, lengths, starts) -> int:
    """Raises for operands that do not belong together; returns the number of
    sequences."""
    if len(q._shape) not in (3, 4) or not is_float(q._storage._dtype):
        raise ValueError(f"Queries are float [B, T, heads, D] or [T, heads, D], got "
                         f"{q.dtype.name} {q.shape}.")
    if any([t._storage._dtype != q._storage._dtype for t in (k, v)]):
        raise ValueError(f"Queries, keys and values have one dtype, got {q.dtype.name}, "
                         f"{k.dtype.name}, {v.dtype.name}.")
    if k._shape != v._shape:
        raise ValueError(f"Keys and values have one shape, got {k.shape} and {v.shape}.")
    if (len(k._shape) != len(q._shape) or k._shape[-1] != q._shape[-1]
            or k._shape[:-3] != q._shape[:-3]):
        raise ValueError(f"Queries {q.shape} and keys {k.shape} differ in sequences or in "
                         f"the heads' width.")
    heads, shared = q._shape[-2], k._shape[-2]
    if not shared or not heads or heads % shared:
        raise ValueError(f"{heads} query heads cannot share {shared} key heads evenly.")
    if not 1 <= q._shape[-1] <= 256:
        raise ValueError(f"Heads have 1 to 256 elements, got {q.shape[-1]}.")
    sequences = math.prod(q._shape[:-3])
    for what, t in (("lengths", lengths), ("starts", starts)):
        if t is None or what == "starts" and not isinstance(t, Tensor):
            continue
        if not isinstance(t, Tensor):
            raise TypeError(f"{what} are a Tensor, got {type(t).__name__}.")
        if not is_int(t._storage._dtype) or t._shape != (sequences,):
            raise ValueError(f"{what} are int32 or int64, one for each of {sequences} "
                             f"sequences, got {t.dtype.name} {t.shape}.")
    return sequences
