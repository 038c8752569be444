"""Differentiable ops of a model over token numbers: the embedding lookup,
dropout, and the log probabilities of given tokens with the rows' entropies.
The reference has none of them.

Each backward is one fused pass that writes a new gradient or adds into an
existing one (``_backward_into``), by way of a new one where that is of
another float type or its rows cannot be walked; token numbers have no
gradient.
"""

from __future__ import annotations

import math

from .. import _kernels as K
from .. import _lib
from .._data_type import Dtype, is_float, is_int, sizeof
from .._indexing import row_major_strides
from .._storage import Storage
from ..core import Tensor, reshape_view
from ..cuda import Device
from .function import Function
from .grad_mode import is_grad_enabled


def _check_tokens(tokens: Tensor) -> None:
    if not is_int(tokens._storage._dtype):
        raise ValueError(f"Tokens must be int32 or int64, got {tokens.dtype.name}.")


def _vector(x: Tensor) -> Tensor:
    """x as a 1-D view, copied only where it is neither 1-D nor contiguous."""
    return x if len(x._shape) == 1 else reshape_view(x, (x.numel,))


def _rows_in_place(x: Tensor) -> Tensor | None:
    """x [..., n] as a [rows, n] view of adjacent elements; None if its
    strides do not allow one."""
    shape, st = x._shape, x._strides
    if shape[-1] > 1 and st[-1] != 1:
        return None
    rows, step = 1, 0  # the leading axes merged so far, innermost first
    for s, t in zip(reversed(shape[:-1]), reversed(st[:-1])):
        if s == 1:
            continue
        if rows == 1:
            step = t
        elif t != step * rows:
            return None
        rows *= s
    if rows == 1:
        rows, step = math.prod(shape[:-1]), shape[-1]
    return Tensor._unchecked_view(x._storage, (rows, shape[-1]), (step, 1), x._offset)


def _as_rows(x: Tensor) -> Tensor:
    v = _rows_in_place(x)
    return v if v is not None else _rows_in_place(x._to_contiguous(force=True))


def _added(target: Tensor, storage, shape) -> Tensor:
    """Adds a new gradient's storage into `target` of any strides and float
    type."""
    new = Tensor._new_contiguous(storage, shape)
    K.inplace(_lib.ADD, target, new.to(target._storage._dtype))
    return target


class EmbeddingOp(Function):
    """scale * table[tokens]; zero rows where a token is padding_idx."""

    def forward(self, table: Tensor, tokens: Tensor, scale: float = 1.0,
                padding_idx: int | None = None) -> Tensor:
        shape = table._shape
        if len(shape) != 2 or not is_float(table._storage._dtype):
            raise ValueError(
                f"An embedding table is 2-D and float, got {table.dtype.name} {shape}.")
        _check_tokens(tokens)
        if padding_idx is None:
            padding_idx = -1
        elif not 0 <= padding_idx < shape[0]:
            raise ValueError(f"padding_idx {padding_idx} is no row of a table of {shape[0]}.")
        self.save_for_backward(tokens)
        self._scale, self._padding, self._shape = float(scale), padding_idx, shape
        self._dtype = table._storage._dtype
        self._flat = _vector(tokens)
        st = K.embedding(table, self._flat, self._scale, padding_idx)
        return Tensor._unchecked_view(
            st, tokens._shape + shape[1:], row_major_strides(tokens._shape + shape[1:]), 0)

    def backward(self, grad_out: Tensor) -> tuple:
        return (self._grad(grad_out, None), None)

    def fused_ok(self) -> bool:
        return True

    def _backward_into(self, g: Tensor, needs, targets):
        return [self._grad(g, targets[0]) if needs[0] else None, None]

    def _grad(self, g: Tensor, target: Tensor | None) -> Tensor:
        self.saved_tensors  # raises if the tokens were modified in place
        shape = self._shape
        g = reshape_view(g.to(self._dtype), (self._flat._shape[0], shape[1]))._to_contiguous()
        into = target
        if target is not None and ((shape[1] > 1 and target._strides[1] != 1)
                                   or target._storage._dtype != self._dtype):
            into = None
        st = K.embedding_bwd(g, self._flat, self._scale, self._padding, shape, into)
        if into is not None:
            return target
        if target is not None:
            return _added(target, st, shape)
        return Tensor._unchecked_view(st, shape, (shape[1], 1), 0)

    @classmethod
    def flops(cls, table: Tensor, tokens: Tensor, *args) -> int:
        return tokens.numel * table.shape[1]

    @classmethod
    def mem_bytes(cls, table: Tensor, tokens: Tensor, *args) -> int:
        return (tokens.numel * sizeof(tokens.dtype)
                + 2 * tokens.numel * table.shape[1] * sizeof(table.dtype))


class DropoutOp(Function):
    """x / (1 - p) where word i mod 4 of Philox4x32-10 (key seed, counter
    (i div 4, offset)) is at least round(p * 2^32), else 0, for the row-major
    index i.  The mask is drawn again in the backward pass, never stored."""

    def forward(self, x: Tensor, p: float, seed: int, offset: int) -> Tensor:
        if not is_float(x._storage._dtype):
            raise ValueError(f"dropout() needs a float tensor, got {x.dtype.name}.")
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout() needs 0 <= p <= 1, got {p}.")
        self._args = (float(p), seed, offset)
        self._dtype, self._shape = x._storage._dtype, x._shape
        return Tensor._unchecked_view(
            K.dropout(x, *self._args), x._shape, row_major_strides(x._shape), 0)

    def backward(self, grad_out: Tensor) -> tuple:
        return (self._grad(grad_out, None),)

    def fused_ok(self) -> bool:
        return True

    def _backward_into(self, g: Tensor, needs, targets):
        return [self._grad(g, targets[0]) if needs[0] else None]

    def _grad(self, g: Tensor, target: Tensor | None) -> Tensor:
        g = reshape_view(g.to(self._dtype), self._shape)
        into = target
        if target is not None and target._storage._dtype != self._dtype:
            into = None
        st = K.dropout(g, *self._args, into)
        if into is not None:
            return target
        if target is not None:
            return _added(target, st, g._shape)
        return Tensor._unchecked_view(st, g._shape, row_major_strides(g._shape), 0)

    @classmethod
    def flops(cls, x: Tensor, *args) -> int:
        return x.numel

    @classmethod
    def mem_bytes(cls, x: Tensor, *args) -> int:
        return 2 * x.numel * sizeof(x.dtype)


class TokenLogProbOp(Function):
    """Log probabilities of given tokens and entropies of rows of logits.

    Returns the one that is wanted, or both as [2, ...] (log probabilities
    first), so that one pass computes the logits' gradient of both.  The top
    alternatives go into `extras`; they have no gradient."""

    def forward(self, logits: Tensor, tokens: Tensor | None, ignore_index: int,
                entropy: bool, top: int, extras: list) -> Tensor:
        lead = logits._shape[:-1]
        z = _as_rows(logits)
        flat = None if tokens is None else _vector(tokens)
        keep = bool(is_grad_enabled() and logits.requires_grad)
        out, token = K.token_logprobs(z, flat, ignore_index, entropy, top, keep)
        if top:
            n = entropy + (tokens is not None)
            extras.extend(top_views(out, n * z._shape[0], token, lead + (top,)))
        self._both = entropy and tokens is not None
        if keep:
            self.save_for_backward(*((logits,) if tokens is None else (logits, tokens)))
            self._call = (z, flat, ignore_index, out)
            self._shape = logits._shape
        shape = (2,) + lead if self._both else lead
        return Tensor._unchecked_view(out, shape, row_major_strides(shape), 0)

    def backward(self, grad_out: Tensor) -> tuple:
        return (self._grad(grad_out, None), None)

    def fused_ok(self) -> bool:
        return True

    def _backward_into(self, g: Tensor, needs, targets):
        none = [None] * (len(needs) - 1)
        return [self._grad(g, targets[0]) if needs[0] else None] + none

    def _grad(self, g: Tensor, target: Tensor | None) -> Tensor:
        self.saved_tensors  # raises if logits or tokens were modified in place
        z, flat, ignore, results = self._call
        rows = z._shape[0]
        if not self._both:
            ga, gb = (None, g) if flat is None else (g, None)
        elif isinstance(g, _RowGradients):
            ga, gb = g.rows.get(0), g.rows.get(1)
        else:
            g = reshape_view(g, (2, rows))._to_contiguous()
            ga, gb = _row_of(g, 0), _row_of(g, 1)
        dtype = z._storage._dtype
        ga, gb = [x if x is None else _vector(x if x._storage._dtype == dtype else x.to(dtype))
                  for x in (ga, gb)]
        into = None
        if target is not None and target._storage._dtype == dtype:
            into = _rows_in_place(target)
        st = K.token_logprobs_bwd(z, flat, ignore, results, ga, gb, into)
        if into is not None:
            return target
        if target is not None:
            return _added(target, st, self._shape)
        return Tensor._unchecked_view(st, self._shape, row_major_strides(self._shape), 0)

    @classmethod
    def flops(cls, logits: Tensor, *args) -> int:
        return 5 * logits.numel

    @classmethod
    def mem_bytes(cls, logits: Tensor, *args) -> int:
        return logits.numel * sizeof(logits.dtype)


def top_views(out, offset: int, token, shape) -> tuple[Tensor, Tensor]:
    """The alternatives' log probabilities, in `out` from `offset` on with a
    version of their own, and their tokens."""
    strides = row_major_strides(shape)
    if offset:
        out = out.part(offset, token._size)
    return (Tensor._unchecked_view(out, shape, strides, 0),
            Tensor._unchecked_view(token, shape, strides, 0))


class _RowGradients(Tensor):
    """The gradient of TokenLogProbOp's x [2, ...] while the engine carries it:
    the gradients of its rows as they arrived, not copied into one tensor, as
    on few rows three launches are most of what the backward pass costs.

    It has no memory, so nothing but TokenLogProbOp can take it for values; a
    copy of it, which the engine makes of gradients that may be shared, is the
    same object."""

    _NONE = Storage(0, Dtype.Float32, Device.Cpu)

    @classmethod
    def of(cls, x: Tensor) -> "_RowGradients":
        new = cls._unchecked_view(cls._NONE, x._shape, x._strides, 0)
        new.rows = {}
        return new

    def _to_contiguous(self, force: bool = False) -> Tensor:
        return self


def result_row(x: Tensor, i: int) -> Tensor:
    """x[i] of TokenLogProbOp's x [2, ...], with a version of its own: a change
    of one row in place leaves a graph that needs the other."""
    shape = x._shape[1:]
    if i == 0:  # x itself is no one's result
        return Tensor._unchecked_view(x._storage, shape, x._strides[1:], 0)
    n = math.prod(shape)
    return Tensor._unchecked_view(x._storage.part(n, n), shape, x._strides[1:], 0)


class RowOp(Function):
    """result_row, differentiable."""

    def forward(self, x: Tensor, i: int) -> Tensor:
        self._i, self._x = i, x
        return result_row(x, i)

    def backward(self, grad_out: Tensor) -> tuple:
        full = Tensor._new_contiguous(
            K.fill(self._x.numel, 0, grad_out.dtype, grad_out.device), self._x._shape)
        K.copy_view(grad_out, _row_of(full, self._i))
        return (full,)

    def fused_ok(self) -> bool:
        return True

    def _backward_into(self, g: Tensor, needs, targets):
        if not needs[0]:
            return [None]
        into = targets[0]
        if into is None:
            into = _RowGradients.of(self._x)
        elif not isinstance(into, _RowGradients):
            K.inplace(_lib.ADD, _row_of(into, self._i), g)
            return [into]
        into.rows[self._i] = g
        return [into]


def _row_of(x: Tensor, i: int) -> Tensor:
    return Tensor._unchecked_view(
        x._storage, x._shape[1:], x._strides[1:], x._offset + i * x._strides[0])

