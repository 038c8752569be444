"""Functional forms of the Tensor ops (reference: src/nanotorch/ops.py)."""

from __future__ import annotations

import math
import operator
from typing import NamedTuple

from . import _kernels as K
from . import _lib
from . import autograd
from ._data_type import Dtype, is_float, promote_dtypes
from ._indexing import broadcast_shapes
from .autograd.ops_token import RowOp, _as_rows, _check_tokens, result_row, top_views
from .autograd.ops_transformer import NormRowOp, check_attention
from .core import Tensor
from .factories import next_dropout_counter


def clone(x: Tensor) -> Tensor:
    return x.clone()


def reshape(x: Tensor, *dims: int) -> Tensor:
    return x.reshape(*dims)


def transpose(x: Tensor, dim0: int, dim1: int) -> Tensor:
    return x.transpose(dim0, dim1)


def flatten(x: Tensor) -> Tensor:
    return x.flatten()


def equals(x: Tensor, y: Tensor) -> bool:
    return x.equals(y)


def add(x, y) -> Tensor:
    return x + y


def subtract(x, y) -> Tensor:
    return x - y


def multiply(x, y) -> Tensor:
    return x * y


def divide(x, y) -> Tensor:
    return x / y


def eq(x, y) -> Tensor:
    return x == y


def gt(x, y) -> Tensor:
    return x > y


def geq(x, y) -> Tensor:
    return x >= y


def lt(x, y) -> Tensor:
    return x < y


def leq(x, y) -> Tensor:
    return x <= y


def negate(x: Tensor) -> Tensor:
    return -x


def matmul(x: Tensor, y: Tensor) -> Tensor:
    return x @ y


def sum(x: Tensor, axis=None, keepdim: bool = False, *, dtype: Dtype | None = None) -> Tensor:
    return x.sum(axis, keepdim, dtype=dtype)


def mean(x: Tensor, axis=None, keepdim: bool = False, *, dtype: Dtype | None = None) -> Tensor:
    return x.mean(axis, keepdim, dtype=dtype)


def exp(x: Tensor) -> Tensor:
    return x.exp()


def log(x: Tensor) -> Tensor:
    return x.log()


def pow(x: Tensor, exponent) -> Tensor:
    return x.pow(exponent)


def relu(x: Tensor) -> Tensor:
    return autograd.ReluOp.apply(x)


def tanh(x: Tensor) -> Tensor:
    return autograd.TanhOp.apply(x)


def sqrt(x: Tensor) -> Tensor:
    return autograd.SqrtOp.apply(x)


def sigmoid(x: Tensor) -> Tensor:
    return autograd.SigmoidOp.apply(x)


def embedding(table: Tensor, tokens: Tensor, scale: float = 1.0, *,
              padding_idx: int | None = None) -> Tensor:
    """scale * table[tokens]: the rows of a [V, D] float table that int32 or
    int64 tokens of any shape name, [*tokens.shape, D].

    A token equal to ``padding_idx`` gives a zero row and no gradient.  Tokens
    are checked on the device: one outside the table gives a zero row, and the
    next synchronisation (``sync``, ``cpu``) raises IndexError.  The table's
    gradient sums each row's terms in an order that the tokens alone fix, so it
    comes out the same every time."""
    return autograd.EmbeddingOp.apply(table, tokens, scale, padding_idx)


def dropout(x: Tensor, p: float = 0.5, *, seed: int | None = None,
            offset: int | None = None) -> Tensor:
    """x / (1 - p) with each element kept with probability 1 - p, else 0.

    Element i (row-major) is kept where word i mod 4 of Philox4x32-10 under the
    64-bit key ``seed`` at the counter (i div 4, ``offset``) is at least
    round(p * 2^32): one seed and offset give one mask, whatever x's strides,
    and the backward pass draws it again.  Without a seed every call takes the
    next offset of the generator that ``manual_seed`` sets, and none can be
    given; with one the offset is 0 unless given."""
    if seed is None:
        if offset is not None:
            raise ValueError("dropout() takes an offset only with a seed.")
        seed, offset = next_dropout_counter()
    return autograd.DropoutOp.apply(x, p, int(seed) & (2**64 - 1),
                                    int(offset or 0) & (2**64 - 1))


class TokenLogProbs(NamedTuple):
    """What token_logprobs returns; None for what was not asked for."""

    logprob: Tensor | None
    entropy: Tensor | None
    top_logprobs: Tensor | None
    top_tokens: Tensor | None


def token_logprobs(logits: Tensor, tokens: Tensor | None = None, *, entropy: bool = False,
                   top: int = 0, ignore_index: int = -100) -> TokenLogProbs:
    """Log probabilities under softmax over the last axis of float logits
    [..., V], in one pass over them.

    * ``logprob`` [...]: of the given int32 or int64 tokens [...];
    * ``entropy`` [...]: -sum p log p of each row, if asked for;
    * ``top_logprobs`` and ``top_tokens`` [..., top]: the most likely tokens,
      0 <= top <= min(V, 64), ties to the lowest token; without a gradient.

    ``logprob`` and ``entropy`` are differentiable, together in one pass.  A
    row whose token is ``ignore_index`` is left out: logprob and entropy 0, no
    gradient, alternatives -inf and -1.  Logits of -inf are tokens that cannot
    occur; a row of nothing else has logprob -inf, entropy 0 and no gradient.
    Tokens are checked on the device: one outside [0, V) leaves its row out,
    and the next synchronisation (``sync``, ``cpu``) raises IndexError."""
    shape, entropy = logits._shape, bool(entropy)
    if not shape or not is_float(logits._storage._dtype):
        raise ValueError(f"Logits are float with an axis of tokens, got {logits.dtype.name} "
                         f"{shape}.")
    if not -2**63 <= ignore_index < 2**63:  # the library's 64 bits would wrap round
        raise ValueError(f"ignore_index must fit 64 bits, got {ignore_index}.")
    if not 0 <= top <= min(shape[-1], 64):
        raise ValueError(f"top must lie in [0, min(V, 64)], got {top} with V = {shape[-1]}.")
    if tokens is None:
        if not entropy and not top:
            raise ValueError("token_logprobs() needs tokens, entropy=True or top > 0.")
    else:
        _check_tokens(tokens)
        if tokens._shape != shape[:-1]:
            raise ValueError(f"One token for each row of {shape[:-1]}, got {tokens.shape}.")
    extras = [] if top else [None, None]
    logprob = ent = None
    if tokens is None and not entropy:
        out, token = K.token_logprobs(_as_rows(logits), None, ignore_index, False, top, False)
        extras = top_views(out, 0, token, shape[:-1] + (top,))
    else:
        op, tracked = autograd.TokenLogProbOp, logits.requires_grad and autograd.is_grad_enabled()
        call = op.apply if tracked else op().forward  # a serving call has no node to attach
        out = call(logits, tokens, ignore_index, entropy, top, extras)
        if tokens is None:
            ent = out
        elif not entropy:
            logprob = out
        else:
            row = RowOp.apply if tracked else result_row
            logprob, ent = row(out, 0), row(out, 1)
    return TokenLogProbs(logprob, ent, *extras)


def rms_norm(x: Tensor, weight: Tensor | None = None, *, residual: Tensor | None = None,
             eps: float = 1e-6) -> Tensor | tuple[Tensor, Tensor]:
    """x (mean x^2 + eps)^-1/2 weight over the last axis of a float tensor.

    With a ``residual`` of x's shape, the sum s = x + residual takes x's place,
    and (y, s) is returned: s is what the next block adds to.  ``weight`` is
    1-D.  One pass forward; one backward for the gradients of both results,
    with the weight's summed in an order that the shape alone fixes."""
    out = autograd.RmsNormOp.apply(x, weight, residual, eps)
    if residual is None:
        return out
    rows = out._rows
    if out._grad_fn is None:
        return rows
    return NormRowOp.apply(out, 0), NormRowOp.apply(out, 1)


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool | None = None,
              lengths: Tensor | None = None, starts: Tensor | int | None = None,
              scale: float | None = None) -> Tensor:
    """softmax(scale q . k) v: queries [B, Tq, H, D] over keys and values
    [B, Tk, Hk, D], or all without B; returns [B, Tq, H, D].

    Hk divides H: query head h reads key head h // (H // Hk).  D is at most
    256, ``scale`` D**-0.5 unless given.  Query i of sequence b sees key j where

    * j < ``lengths[b]`` (int32 or int64 [B]; Tk unless given), and
    * if ``causal``, j <= ``starts[b]`` + i, with starts an int for all or an
      int32 or int64 tensor [B].  Unless given, the queries are the last ones of
      their sequences: starts = lengths - Tq.  (A batch of texts padded at
      their ends has starts=0.)

    With ``causal=False`` starts have no effect.  Starts without a word on causal,
    which is then False, are refused: their caller meant it to be True.

    A query that sees no key gives zeros and has no gradient.  What lies behind a length
    does not reach a result.  What a query does not see within it, later than
    itself, reaches no more than its result's rounding, whatever it holds.  Lengths are checked on the device: one
    outside [0, Tk] is taken as the nearer end, and the next synchronisation
    (``sync``, ``cpu``) raises IndexError.

    The probabilities are never stored: the backward pass forms them again.
    Every result comes out the same every time."""
    check_attention(q, k, v, lengths, starts)
    start, mode = 0, 0
    if starts is not None and causal is None:
        raise ValueError("attention() takes starts only where causal is given.")
    if causal:
        mode = 1 if starts is None else 2
    if starts is not None and not isinstance(starts, Tensor):
        start, starts = operator.index(starts), None  # TypeError for a float or a list
        if not -2**63 <= start < 2**63:  # the library's 64 bits would wrap round
            raise ValueError(f"starts must fit 64 bits, got {start}.")
    if not causal:
        start, starts = 0, None
    scale = q._shape[-1] ** -0.5 if scale is None else float(scale)
    # times log2 e in the operands' type, in which the kernels hold it
    if not abs(scale) < (2.0**127 if q._storage._dtype is Dtype.Float32 else 2.0**1023):
        raise ValueError(f"attention() needs a finite scale, got {scale}.")
    return autograd.AttentionOp.apply(q, k, v, mode, lengths, starts, start, scale)


def _arg_reduce(op: int, name: str, x: Tensor, axis, keepdim: bool) -> Tensor:
    if isinstance(axis, int):
        full_axis = (axis if axis >= 0 else axis + x.ndim,)
    elif axis is None:
        full_axis = tuple(range(x.ndim))
    else:
        raise ValueError(f"Axis must be int or None, found {type(axis)}")
    if keepdim:
        new_shape = tuple(1 if i in full_axis else s for i, s in enumerate(x.shape))
    else:
        new_shape = tuple(s for i, s in enumerate(x.shape) if i not in full_axis)
    if x.is_empty:
        if math.prod(new_shape) != 0:
            raise IndexError(f"{name}() expects reduction dim to be specified for numel=0.")
        return Tensor._new_contiguous(
            K.fill(math.prod(new_shape), 0, x.dtype, x.device), new_shape
        )
    return Tensor._new_contiguous(K.reduce(op, x, full_axis, Dtype.Int64), new_shape)


def argmin(x: Tensor, axis: int | None = None, keepdim: bool = False) -> Tensor:
    """Index of the first minimum along `axis` (flattened index if None)."""
    return _arg_reduce(_lib.R_ARGMIN, "argmin", x, axis, keepdim)


def argmax(x: Tensor, axis: int | None = None, keepdim: bool = False) -> Tensor:
    """Index of the first maximum along `axis` (flattened index if None)."""
    return _arg_reduce(_lib.R_ARGMAX, "argmax", x, axis, keepdim)


def _compare(op: int, x1: Tensor, x2: Tensor) -> Tensor:
    dtype = promote_dtypes(x1.dtype, x2.dtype)
    shape = broadcast_shapes(x1.shape, x2.shape)
    a = x1.to(dtype).expand(*shape)
    b = x2.to(dtype).expand(*shape)
    return Tensor._new_contiguous(K.binary(op, a, b), a.shape)


def equal_op_(x1: Tensor, x2: Tensor) -> Tensor:
    return _compare(_lib.EQ, x1, x2)


def greater_op_(x1: Tensor, x2: Tensor) -> Tensor:
    return _compare(_lib.GT, x1, x2)


def greater_eq_op_(x1: Tensor, x2: Tensor) -> Tensor:
    return _compare(_lib.GE, x1, x2)
