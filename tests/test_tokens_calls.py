"""What the token operators hand to the library, recorded in place of it: the
memory that views cover, and the gradients that reach the backward pass.  No
device is needed."""

from __future__ import annotations

import collections
import math
import struct

import numpy as np
import pytest

import nanotorch_amd as nt
from nanotorch_amd import _kernels as K
from nanotorch_amd import _lib
from nanotorch_amd._data_type import Dtype, sizeof
from nanotorch_amd._storage import Storage
from nanotorch_amd.autograd.function import Function
from nanotorch_amd.core import Tensor
from nanotorch_amd.cuda import Device

View = collections.namedtuple("View", "ptr offset dtype shape strides")


def parse(view: bytes) -> View:
    f = struct.unpack("=Qqii16q", view)
    return View(f[0], f[1], Dtype(f[2]), f[4:4 + f[3]], f[12:12 + f[3]])


class Recorder:
    """Stands in for the library: addresses that no memory is behind, calls
    that do nothing but are kept."""

    def __init__(self) -> None:
        self.sizes: dict[int, int] = {}  # bytes of each allocation
        self.freed: list[int] = []
        self.calls: list[tuple[str, tuple]] = []

    def nt_malloc(self, p, nbytes) -> int:
        p._obj.value = (1 << 40) * (len(self.sizes) + 1)
        self.sizes[p._obj.value] = int(nbytes)
        return 0

    def nt_free(self, ptr) -> int:
        self.freed.append(ptr)
        return 0

    def __getattr__(self, name):
        def call(*args) -> int:
            self.calls.append((name, args))
            return 0
        return call

    __getitem__ = __getattr__

    def args(self, name: str) -> tuple:
        """Of the last such call, views parsed."""
        found = [a for n, a in self.calls if n == name][-1]
        return tuple(parse(a) if isinstance(a, bytes) else a for a in found)

    def within(self, v: View) -> range:
        """The bytes of a contiguous view, which its allocation has to hold."""
        item, n = sizeof(v.dtype), math.prod(v.shape)
        base = v.ptr // (1 << 40) * (1 << 40)
        beg = v.ptr - base + v.offset * item
        assert 0 <= beg and beg + n * item <= self.sizes[base], v
        return range(base + beg, base + beg + n * item)


@pytest.fixture
def lib(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(_lib, "_lib", r)
    monkeypatch.setattr(_lib, "_packed", r)
    return r


def tensor(*shape, dtype=Dtype.Float32, requires_grad=False) -> Tensor:
    shape = tuple(int(n) for n in shape)
    t = Tensor._new_contiguous(Storage.allocate(math.prod(shape), dtype, Device.Cuda), shape)
    t._requires_grad = requires_grad
    return t


@pytest.mark.parametrize("size", [7, np.int64(7), np.uint8(200), np.int32(600_000_000),
                                  np.int32(1_200_000_000), True])
def test_an_allocation_holds_its_elements(lib, size):
    """Sizes of numpy's small integers, whose products with an element's size
    do not fit them."""
    st = Storage.allocate(size, Dtype.Float64, Device.Cuda)
    assert lib.sizes[st.data_ptr()] == int(size) * 8
    assert type(st.size) is int and st.nbytes == int(size) * 8


@pytest.mark.parametrize("rows,V", [(np.uint8(200), 64), (np.int32(3_000_000), 1000)])
def test_outputs_of_small_integer_shapes(lib, rows, V):
    """Shapes hold what they were given, numpy's small integers too."""
    z, w = tensor(rows, V), tensor(50, V)
    z._shape = (rows, V)  # as reshape keeps it
    t = tensor(rows, dtype=Dtype.Int64)
    t._shape = (rows,)
    lib.calls.clear()
    K.embedding(w, t, 1.0, -1)
    lib.within(lib.args("nt_embedding")[4])
    K.embedding_bwd(z, t, 1.0, -1, (rows, V), None)
    assert len(lib.within(lib.args("nt_embedding_bwd")[4])) == int(rows) * V * 4
    out, _ = K.token_logprobs(z, t, -100, True, 2, True)
    for v in lib.args("nt_token_logprobs")[3:]:
        lib.within(v)
    K.token_logprobs_bwd(z, t, -100, out, None, None, None)
    assert len(lib.within(lib.args("nt_token_logprobs_bwd")[6])) == int(rows) * V * 4


@pytest.mark.parametrize("entropy", [np.True_, np.False_, 1, 2, "yes", "", None])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("grad", [False, True])
def test_entropy_is_a_truth_value(lib, entropy, top, grad):
    """The results lie side by side in their allocation, whatever the truth
    value's type: True + numpy's True is one result, not two."""
    z, t = tensor(700, 20, requires_grad=grad), tensor(700, dtype=Dtype.Int64)
    out = nt.token_logprobs(z, t, entropy=entropy, top=top)
    assert (out.entropy is not None) == bool(entropy)
    _, _, _, logprob, ent, stats, value, token = lib.args("nt_token_logprobs")
    assert (ent is None, stats is None, value is None) == (not entropy, not grad, not top)
    used = [lib.within(v) for v in (logprob, ent, stats, value, token) if v is not None]
    for i, a in enumerate(used):
        for b in used[:i]:
            assert a.stop <= b.start or b.stop <= a.start


@pytest.mark.parametrize("flag", [True, 1, 2, "yes"])
@pytest.mark.parametrize("entropy,top", [(False, 0), (True, 2)])
def test_the_backward_pass_reads_the_statistics_written(lib, flag, entropy, top):
    """requires_grad is taken by its truth; the constructor keeps what it was
    given."""
    z, t = tensor(30, 20, requires_grad=flag), tensor(30, dtype=Dtype.Int64)
    out = nt.token_logprobs(z, t, entropy=entropy, top=top)
    written = lib.args("nt_token_logprobs")[5]
    out.logprob.sum().backward()
    assert lib.within(lib.args("nt_token_logprobs_bwd")[3]) == lib.within(written)


class Hands(Function):
    """Over (logprob, entropy), with the backward pass's results given."""

    def forward(self, x, y, grads):
        self._grads = grads
        return tensor()

    def backward(self, grad_out):
        return self._grads(*self.inputs[:2])


@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
@pytest.mark.parametrize("which", ["itself", "other", "upstream", "new"])
@pytest.mark.parametrize("rows", [4, 0])
def test_row_gradients_reach_the_backward_pass(lib, rows, which, order):
    """Gradients that are the results' own tensors, one tensor for both, or
    new ones: the backward pass reads each as it is, and nothing else runs."""
    z, t = tensor(rows, 20, requires_grad=True), tensor(rows, dtype=Dtype.Int64)
    out = nt.token_logprobs(z, t, entropy=True)
    one = tensor(rows)
    grads = {"itself": lambda x, y: (x, y), "other": lambda x, y: (y, x),
             "upstream": lambda x, y: (one, one),
             "new": lambda x, y: (tensor(rows), tensor(rows))}[which]
    given = {}

    def record(x, y):
        given["all"] = grads(x, y)
        return given["all"]

    pair = [out.logprob, out.entropy]
    loss = Hands.apply(pair[order[0]], pair[order[1]], record)
    lib.calls.clear()
    loss.backward()
    assert [n for n, _ in lib.calls if n != "nt_fill"] == ["nt_token_logprobs_bwd"]
    got = lib.args("nt_token_logprobs_bwd")[4:6]
    for k, g in zip(order, given["all"]):
        assert got[k][:4] == (g.storage.data_ptr(), g.strides[1], g.dtype, (rows,))


@pytest.mark.parametrize("i", [0, 1])
def test_one_row_gradient_reaches_the_backward_pass(lib, i):
    z, t = tensor(4, 20, requires_grad=True), tensor(4, dtype=Dtype.Int64)
    out = nt.token_logprobs(z, t, entropy=True)
    out[i].sum().backward()
    got = lib.args("nt_token_logprobs_bwd")[4:6]
    assert got[i] is not None and got[1 - i] is None


NAMES = ["logprob", "entropy", "top_logprobs", "top_tokens"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("wanted", [NAMES, ["logprob", "top_logprobs", "top_tokens"],
                                    ["entropy", "top_logprobs"], ["logprob", "entropy"]])
def test_each_result_has_a_version_of_its_own(lib, wanted, grad):
    z, t = tensor(40, 20, requires_grad=grad), tensor(40, dtype=Dtype.Int64)
    out = nt.token_logprobs(z, t if "logprob" in wanted else None, entropy="entropy" in wanted,
                            top=3 * ("top_logprobs" in wanted))
    for name in wanted:
        before = {n: getattr(out, n).version for n in wanted}
        x = getattr(out, name)
        with nt.no_grad():
            x += x
        after = {n: getattr(out, n).version for n in wanted}
        assert [n for n in wanted if after[n] != before[n]] == [name]


@pytest.mark.parametrize("last", NAMES)
def test_results_keep_their_memory(lib, last):
    """The results' allocation goes back with the last of them."""
    z, t = tensor(40, 20), tensor(40, dtype=Dtype.Int64)
    with nt.no_grad():
        out = nt.token_logprobs(z, t, entropy=True, top=3)
    x = getattr(out, last)
    used = lib.within(View(x.storage.data_ptr(), x.strides[1], x.dtype, x.shape, None))
    assert len(used) == x.numel * sizeof(x.dtype)
    base = used.start // (1 << 40) * (1 << 40)
    del out
    assert base not in lib.freed
    del x
    assert lib.freed.count(base) == 1
    assert len(lib.freed) == 2  # the results and the alternatives' tokens


def test_dropout_seeds_and_offsets(lib):
    x = tensor(5)
    nt.manual_seed(9)
    for given, want in (({}, (9, 0)), ({"seed": 3}, (3, 0)), ({"seed": 3, "offset": 7}, (3, 7)),
                        ({"seed": 0, "offset": 0}, (0, 0)), ({}, (9, 1)),
                        ({"seed": -1, "offset": -1}, (2 ** 64 - 1, 2 ** 64 - 1))):
        nt.dropout(x, 0.5, **given)
        assert lib.args("nt_dropout")[2:4] == want


@pytest.mark.parametrize("op", ["embedding", "dropout", "logprob", "entropy"])
def test_gradients_on_the_host_are_refused(lib, op):
    x, t = tensor(6, 5, requires_grad=True), tensor(6, dtype=Dtype.Int64)
    y = {"embedding": lambda: nt.embedding(x, t), "dropout": lambda: nt.dropout(x, 0.5),
         "logprob": lambda: nt.token_logprobs(x, t).logprob,
         "entropy": lambda: nt.token_logprobs(x, entropy=True).entropy}[op]()
    lib.calls.clear()
    with pytest.raises(RuntimeError):
        y.grad_fn.backward(nt.ones(*y.shape))
    needs = [True] * sum(isinstance(a, Tensor) for a in y.grad_fn.inputs)
    targets = [nt.ones(6, 5)] + [None] * (len(needs) - 1)
    with pytest.raises(RuntimeError):
        y.grad_fn._backward_into(tensor(*y.shape), needs, targets)
    assert not lib.calls


@pytest.mark.parametrize("op", ["embedding", "dropout", "logprob"])
def test_gradients_of_another_size_are_refused(lib, op):
    """Of another shape they are taken in row-major order, as by the other
    operators."""
    x, t = tensor(6, 5, requires_grad=True), tensor(6, dtype=Dtype.Int64)
    y = {"embedding": lambda: nt.embedding(x, t), "dropout": lambda: nt.dropout(x, 0.5),
         "logprob": lambda: nt.token_logprobs(x, t).logprob}[op]()
    if op != "logprob":  # its library call checks one gradient per row
        for shape in ((5, 5), (30, 2), (1,), ()):
            with pytest.raises((RuntimeError, ValueError)):
                y.grad_fn.backward(tensor(*shape))
    (dx, *_) = y.grad_fn.backward(tensor(*y.shape[::-1]))
    assert dx.shape == (6, 5)


def test_ignore_index_fits_64_bits(lib):
    z, t = tensor(6, 5), tensor(6, dtype=Dtype.Int64)
    for bad in (2 ** 63, 2 ** 64, -2 ** 63 - 1, 2 ** 64 - 100):
        with pytest.raises(ValueError):
            nt.token_logprobs(z, t, ignore_index=bad)
    for good in (-2 ** 63, 2 ** 63 - 1, -100, 0, np.int32(-1)):
        nt.token_logprobs(z, t, ignore_index=good)
        assert lib.args("nt_token_logprobs")[2] == good


@pytest.mark.parametrize("i", [0, 1])
def test_a_row_gradient_is_added_to_a_plain_one(lib, i):
    """As the ops' contract has it; the engine itself never holds one here."""
    z, t = tensor(4, 20, requires_grad=True), tensor(4, dtype=Dtype.Int64)
    op = nt.token_logprobs(z, t, entropy=True)[i].grad_fn
    both, g = tensor(2, 4), tensor(4)
    assert op._backward_into(g, [True], [both]) == [both]
    _, out, other = lib.args("nt_inplace")
    assert out[:4] == (both.storage.data_ptr(), 4 * i, Dtype.Float32, (4,))
    assert other.ptr == g.storage.data_ptr()
    (full,) = op.backward(g)
    assert full.shape == (2, 4)
    assert lib.args("nt_copy")[1][:2] == (full.storage.data_ptr(), 4 * i)
