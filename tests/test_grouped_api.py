"""What the Python operators of the grouped products hand to the C functions, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

from ops_sparse_b200 import _lib as L
from ops_sparse_b200 import api


class Recorded(api._Grouped):
    """A product whose C functions note the scalars that they are given."""

    name = "product"

    def __init__(self, monkeypatch):
        self.seen = []

        class Lib:
            def __getattr__(lib, name):
                return self.take

        monkeypatch.setattr(L, "lib", Lib)
        self.buffer = torch.empty(64, dtype=torch.uint8)

    def _args(self, pa, pb):
        return pa, pb

    def take(self, pa, pb, last):
        self.seen.append(tuple(ctypes.cast(p, ctypes.POINTER(ctypes.c_float))[0] for p in (pa, pb)))
        return L.SUCCESS


@pytest.mark.parametrize("make", [lambda v: torch.tensor(v), lambda v: torch.tensor([v]), lambda v: np.full((), v)])
def test_a_scalar_that_changes_its_value_is_read_at_every_call(monkeypatch, make):
    op = Recorded(monkeypatch)
    beta = make(0.5)
    op(1.0, beta)
    beta[...] = 2.0
    op(1.0, beta)
    op(2, np.float32(0.25))
    op(True, 1)
    assert op.seen[-4:] == [(1.0, 0.5), (1.0, 2.0), (2.0, 0.25), (1.0, 1.0)]


def shifted(shape, stride, shift, dtype=torch.float16):
    store = torch.zeros(shift + 1 + sum((n - 1) * s for n, s in zip(shape, stride)), dtype=dtype)
    assert store.data_ptr() % 16 == 0
    return store[shift:].as_strided(shape, stride, store.storage_offset() + shift)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.int8])
def test_adapter_copies_operands_that_are_merely_shifted(dtype):
    """One row, one matrix, one column: the strides of what there is only one of do not make an operand odd."""
    from ops_sparse_b200 import torch_adapter as A
    rows, batch = A._rows_descr, A._batch_descr
    for describe, shape, stride in ((rows, (1, 784), (777, 1)), (rows, (3, 784), (784, 1)), (rows, (1, 784), (1, 1)),
                                    (rows, (5, 16), (800, 1)), (batch, (1, 9, 784), (6993, 784, 1)),
                                    (batch, (1, 1, 784), (6993, 777, 1)), (batch, (3, 1, 784), (784, 777, 1)),
                                    (batch, (1, 784, 9), (7001, 1, 784))):
        for shift in (1, 3, 15):
            t = shifted(shape, stride, shift, dtype)
            t.copy_(torch.arange(t.numel()).reshape(shape) % 100)
            d = A._loadable(describe, t)
            assert d.values.data_ptr() % 16 == 0 and torch.equal(d.values, t)
            assert d.ld == {3: lambda: d.ld, 2: lambda: d.values.stride(0) if shape[0] > 1 else shape[1]}[len(shape)]()
        d = A._loadable(describe, shifted(shape, stride, 0, dtype))
        assert d.values.data_ptr() % 16 == 0
    # rows that the library copies anyway are described as they are, wherever they start
    for describe, shape, stride in ((rows, (1, 777), (784, 1)), (rows, (3, 777), (777, 1)), (batch, (2, 5, 48), (777, 48, 1)),
                                    (batch, (1, 784, 1), (7001, 1, 777))):  # the last: rows of one element, one apart
        t = shifted(shape, stride, 1, dtype)
        assert A._loadable(describe, t).values.data_ptr() == t.data_ptr()


@pytest.mark.parametrize("dtype", [torch.complex32, torch.complex64])
def test_adapter_resolves_views_that_stand_for_a_negative(dtype):
    """The imaginary part of a conjugate is the memory's negative, not the memory."""
    from ops_sparse_b200 import torch_adapter as A
    z = torch.arange(48, dtype=torch.float32).to(dtype) * 1j
    for describe, shape in ((A._rows_descr, (48, 1)), (A._rows_descr, (6, 8)), (A._batch_descr, (2, 3, 8)), (A._batch_descr, (2, 24, 1))):
        t = z.reshape(shape).conj().imag
        assert t.is_neg()
        d = describe(t)
        assert not d.values.is_neg()
        assert torch.equal(d.values.float().flatten(), -torch.arange(48, dtype=torch.float32))


def test_count_of_wait_failures_refuses_no_result(lib):
    assert lib.aclsparseB200GroupedMMTotalWaitFailures(None, None) == L.INVALID_VALUE


def test_a_product_without_results_needs_no_gpu(lib):
    h, one, made = ctypes.c_void_p(None), ctypes.byref(ctypes.c_float(1.0)), []
    assert lib.aclsparseCreate(ctypes.byref(h)) == L.SUCCESS
    for rows, cols in ((0, 16), (24, 16), (0, 24)):
        d = ctypes.c_void_p(None)
        assert lib.aclsparseCreateDnMat(ctypes.byref(d), rows, cols, cols, 0x10000, L.ACL_BF16, L.ORDER_ROW) == L.SUCCESS
        made.append(d)
    buffer = np.zeros(1 << 17, np.uint8)  # what stands for the device's memory where there is none
    if not torch.cuda.is_available():
        at = buffer.ctypes.data + -buffer.ctypes.data % 64
        assert lib.aclsparseB200GroupedMM(h, L.OP_T, one, made[0], None, made[1], None, None, one, made[2], L.ACL_FLOAT, at) == L.SUCCESS
    for d in made:
        assert lib.aclsparseDestroyDnMat(d) == L.SUCCESS
    assert lib.aclsparseDestroy(h) == L.SUCCESS
