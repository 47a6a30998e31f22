"""Bounded waits of the grouped products: a wait that runs out ends the kernel, is counted, and leaves the GPU and its
buffer usable.

The launch parameter waitLimitNs makes healthy waits run out: a tile's sums are waited for while the tile computes, for
milliseconds here, and the clock is looked at twice within one.  Nothing is missing or out of range in these products."""
import ctypes

import pytest
import torch

from ops_sparse_b200 import _lib as L
from ops_sparse_b200 import api

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = 2          # ACLSP_TYPE_BF16
OVERLAP = 8       # elements from row to row: the operands' rows overlap, so that long sums need little memory
GUARD = 64


class Long:
    """A product whose tiles take milliseconds, launched through the shim.  Forward: rows x n results, sums over k;
    gradient: m x n results, sums over the rows."""

    def __init__(self, rows, n, k=0, m=0):
        gen = torch.Generator(device=DEV).manual_seed(1)
        self.gradient = m != 0
        length, outer = (rows, m) if self.gradient else (k, rows)
        size = length + OVERLAP * max(outer, n) if not self.gradient else OVERLAP * rows + max(m, n)
        self.a = torch.randn(size, generator=gen, device=DEV).bfloat16()
        self.b = torch.randn(size, generator=gen, device=DEV).bfloat16()
        self.c = torch.full((outer * n + GUARD,), 7.0, device=DEV)
        p = self.p = L.GroupedParams()
        p.rows, p.groups, p.n, p.inType, p.outType = rows, 1, n, BF16, 0
        if self.gradient:
            p.weightGrad, p.m = 1, m
            p.aOuter, p.aInner, p.bOuter, p.bInner = 1, OVERLAP, 1, OVERLAP
        else:
            p.k = k
            p.aOuter, p.aInner, p.bOuter, p.bInner = OVERLAP, 1, OVERLAP, 1
        p.ldc, p.alpha = n, 1.0
        self.buffer = torch.empty(L.lib().aclsp_b200_grouped_buffer_bytes(ctypes.byref(p)), dtype=torch.uint8, device=DEV)
        self.stream = torch.cuda.current_stream().cuda_stream

    def clear(self):
        L.lib().aclsp_b200_grouped_preprocess_kernel_do(self.buffer.data_ptr(), self.stream)

    def run(self, limit_ns):
        self.p.waitLimitNs = limit_ns
        L.lib().aclsp_b200_grouped_mm_kernel_do(self.a.data_ptr(), self.b.data_ptr(), self.c.data_ptr(),
                                                self.buffer.data_ptr(), ctypes.byref(self.p), self.stream)

    def failures(self):
        count = ctypes.c_uint32(0)
        assert L.lib().aclsparseB200GroupedMMWaitFailures(self.stream, self.buffer.data_ptr(), ctypes.byref(count)) == L.SUCCESS
        return count.value


LONG = {"single": dict(rows=120, n=148 * 128, k=2 ** 20),
        "several tiles": dict(rows=120, n=3 * 148 * 128, k=2 ** 19),
        "pair": dict(rows=250, n=74 * 256, k=2 ** 20),
        "pair, several tiles": dict(rows=250, n=3 * 74 * 256, k=2 ** 19),
        "gradient, cut": dict(rows=2 ** 19 + 5, n=3328, m=3328)}


@pytest.mark.parametrize("form", list(LONG))
def test_a_wait_that_runs_out_ends_the_product_and_is_counted(form):
    case = Long(**LONG[form])
    case.clear()
    case.run(0)
    torch.cuda.synchronize()
    want = case.c.clone()
    assert case.failures() == 0 and (want[-GUARD:] == 7).all() and not (want[:-GUARD] == 7).all()
    case.run(1)
    torch.cuda.synchronize()
    assert 1 <= case.failures() <= 148 and (case.c[-GUARD:] == 7).all()
    # the query has cleared the counters: the same buffer serves again
    case.c[:-GUARD] = 0
    case.run(0)
    torch.cuda.synchronize()
    assert case.failures() == 0 and torch.equal(case.c, want)
