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


SLOW = """
#include <cuda_runtime.h>
// Lets the next kernel of the stream start at once, and ends after `ns` nanoseconds.
__global__ void Slow(unsigned long long ns)
{
    asm volatile("griddepcontrol.launch_dependents;");
    unsigned long long began, now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(began));
    do {
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    } while (now - began < ns);
}
extern "C" int slow(unsigned long long ns, void* stream)
{
    Slow<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(ns);
    return static_cast<int>(cudaGetLastError());
}
"""


@pytest.fixture(scope="module")
def slow(tmp_path_factory):
    """A kernel as other libraries may have them: its dependents start early, and it takes its time."""
    import os
    import subprocess
    nvcc = "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no CUDA compiler")
    where = tmp_path_factory.mktemp("slow")
    (where / "slow.cu").write_text(SLOW)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", str(where / "slow.cu"),
                    "-o", str(where / "slow.so")], check=True)
    fn = ctypes.CDLL(str(where / "slow.so")).slow
    fn.argtypes, fn.restype = [ctypes.c_uint64, ctypes.c_void_p], ctypes.c_int
    return fn


BEHIND = {"narrow": dict(rows=20, n=600, k=1000), "wide": dict(rows=2000, n=1000, k=512),
          "many tiles": dict(rows=2500, n=5000, k=128), "gradient, cut": dict(rows=1003, n=520, m=264),
          "gradient, many tiles": dict(rows=1003, n=4000, m=4000)}


@pytest.mark.parametrize("offsets", [False, True])
@pytest.mark.parametrize("form", list(BEHIND))
def test_the_limit_of_a_wait_does_not_count_the_kernel_before(slow, form, offsets):
    """A product that starts 200 ms before the kernel in front of it ends, and may wait for 20 ms."""
    case = Long(**BEHIND[form])
    rows = torch.tensor([0, case.p.rows], dtype=torch.int32, device=DEV)
    case.p.offsets = rows.data_ptr() if offsets else None
    case.clear()
    case.run(0)
    torch.cuda.synchronize()
    want = case.c.clone()
    case.c[:-GUARD] = 0
    case.clear()
    torch.cuda.synchronize()
    assert slow(200_000_000, case.stream) == 0
    case.run(20_000_000)
    assert case.failures() == 0
    assert torch.equal(case.c, want) and not (want[:-GUARD] == 0).all()


def test_failures_outlive_the_buffer_and_the_next_product():
    """What the adapter's user can ask: its buffers are gone after each call, and cleared before each."""
    from ops_sparse_b200 import torch_adapter as A
    case = Long(**LONG["several tiles"])
    case.clear()
    before = A.wait_failures()
    case.run(1)
    after = A.wait_failures()
    assert 1 <= after - before <= 148
    case.clear()                        # as a product does that finds no Preprocess
    case.run(0)
    assert case.failures() == 0         # the buffer's own count speaks of that product alone
    del case
    x, w = torch.randn(40, 64, device=DEV).bfloat16(), torch.randn(1, 48, 64, device=DEV).bfloat16()
    y = A.grouped_mm(x, w)
    assert torch.isfinite(y).all() and A.wait_failures(DEV) == after == api.grouped_wait_failures()


def test_counts_are_refused_in_a_capture_and_leave_it_alone():
    x, w = torch.randn(300, 512, device=DEV).bfloat16(), torch.randn(1, 256, 512, device=DEV).bfloat16()
    c = torch.zeros(300, 256, device=DEV)
    side = torch.cuda.Stream()
    op = api.GroupedMM(api.Handle(side), api.DnMat(300, 512, 512, x), api.DnMat(256, 512, 512, w), api.DnMat(300, 256, 256, c),
                       op_b=L.OP_T)
    op.allocate()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        op()
        for ask in (op.wait_failures, api.grouped_wait_failures):
            with pytest.raises(api.AclsparseError) as refused:
                ask()
            assert refused.value.status == L.NOT_SUPPORTED
    graph.replay()
    torch.cuda.synchronize()
    assert op.wait_failures() == 0
    want = x.double() @ w[0].double().T
    assert ((c.double() - want).abs() <= 520 * 2.0 ** -23 * (x.double().abs() @ w[0].double().abs().T)).all()
