"""Refusals and bookkeeping of the grouped products and the row quantisation, decided before anything is launched."""
import ctypes
from ctypes import byref, c_float, c_size_t, c_void_p

import pytest

from ops_sparse_b200 import _lib as L

FAKE = [c_void_p(0x10000 + 0x1000 * i) for i in range(16)]
ONE = ctypes.cast(byref(c_float(1.0)), c_void_p)


@pytest.fixture()
def handle(lib):
    h = c_void_p(None)
    assert lib.aclsparseCreate(byref(h)) == L.SUCCESS
    yield h
    assert lib.aclsparseDestroy(h) == L.SUCCESS


@pytest.fixture()
def mat(lib):
    made = []

    def make(rows, cols, ld=None, dtype=L.ACL_BF16, order=L.ORDER_ROW, values=FAKE[0], batch=1, stride=None):
        d = c_void_p(None)
        ld = (cols if order == L.ORDER_ROW else rows) if ld is None else ld
        assert lib.aclsparseCreateDnMat(byref(d), rows, cols, ld, values, dtype, order) == L.SUCCESS
        if batch != 1:
            stride = (rows if order == L.ORDER_ROW else cols) * ld if stride is None else stride
            assert lib.aclsparseDnMatSetStridedBatch(d, batch, stride) == L.SUCCESS
        made.append(d)
        return d

    yield make
    for d in made:
        assert lib.aclsparseDestroyDnMat(d) == L.SUCCESS


def size_of(lib, h, a, b, c, offsets=FAKE[9], op=L.OP_T, compute=L.ACL_FLOAT, rs=None, cs=None, alpha=ONE, beta=ONE):
    size = c_size_t(0)
    st = lib.aclsparseB200GroupedMMGetBufferSize(h, op, alpha, a, offsets, b, rs, cs, beta, c, compute, byref(size))
    return st, size.value


def grad_size(lib, h, a, b, c, offsets=FAKE[9], compute=L.ACL_FLOAT):
    size = c_size_t(0)
    st = lib.aclsparseB200GroupedMMWeightGradGetBufferSize(h, ONE, a, b, offsets, ONE, c, compute, byref(size))
    return st, size.value


def test_forward_accepts_its_layouts_and_types(lib, handle, mat):
    for op, shape in ((L.OP_T, (24, 16)), (L.OP_H, (24, 16)), (L.OP_N, (16, 24))):
        for order in (L.ORDER_ROW, L.ORDER_COL):
            b = mat(*shape, order=order, batch=4)
            st, size = size_of(lib, handle, mat(10, 16), b, mat(10, 24), op=op)
            assert st == L.SUCCESS and size >= 64
    ok = {(L.ACL_BF16, L.ACL_BF16), (L.ACL_BF16, L.ACL_FLOAT), (L.ACL_FLOAT16, L.ACL_FLOAT16),
          (L.ACL_FLOAT16, L.ACL_FLOAT), (L.ACL_INT8, L.ACL_FLOAT), (L.ACL_INT8, L.ACL_FLOAT16), (L.ACL_INT8, L.ACL_BF16)}
    types = (L.ACL_FLOAT, L.ACL_FLOAT16, L.ACL_BF16, L.ACL_INT8, L.ACL_INT32)
    for t in types:
        for u in types:
            for out in types:
                got, _ = size_of(lib, handle, mat(10, 16, dtype=t), mat(24, 16, dtype=u, batch=2), mat(10, 24, dtype=out))
                assert got == (L.SUCCESS if t == u and (t, out) in ok else L.NOT_SUPPORTED), (t, u, out)
    b = mat(24, 16, batch=2)
    assert size_of(lib, handle, mat(10, 16), b, mat(10, 24), compute=L.ACL_INT32)[0] == L.NOT_SUPPORTED
    assert size_of(lib, handle, mat(10, 16), mat(24, 16), mat(10, 24), offsets=None)[0] == L.SUCCESS
    # nothing to read and nothing to write
    assert size_of(lib, handle, mat(0, 16, values=None), b, mat(0, 24, values=None))[0] == L.SUCCESS
    assert size_of(lib, handle, mat(10, 0, values=None), mat(24, 0, values=None, batch=2), mat(10, 24))[0] == L.SUCCESS


def test_forward_refusals(lib, handle, mat):
    a, b, c = mat(10, 16), mat(24, 16, batch=3), mat(10, 24)
    assert size_of(lib, None, a, b, c)[0] == L.HANDLE_IS_NULLPTR
    assert size_of(lib, handle, None, b, c)[0] == L.HANDLE_IS_NULLPTR
    assert size_of(lib, handle, a, b, c, alpha=None)[0] == L.INVALID_VALUE
    assert size_of(lib, handle, a, b, c, beta=None)[0] == L.INVALID_VALUE
    assert size_of(lib, handle, a, b, c, op=7)[0] == L.NOT_SUPPORTED
    assert size_of(lib, handle, a, b, c, offsets=None)[0] == L.INVALID_VALUE          # three groups
    assert size_of(lib, handle, a, b, c, offsets=c_void_p(0x10002))[0] == L.INVALID_VALUE
    assert size_of(lib, handle, a, b, c, rs=c_void_p(0x10002))[0] == L.INVALID_VALUE
    assert size_of(lib, handle, a, b, c, cs=c_void_p(0x10001))[0] == L.INVALID_VALUE
    assert size_of(lib, handle, mat(10, 17), b, c)[0] == L.INVALID_VALUE
    assert size_of(lib, handle, mat(11, 16), b, c)[0] == L.INVALID_VALUE
    assert size_of(lib, handle, a, b, mat(10, 23))[0] == L.INVALID_VALUE
    assert size_of(lib, handle, a, b, c, op=L.OP_N)[0] == L.INVALID_VALUE
    assert size_of(lib, handle, mat(10, 16, order=L.ORDER_COL), b, c)[0] == L.NOT_SUPPORTED
    assert size_of(lib, handle, a, b, mat(10, 24, order=L.ORDER_COL))[0] == L.NOT_SUPPORTED
    assert size_of(lib, handle, mat(10, 16, batch=2), b, c)[0] == L.NOT_SUPPORTED
    assert size_of(lib, handle, mat(10, 16, values=c_void_p(0x10001)), b, c)[0] == L.INVALID_VALUE
    k = 131072  # the first length whose int8 sums can pass int32
    for length, want in ((k, L.NOT_SUPPORTED), (k - 1, L.SUCCESS)):
        got, _ = size_of(lib, handle, mat(2, length, dtype=L.ACL_INT8), mat(24, length, dtype=L.ACL_INT8),
                         mat(2, 24, dtype=L.ACL_FLOAT))
        assert got == want
    mirrors = (c_void_p * 1)(FAKE[3].value)
    assert lib.aclsparseB200DnMatSetMirrors(c, 1, mirrors) == L.SUCCESS
    assert size_of(lib, handle, a, b, c)[0] == L.NOT_SUPPORTED
    vec = c_void_p(None)
    assert lib.aclsparseCreateDnVec(byref(vec), 4, FAKE[0], L.ACL_BF16) == L.SUCCESS
    assert size_of(lib, handle, vec, b, mat(10, 24))[0] == L.INVALID_VALUE
    assert lib.aclsparseDestroyDnVec(vec) == L.SUCCESS


def test_forward_buffer_refusals(lib, handle, mat):
    a, b, c = mat(10, 16), mat(24, 16, batch=3), mat(10, 24)
    for fn in (lib.aclsparseB200GroupedMM, lib.aclsparseB200GroupedMMPreprocess):
        call = lambda buf: fn(handle, L.OP_T, ONE, a, FAKE[9], b, None, None, ONE, c, L.ACL_FLOAT, buf)  # noqa: E731
        assert call(None) == L.INSUFFICIENT_RESOURCES
        assert call(c_void_p(0x10020)) == L.INVALID_VALUE
    assert lib.aclsparseB200GroupedMMGetBufferSize(handle, L.OP_T, ONE, a, FAKE[9], b, None, None, ONE, c, L.ACL_FLOAT,
                                                   None) == L.INVALID_VALUE


def test_gradient_accepts_and_refuses(lib, handle, mat):
    a, b, c = mat(10, 16), mat(10, 24), mat(16, 24, batch=3)
    assert grad_size(lib, handle, a, b, c)[0] == L.SUCCESS
    assert grad_size(lib, handle, a, b, mat(16, 24, batch=3, order=L.ORDER_COL))[0] == L.SUCCESS
    assert grad_size(lib, handle, a, b, mat(16, 24, batch=3, dtype=L.ACL_FLOAT))[0] == L.SUCCESS
    assert grad_size(lib, handle, mat(0, 16, values=None), mat(0, 24, values=None), c)[0] == L.SUCCESS
    assert grad_size(lib, None, a, b, c)[0] == L.HANDLE_IS_NULLPTR
    assert grad_size(lib, handle, a, None, c)[0] == L.HANDLE_IS_NULLPTR
    assert grad_size(lib, handle, a, b, c, offsets=None)[0] == L.INVALID_VALUE
    assert grad_size(lib, handle, a, mat(11, 24), c)[0] == L.INVALID_VALUE
    assert grad_size(lib, handle, a, b, mat(24, 16, batch=3))[0] == L.INVALID_VALUE
    assert grad_size(lib, handle, a, mat(10, 24, order=L.ORDER_COL), c)[0] == L.NOT_SUPPORTED
    assert grad_size(lib, handle, a, b, c, compute=L.ACL_INT32)[0] == L.NOT_SUPPORTED
    int8 = dict(dtype=L.ACL_INT8)
    assert grad_size(lib, handle, mat(10, 16, **int8), mat(10, 24, **int8),
                     mat(16, 24, batch=3, dtype=L.ACL_FLOAT))[0] == L.NOT_SUPPORTED
    assert grad_size(lib, handle, a, mat(10, 24, dtype=L.ACL_FLOAT16), c)[0] == L.NOT_SUPPORTED
    for fn in (lib.aclsparseB200GroupedMMWeightGrad, lib.aclsparseB200GroupedMMWeightGradPreprocess):
        assert fn(handle, ONE, a, b, FAKE[9], ONE, c, L.ACL_FLOAT, None) == L.INSUFFICIENT_RESOURCES
        assert fn(handle, ONE, a, b, FAKE[9], ONE, c, L.ACL_FLOAT, c_void_p(0x10010)) == L.INVALID_VALUE


def test_wait_failure_counter_refusals(lib):
    count = ctypes.c_uint32(7)
    assert lib.aclsparseB200GroupedMMWaitFailures(FAKE[1], None, byref(count)) == L.INVALID_VALUE
    assert lib.aclsparseB200GroupedMMWaitFailures(FAKE[1], FAKE[0], None) == L.INVALID_VALUE


def test_quantize_refusals(lib, handle, mat):
    x, q = mat(4, 8), mat(4, 8, dtype=L.ACL_INT8)
    call = lib.aclsparseB200QuantizeRows
    assert call(None, x, q, FAKE[2]) == L.HANDLE_IS_NULLPTR
    assert call(handle, None, q, FAKE[2]) == L.HANDLE_IS_NULLPTR
    assert call(handle, x, q, None) == L.INVALID_VALUE
    assert call(handle, x, q, c_void_p(0x10002)) == L.INVALID_VALUE
    assert call(handle, x, mat(4, 9, dtype=L.ACL_INT8), FAKE[2]) == L.INVALID_VALUE
    assert call(handle, x, mat(4, 8), FAKE[2]) == L.NOT_SUPPORTED
    assert call(handle, mat(4, 8, dtype=L.ACL_INT8), q, FAKE[2]) == L.NOT_SUPPORTED
    assert call(handle, mat(4, 8, order=L.ORDER_COL), q, FAKE[2]) == L.NOT_SUPPORTED
    assert call(handle, mat(4, 8, batch=2), q, FAKE[2]) == L.NOT_SUPPORTED
    assert call(handle, mat(0, 8, values=None), mat(0, 8, values=None, dtype=L.ACL_INT8), None) == L.SUCCESS


def test_adapter_refusals():
    import torch

    from ops_sparse_b200 import torch_adapter as A
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 6, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        A.grouped_mm(x, w, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        A.int8_mm(x.to(torch.int8), w.to(torch.int8), torch.ones(4), torch.ones(2, 6))
    with pytest.raises(ValueError, match="CUDA"):
        A.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        A.grouped_mm(None, w)


def test_parameter_block_matches_its_mirror(tmp_path):
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [n for n, _ in L.GroupedParams._fields_]
    src = tmp_path / "block.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "aclsparse_b200_kernels.h"\nint main(void) {\n' +
                   "".join(f'printf("%zu ", offsetof(AclspGroupedParams, {n}));\n' for n in names) +
                   'printf("%zu\\n", sizeof(AclspGroupedParams)); return 0; }\n')
    exe = tmp_path / "block"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(L.GroupedParams, n).offset for n in names] + [ctypes.sizeof(L.GroupedParams)]
