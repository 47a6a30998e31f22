"""PyTorch adapter: ``torch.mv`` / ``torch.addmm`` semantics on CSR CUDA tensors, served by this library.

Counterpart of the reference's torch extension (sparse/spmv/torch_extension/csrc/spmv.cpp:255-330,
sparse/spmv/torch_extension/spmv.py:44-47 and the SpMM twin under sparse/spmm/torch_extension), which routes
``aten::mv`` for CSR tensors of its device to ``aclsparseSpMV`` and exposes two test entries that take the CSR
arrays directly.  Same entry names and argument meaning here:

    mv(mat, vec)                                          y = A @ vec        (alpha = 1, beta = 0)
    addmm(input, mat, dense, beta=1, alpha=1)             beta * input + alpha * A @ dense
    spmv_csr(row_ptr, col_ind, values, x, y, alpha, beta, base=0, trans="N", cols=None)   in place on y
    spmv_workspace(...)                                   bytes aclsparseSpMVGetBufferSize asks for

The products between the sparse steps of a mixture-of-experts layer have no counterpart in the reference:

    grouped_mm(x, weight, offsets)                        y[r] = x[r] @ weight[g].T for the rows r of group g, with gradients
    int8_mm(x, weight, x_scales, w_scales, offsets)       the same on int8 with one scale per row and per output column
    quantize_rows(x)                                      int8 rows and their scales
    wait_failures(device)                                 whether products have ended without their results: 0 if none

Argument errors are raised as ``ValueError`` / ``TypeError`` before anything is launched, in the order the reference
checks them; the product itself runs through the C API on the current CUDA stream.  Like the reference's adapter,
every call builds its descriptors and preprocesses (the plan build is tens of microseconds on the device and needs
no host round trip).  ``install()`` additionally registers ``mv`` as the ``aten::mv`` kernel of CSR CUDA tensors.
"""
from __future__ import annotations

import contextlib
import threading

import torch

from . import _lib as L

INT32_MAX = 2 ** 31 - 1
_OPS = {"N": L.OP_N, "T": L.OP_T, "H": L.OP_H}


def _check_matrix_and_operand(mat: torch.Tensor, other: torch.Tensor, other_name: str, other_dim: int) -> None:
    """The reference's CheckMvInputs (spmv.cpp:261-287), CUDA in place of its device type."""
    if not isinstance(mat, torch.Tensor):
        raise TypeError("mat must be a defined tensor")
    if mat.layout != torch.sparse_csr:
        raise ValueError(f"mat must use the sparse CSR layout, but got {mat.layout}")
    if mat.device.type != "cuda":
        raise ValueError(f"mat must be on a CUDA device, but got {mat.device}")
    if mat.dim() != 2:
        raise ValueError(f"mat must be a 2-D sparse matrix, but got {mat.dim()} dimensions")
    if not isinstance(other, torch.Tensor):
        raise TypeError(f"{other_name} must be a defined tensor")
    if other.layout != torch.strided:
        raise ValueError(f"{other_name} must be a dense tensor, but got layout {other.layout}")
    if other.device.type != "cuda":
        raise ValueError(f"{other_name} must be on a CUDA device, but got {other.device}")
    if other.dim() != other_dim:
        raise ValueError(f"{other_name} must be a {other_dim}-D dense tensor, but got {other.dim()} dimensions")
    if mat.device != other.device:
        raise ValueError(f"mat and {other_name} must be on the same device, but got {mat.device} and {other.device}")
    if mat.dtype != other.dtype:
        raise TypeError(f"mat and {other_name} must have the same dtype, but got {mat.dtype} and {other.dtype}")
    if mat.dtype != torch.float32:
        raise TypeError(f"this build computes in float32 only, but got {mat.dtype}")
    if mat.size(1) != other.size(0):
        raise ValueError(f"size mismatch: mat is {tuple(mat.shape)}, {other_name} has {other.size(0)} rows")
    if mat.size(0) > INT32_MAX or mat.size(1) > INT32_MAX or mat._nnz() > INT32_MAX:
        raise ValueError("rows, columns and non-zeros must fit int32")


def _csr_arrays(mat: torch.Tensor):
    """int32 row offsets / column indices (PyTorch keeps int64 by default) and contiguous values."""
    crow = mat.crow_indices()
    col = mat.col_indices()
    if crow.dtype != torch.int32:
        crow = crow.to(torch.int32)
    if col.dtype != torch.int32:
        col = col.to(torch.int32)
    return crow.contiguous(), col.contiguous(), mat.values().contiguous()


def _handle():
    from . import api
    return api.Handle()  # bound to the current torch stream


def mv(mat: torch.Tensor, vec: torch.Tensor) -> torch.Tensor:
    """``A @ vec`` for a CSR sparse matrix and a dense vector on the GPU (aten::mv semantics)."""
    _check_matrix_and_operand(mat, vec, "vec", 1)
    from . import api
    rows, cols = mat.shape
    crow, col, val = _csr_arrays(mat)
    y = torch.empty(rows, dtype=torch.float32, device=mat.device)
    if rows == 0:
        return y
    if mat._nnz() == 0 or cols == 0:
        return y.zero_()
    with torch.cuda.device(mat.device):
        a = api.CsrMatrix(rows, cols, crow, col, val, L.BASE_ZERO, nnz=int(val.numel()))
        op = api.SpMV(_handle(), a, api.DnVec(vec.contiguous()), api.DnVec(y))
        op.preprocess(1.0, 0.0)
        op(1.0, 0.0)
    return y


def addmm(input: torch.Tensor, mat: torch.Tensor, dense: torch.Tensor, *, beta: float = 1.0,
          alpha: float = 1.0) -> torch.Tensor:
    """``beta * input + alpha * (A @ dense)`` for a CSR ``A`` and row-major dense operands (aten::addmm semantics)."""
    _check_matrix_and_operand(mat, dense, "dense", 2)
    from . import api
    rows, cols = mat.shape
    n = dense.size(1)
    if not isinstance(input, torch.Tensor) or input.device != mat.device or input.dtype != torch.float32:
        raise TypeError("input must be a float32 tensor on the device of mat")
    c = input.expand(rows, n).contiguous().clone() if beta != 0.0 else torch.empty(rows, n, dtype=torch.float32,
                                                                                   device=mat.device)
    if rows == 0 or n == 0:
        return c
    if mat._nnz() == 0 or cols == 0:
        return c.mul_(beta) if beta != 0.0 else c.zero_()
    crow, col, val = _csr_arrays(mat)
    b = dense.contiguous()
    with torch.cuda.device(mat.device):
        a = api.CsrMatrix(rows, cols, crow, col, val, L.BASE_ZERO, nnz=int(val.numel()))
        op = api.SpMM(_handle(), a, api.DnMat(cols, n, n, b), api.DnMat(rows, n, n, c))
        op.preprocess(alpha, beta)
        op(alpha, beta)
    return c


def mm(mat: torch.Tensor, dense: torch.Tensor) -> torch.Tensor:
    """``A @ dense``."""
    _check_matrix_and_operand(mat, dense, "dense", 2)
    zero = torch.empty(0, dtype=torch.float32, device=mat.device)
    return addmm(zero, mat, dense, beta=0.0, alpha=1.0)


def _check_arrays(row_ptr, col_ind, values, x, y, base, trans, cols):
    """The reference's CheckSpmvNpuInputs (spmv.cpp:336-377)."""
    tensors = dict(row_ptr=row_ptr, col_ind=col_ind, values=values, x=x, y=y)
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
            raise ValueError(f"{name} must be a CUDA tensor")
    if len({t.device for t in tensors.values()}) != 1:
        raise ValueError("row_ptr, col_ind, values, x and y must be on the same device")
    if row_ptr.dtype != torch.int32 or col_ind.dtype != torch.int32:
        raise TypeError("row_ptr and col_ind must be int32")
    if col_ind.numel() != values.numel():
        raise ValueError(f"col_ind and values length mismatch: {col_ind.numel()} vs {values.numel()}")
    if x.dtype != values.dtype:
        raise TypeError(f"x and values must have the same dtype, but got {x.dtype} and {values.dtype}")
    if base not in (0, 1):
        raise ValueError(f"base must be 0 or 1, but got {base}")
    if trans not in _OPS:
        raise ValueError(f"trans must be N, T or H, but got {trans}")
    if x.dim() != 1 or y.dim() != 1:
        raise ValueError("x and y must be one-dimensional")
    if row_ptr.numel() < 1:
        raise ValueError("row_ptr must not be empty")
    rows = row_ptr.numel() - 1
    if max(rows, x.numel(), y.numel(), values.numel()) > INT32_MAX:
        raise ValueError("sizes must fit int32")
    if values.dtype != torch.float32 or y.dtype != torch.float32:
        raise TypeError("this build computes in float32 only")
    is_trans = trans != "N"
    cols = (y.numel() if is_trans else x.numel()) if cols is None else cols
    x_size, y_size = (rows, cols) if is_trans else (cols, rows)
    if x.size(0) < x_size:
        raise ValueError(f"x is too small for the requested op: need {x_size}, got {x.size(0)}")
    if y.size(0) < y_size:
        raise ValueError(f"y is too small for the requested op: need {y_size}, got {y.size(0)}")
    return rows, cols, x_size, y_size


def _spmv_op(row_ptr, col_ind, values, x, y, base, trans, cols, sizes):
    from . import api
    rows, cols, x_size, y_size = sizes
    a = api.CsrMatrix(rows, cols, row_ptr, col_ind if col_ind.numel() else None, values if values.numel() else None,
                      base, nnz=int(values.numel()))
    return api.SpMV(_handle(), a, api.DnVec(x, size=x_size), api.DnVec(y, size=y_size), op=_OPS[trans])


def spmv_csr(row_ptr, col_ind, values, x, y, alpha: float = 1.0, beta: float = 0.0, base: int = 0, trans: str = "N",
             cols: "int | None" = None) -> torch.Tensor:
    """``y = alpha * op(A) * x + beta * y`` from explicit CSR arrays, in place on ``y`` (the reference's ``spmv_npu``).

    op(A) = T / H is answered with the library's NOT_SUPPORTED status (an ``AclsparseError``) in this build.
    """
    sizes = _check_arrays(row_ptr, col_ind, values, x, y, base, trans, cols)
    with torch.cuda.device(y.device):
        op = _spmv_op(row_ptr, col_ind, values, x, y, base, trans, cols, sizes)
        op.preprocess(alpha, beta)
        op(alpha, beta)
    return y


def spmv_workspace(row_ptr, col_ind, values, x, y, alpha: float = 1.0, beta: float = 0.0, base: int = 0,
                   trans: str = "N", cols: "int | None" = None) -> int:
    """Bytes of external buffer ``aclsparseSpMVGetBufferSize`` asks for (the reference's ``spmv_npu_workspace``)."""
    sizes = _check_arrays(row_ptr, col_ind, values, x, y, base, trans, cols)
    with torch.cuda.device(y.device):
        return _spmv_op(row_ptr, col_ind, values, x, y, base, trans, cols, sizes).buffer_size(alpha, beta)


_local = threading.local()


@contextlib.contextmanager
def _stream_handle():
    """This thread's kept handle on the current stream.

    Destroying a handle waits for its stream, which a capture forbids and a training step should not pay for; between
    calls the kept one is on no stream, so that nothing waits for a stream that is gone.
    """
    from . import api
    handle = getattr(_local, "handle", None)
    if handle is None:
        handle = _local.handle = api.Handle(set_stream=False)
    handle.set_stream(torch.cuda.current_stream().cuda_stream)
    try:
        yield handle
    finally:
        L.lib().aclsparseSetStream(handle.raw, None)


def _dense_operand(name: str, t, dim: int, dtypes) -> None:
    if not isinstance(t, torch.Tensor) or t.layout != torch.strided or t.device.type != "cuda":
        raise ValueError(f"{name} must be a dense CUDA tensor")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, but has {t.dim()}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {[str(d) for d in dtypes]}, but is {t.dtype}")


def _check_grouped(x, weight, offsets, dtypes, names=("x", "weight")) -> None:
    _dense_operand(names[0], x, 2, dtypes)
    _dense_operand(names[1], weight, 3, dtypes)
    if weight.dtype != x.dtype:
        raise TypeError(f"{names[0]} and {names[1]} must have the same dtype, but got {x.dtype} and {weight.dtype}")
    if x.size(1) != weight.size(2):
        raise ValueError(f"size mismatch: {names[0]} is {tuple(x.shape)}, {names[1]} is {tuple(weight.shape)}")
    if weight.size(0) < 1 or weight.size(0) > 65535:
        raise ValueError(f"between 1 and 65535 groups are supported, but got {weight.size(0)}")
    _check_offsets(offsets, weight.size(0), x.device)
    if weight.device != x.device:
        raise ValueError(f"{names[0]} and {names[1]} must be on the same device")


def _check_offsets(offsets, groups: int, device) -> None:
    if offsets is None:
        if groups != 1:
            raise ValueError(f"offsets are needed with {groups} groups")
        return
    if not isinstance(offsets, torch.Tensor) or offsets.device != device or offsets.dtype != torch.int32:
        raise TypeError("offsets must be an int32 tensor on the device of the operands")
    if offsets.dim() != 1 or offsets.numel() != groups + 1:
        raise ValueError(f"offsets must hold {groups + 1} row numbers, but has shape {tuple(offsets.shape)}")


def _rows_descr(t: torch.Tensor):
    """Row-major descriptor of a 2-D tensor; a copy is made where a row is not contiguous or rows overlap, and of a view
    that stands for the negative of its memory."""
    from . import api
    t = t.resolve_neg()
    if t.size(1) > 1 and t.stride(1) != 1 or t.size(0) > 1 and t.stride(0) < t.size(1):
        t = t.contiguous()
    return api.DnMat(t.size(0), t.size(1), t.stride(0) if t.size(0) > 1 else t.size(1), t)


def _batch_descr(w: torch.Tensor):
    """Descriptor of a 3-D tensor, one matrix per group, rows or columns contiguous; else a copy is described."""
    from . import api
    w = w.resolve_neg()
    groups, rows, cols = w.shape

    def fits(outer, outer_stride, inner, inner_stride):
        return ((inner_stride == 1 or inner == 1) and (outer == 1 or outer_stride >= inner) and
                (groups == 1 or w.stride(0) >= (outer - 1) * outer_stride + inner))

    if rows and cols and fits(cols, w.stride(2), rows, w.stride(1)) and not fits(rows, w.stride(1), cols, w.stride(2)):
        order, ld = L.ORDER_COL, w.stride(2) if cols > 1 else rows
    else:
        if not fits(rows, w.stride(1), cols, w.stride(2)):
            w = w.contiguous()
        order, ld = L.ORDER_ROW, w.stride(1) if rows > 1 else cols
    return api.DnMat(rows, cols, ld, w, order, groups, w.stride(0) if groups > 1 else 0)


def _loadable(describe, t: torch.Tensor):
    """``describe(t)``, of a copy where its first element alone keeps its rows from multiples of 16 bytes.

    The tensor-core kernels load from such multiples.  Rows of odd widths are copied by the library, in the buffer, but
    that has no room for an operand that is merely shifted.  The strides that count are the descriptor's: a tensor's own
    say nothing where a dimension has one element (a row cut out of a matrix of odd width keeps that width as its stride).
    """
    d = describe(t)
    unit = d.values.element_size()
    even = d.ld * unit % 16 == 0 and d.batch_stride * unit % 16 == 0
    return describe(d.values.clone()) if even and d.values.data_ptr() % 16 else d


def _forward(x, weight, offsets, out_dtype, op_b, row_scales=None, col_scales=None):
    """x[r] @ op(weight[g]); rows in no group are zero."""
    from . import api
    n = weight.size(1) if op_b == L.OP_T else weight.size(2)
    with torch.cuda.device(x.device):
        # without offsets the one group is all rows
        y = (torch.empty if offsets is None else torch.zeros)(x.size(0), n, dtype=out_dtype, device=x.device)
        if y.numel():
            with _stream_handle() as handle:
                api.GroupedMM(handle, _loadable(_rows_descr, x), _loadable(_batch_descr, weight), _rows_descr(y),
                              None if offsets is None else offsets.contiguous(), op_b, row_scales, col_scales)()
    return y


class _GroupedMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, out_dtype):
        ctx.save_for_backward(x, weight, offsets)
        return _forward(x, weight, offsets, out_dtype, L.OP_T)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        from . import api
        x, weight, offsets = ctx.saved_tensors
        dy = dy.to(x.dtype)
        dx = _forward(dy, weight, offsets, x.dtype, L.OP_N) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            with torch.cuda.device(x.device):
                dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
                if dw.numel():
                    with _stream_handle() as handle:
                        api.GroupedMMWeightGrad(handle, _loadable(_rows_descr, dy), _loadable(_rows_descr, x), _batch_descr(dw),
                                                None if offsets is None else offsets.contiguous())()
        return dx, dw, None, None


def grouped_mm(x: torch.Tensor, weight: torch.Tensor, offsets: "torch.Tensor | None" = None, *,
               out_dtype: "torch.dtype | None" = None) -> torch.Tensor:
    """``x[r] @ weight[g].T`` for the rows ``offsets[g] <= r < offsets[g + 1]`` of every group g.

    x: rows x k, weight: groups x n x k, fp16 or bf16; offsets: groups + 1 ascending int32 values on the same device
    (None with one group).  The result has ``out_dtype``: that type (default) or float32; rows in no group are zero.
    Differentiable (once) in x and weight, from the result's gradient rounded to their type; offsets carry no gradient.
    """
    _check_grouped(x, weight, offsets, (torch.float16, torch.bfloat16))
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {x.dtype} or torch.float32, but got {out_dtype}")
    return _GroupedMM.apply(x, weight, offsets, out_dtype)


def int8_mm(x: torch.Tensor, weight: torch.Tensor, x_scales: torch.Tensor, w_scales: torch.Tensor,
            offsets: "torch.Tensor | None" = None, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x_scales[r] * w_scales[g] * (x[r] @ weight[g].T)`` on int8 operands, exact inside the sum; no gradients.

    x: rows x k and weight: groups x n x k (or n x k: one group), int8; x_scales: rows and w_scales: groups x n (or
    n) float32 values.  The result is bfloat16, float16 or float32; rows in no group are zero.
    """
    if isinstance(weight, torch.Tensor) and weight.dim() == 2:
        weight = weight.unsqueeze(0)
    _check_grouped(x, weight, offsets, (torch.int8,))
    if x.size(1) > 131071:
        raise ValueError("sums of more than 131071 int8 products do not fit int32")
    if out_dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"out_dtype must be a 16-bit floating type or torch.float32, but got {out_dtype}")
    for name, t, count in (("x_scales", x_scales, x.size(0)), ("w_scales", w_scales, weight.size(0) * weight.size(1))):
        if not isinstance(t, torch.Tensor) or t.device != x.device or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a float32 tensor on the device of the operands")
        if t.numel() != count:
            raise ValueError(f"{name} must have {count} elements, but has {t.numel()}")
    return _forward(x.detach(), weight.detach(), offsets, out_dtype, L.OP_T, x_scales.detach().contiguous(),
                    w_scales.detach().contiguous())


def quantize_rows(x: torch.Tensor) -> "tuple[torch.Tensor, torch.Tensor]":
    """int8 rows ``q`` and float32 ``scales`` with ``x[r]`` close to ``scales[r] * q[r]``: scales[r] = max|x[r]| / 127
    (as the fp32 product with the fp32 number nearest to 1 / 127).

    Rows are rounded to the nearest integer, ties to even; a row with an infinity or a NaN gets zeros and that scale.
    """
    _dense_operand("x", x, 2, (torch.float32, torch.float16, torch.bfloat16))
    from . import api
    with torch.cuda.device(x.device):
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        scales = torch.empty(x.size(0), dtype=torch.float32, device=x.device)
        with _stream_handle() as handle:
            api.QuantizeRows(handle, _rows_descr(x.detach()), _rows_descr(q), scales)()
    return q, scales


def wait_failures(device=None) -> int:
    """CTAs of ``grouped_mm`` and ``int8_mm``, gradients among them, that gave up a (four seconds' bounded) wait on
    ``device`` since the program began; waits for its current stream.

    0 in healthy programs.  A reading larger than the one before means that results between them are incomplete.
    """
    from . import api
    with torch.cuda.device(device):
        return api.grouped_wait_failures()


_installed = []


def install() -> None:
    """Registers ``mv`` as the ``aten::mv`` implementation for CSR CUDA tensors (replacing PyTorch's own)."""
    if _installed:
        return
    lib = torch.library.Library("aten", "IMPL")
    lib.impl("mv", mv, "SparseCsrCUDA")
    _installed.append(lib)  # the registration lives as long as the Library object


__all__ = ["mv", "mm", "addmm", "spmv_csr", "spmv_workspace", "grouped_mm", "int8_mm", "quantize_rows", "wait_failures",
           "install"]
