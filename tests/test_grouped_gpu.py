"""Grouped products, their gradients, the int8 product and the row quantisation against plain 64-bit torch.

Tolerance of a floating result, element by element: with S = scale * sum |a||b| in 64 bits, an fp32 sum of k products
in any order, with truncation allowed at every addition, is off by at most (k + 8) * 2^-23 * S (the scales' and beta's
few roundings are in the 8), and the rounding to the type of C by eps / 2 relative to the value, plus half the
smallest subnormal.  int8 sums are exact; up to five roundings of scales and conversion remain: 8 * 2^-24 relative.
"""
import ctypes

import pytest
import torch

from ops_sparse_b200 import _lib as L
from ops_sparse_b200 import api
from ops_sparse_b200 import torch_adapter as A

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def offsets_of(sizes, first=0):
    out = [first]
    for s in sizes:
        out.append(out[-1] + s)
    return out


def randn(*shape, dtype, gen):
    if dtype == torch.int8:
        return torch.randint(-128, 128, shape, generator=gen, device=DEV, dtype=torch.int8)
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def strided(rows, cols, ld, dtype, gen, shift=0):
    """rows x cols inside storage with leading dimension ld, starting `shift` elements in."""
    store = randn(rows * ld + shift + 1, dtype=dtype, gen=gen)
    return store[shift:shift + rows * ld].view(rows, ld)[:, :cols]


def close(got, want, bound):
    """|got - want| <= bound + the rounding to got's type; both infinite or both NaN elsewhere."""
    got64, t = got.double(), got.dtype
    fine = torch.isfinite(want) & (want.abs() + bound < torch.finfo(t).max)
    limit = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + TINY[t]
    bad = fine & ~((got64 - want).abs() <= limit)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float(((got64 - want).abs() - limit)[bad].max())}, first {bad.nonzero()[0].tolist()}")
    assert torch.equal(torch.isnan(got64[~fine]), torch.isnan(want[~fine]))


def sum_bound(k, s, int8):
    return 8 * 2.0 ** -24 * s if int8 else (k + 8) * 2.0 ** -23 * s


class Forward:
    """One product through the C ABI, its operands in chosen layouts, and the 64-bit answer."""

    def __init__(self, sizes, k, n, dtype, out=None, order=L.ORDER_ROW, op=L.OP_T, first=0, behind=0, pad=(0, 0, 0),
                 shift=(0, 0, 0), scales=False, seed=0, batch_pad=0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.int8 = dtype == torch.int8
        out = (torch.float32 if self.int8 else dtype) if out is None else out
        self.bounds = offsets_of(sizes, first)
        rows, groups = self.bounds[-1] + behind, len(sizes)
        self.k, self.n = k, n
        self.a = strided(rows, k, k + pad[0], dtype, gen, shift[0])
        k_inner = (order == L.ORDER_ROW) == (op != L.OP_N)          # the summed index is the contiguous one
        outer, inner = (n, k) if k_inner else (k, n)
        ld = inner + pad[1]
        stride = outer * ld + batch_pad
        store = randn(groups * stride + shift[1] + 1, dtype=dtype, gen=gen)[shift[1]:]
        every = torch.as_strided(store, (groups, outer, inner), (stride, ld, 1))
        self.w = every if k_inner else every.transpose(1, 2)        # groups x n x k
        self.c = strided(rows, n, n + pad[2], out, gen, shift[2])
        self.c0 = self.c.clone()
        self.offsets = torch.tensor(self.bounds, dtype=torch.int32, device=DEV)
        self.row_scales = torch.rand(rows, generator=gen, device=DEV) + 0.5 if scales else None
        self.col_scales = torch.rand(groups, n, generator=gen, device=DEV) + 0.5 if scales else None
        b_shape = (n, k) if op != L.OP_N else (k, n)
        self.op = api.GroupedMM(api.Handle(), api.DnMat(rows, k, k + pad[0], self.a),
                                api.DnMat(*b_shape, ld, store, order, groups, stride),
                                api.DnMat(rows, n, n + pad[2], self.c), self.offsets, op, self.row_scales, self.col_scales)

    def expected(self, alpha=1.0, beta=0.0, bounds=None):
        want, size = self.c0.double(), torch.zeros_like(self.c0, dtype=torch.float64)
        bounds = self.bounds if bounds is None else bounds
        for g in range(len(bounds) - 1):
            rows = slice(bounds[g], bounds[g + 1])
            a, w = self.a[rows].double(), self.w[g].double()
            scale = torch.full((a.shape[0], self.n), alpha, dtype=torch.float64, device=DEV)
            if self.row_scales is not None:
                scale = scale * self.row_scales[rows].double()[:, None] * self.col_scales[g].double()
            old = beta * self.c0[rows].double() if beta else torch.zeros_like(scale)
            want[rows] = scale * (a @ w.T) + old
            size[rows] = scale.abs() * (a.abs() @ w.abs().T) + old.abs()
        return want, size

    def check(self, alpha=1.0, beta=0.0):
        self.op(alpha, beta)
        torch.cuda.synchronize()
        want, size = self.expected(alpha, beta)
        close(self.c, want, sum_bound(self.k, size, self.int8))
        first, last = self.bounds[0], self.bounds[-1]
        assert torch.equal(self.c[:first], self.c0[:first]) and torch.equal(self.c[last:], self.c0[last:])


LAYOUTS = [(L.ORDER_ROW, L.OP_T), (L.ORDER_ROW, L.OP_N), (L.ORDER_COL, L.OP_T), (L.ORDER_COL, L.OP_N), (L.ORDER_ROW, L.OP_H)]
TYPES = [torch.bfloat16, torch.float16, torch.int8]
RAGGED = [0, 1, 17, 0, 64, 129, 3, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order,op", LAYOUTS)
@pytest.mark.parametrize("k,n", [(64, 128), (200, 136), (8, 16), (1, 1), (77, 301), (1024, 40)])
def test_forward_layouts(dtype, order, op, k, n):
    Forward(RAGGED, k, n, dtype, order=order, op=op).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [2], [15], [16], [33], [255], [256], [257], [700], [0], [0, 0, 5], [1] * 70,
                                   [300, 0, 513, 31, 32]])
def test_forward_group_sizes(dtype, sizes):
    Forward(sizes, 192, 272, dtype, seed=len(sizes)).check()


@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                       (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                       (torch.int8, torch.float32), (torch.int8, torch.float16),
                                       (torch.int8, torch.bfloat16)])
@pytest.mark.parametrize("alpha,beta,scales", [(1.0, 1.0, False), (-0.5, 0.25, True), (0.01, 0.0, True), (0.0, 2.0, False)])
def test_forward_scalars_and_scales(dtype, out, alpha, beta, scales):
    case = Forward([40, 0, 9, 300], 160, 144, dtype, out, first=3, behind=5, scales=scales)
    if dtype == torch.int8:
        alpha *= 2.0 ** -12  # fp16 holds the results
    case.check(alpha, beta)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", [L.ORDER_ROW, L.ORDER_COL])
@pytest.mark.parametrize("pad,shift", [((8, 16, 24), (0, 0, 0)), ((16, 16, 1), (0, 0, 1)), ((1, 3, 5), (0, 0, 0)),
                                       ((16, 16, 16), (1, 0, 0)), ((16, 16, 16), (0, 1, 0)), ((16, 16, 2), (16, 16, 2))])
def test_forward_strides_and_alignment(dtype, order, pad, shift):
    Forward([40, 0, 9, 150], 96, 160, dtype, order=order, pad=pad, shift=shift, batch_pad=16).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,k,n", [([700, 1, 0, 1500, 333, 256, 900, 40], 320, 2304), ([130] * 9, 1040, 4096),
                                       ([6000], 208, 1536)])
def test_forward_many_waves_of_tiles(dtype, sizes, k, n):
    """More tiles than CTAs, several times over: every stage of the ring and both halves of the sums are reused."""
    Forward(sizes, k, n, dtype, seed=n, first=1, behind=2).check()


FEW = [[1], [2], [3], [4], [5], [8], [1, 0, 2, 4, 1], [0, 3, 0, 5, 0], [0] * 40 + [2] + [0] * 30 + [5, 1], [2] * 8, [9, 0, 0, 0, 3]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", FEW)
@pytest.mark.parametrize("k,n", [(64, 128), (1040, 97), (16, 1), (2064, 1030)])
def test_forward_few_rows(dtype, sizes, k, n):
    Forward(sizes, k, n, dtype, first=1, behind=1, scales=True, seed=k).check(0.5)


@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                       (torch.int8, torch.float32), (torch.int8, torch.float16), (torch.int8, torch.bfloat16)])
@pytest.mark.parametrize("alpha,beta,scales", [(1.0, 1.0, False), (-0.5, 0.25, True), (0.0, 2.0, False)])
def test_forward_few_rows_scalars(dtype, out, alpha, beta, scales):
    case = Forward([3, 0, 1], 160, 145, dtype, out, scales=scales, pad=(16, 16, 3))
    case.check(alpha * 2.0 ** -12 if dtype == torch.int8 else alpha, beta)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 7, 17, 77, 1033])
@pytest.mark.parametrize("shift", [(0, 0, 0), (1, 0, 0), (0, 1, 1)])
def test_forward_few_rows_of_odd_widths(dtype, k, shift):
    """Rows on multiples of 16 bytes that end between them, with NaN behind; and the same from shifted bases."""
    case = Forward([2, 0, 5], k, 40, dtype, pad=(-k % 16, -k % 16, 0), shift=shift, seed=k)
    for t in (case.a, case.w):
        full = t.as_strided((*t.shape[:-1], t.stride(-2)), t.stride(), t.storage_offset())
        full[..., k:] = 127 if dtype == torch.int8 else float("nan")
    case.check()


def test_forward_few_rows_bad_offsets_and_special_values():
    case = Forward([2, 2, 2], 64, 48, torch.bfloat16)
    case.a[4] = float("inf")
    case.w[1] = float("nan")
    case.offsets.copy_(torch.tensor([-5, 4, 2, 2 ** 31 - 1], dtype=torch.int32))
    case.op()
    torch.cuda.synchronize()
    want, size = case.expected(bounds=[0, 4, 4, 6])
    rows = [0, 1, 2, 3, 5]
    close(case.c[rows], want[rows], sum_bound(case.k, size[rows], False))
    assert not torch.isfinite(case.c[4]).any()


def test_forward_rows_outside_the_groups_stay():
    Forward([5, 0, 70], 64, 64, torch.bfloat16, first=7, behind=300).check()


def test_forward_no_summed_index():
    """k = 0: beta * C in the groups' rows."""
    c = torch.randn(6, 16, device=DEV)
    want = torch.cat([c[:1], 0.5 * c[1:4], c[4:]])
    offsets = torch.tensor([1, 1, 4], dtype=torch.int32, device=DEV)
    op = api.GroupedMM(api.Handle(), api.DnMat(6, 0, 0, torch.empty(0, dtype=torch.bfloat16, device=DEV)),
                       api.DnMat(16, 0, 0, torch.empty(0, dtype=torch.bfloat16, device=DEV), L.ORDER_ROW, 2, 0),
                       api.DnMat(6, 16, 16, c), offsets, L.OP_T)
    op(1.0, 0.5)
    assert torch.equal(c, want)


def test_forward_beta_zero_does_not_read_c():
    case = Forward([9, 30], 64, 48, torch.bfloat16)
    case.c.fill_(float("nan"))
    case.check()


@pytest.mark.parametrize("bounds", [[0, 50, 20, 80], [-7, 10, 10 ** 9, 90], [90, 60, 30, 0], [2 ** 31 - 1, -2 ** 31, 5, 6]])
def test_forward_bad_offsets_stay_inside(bounds):
    """Offsets that do not ascend or leave the matrix are clamped; rows in no group stay, the guard rows too."""
    case = Forward([30, 30, 30], 64, 48, torch.bfloat16)
    case.offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
    case.op()
    torch.cuda.synchronize()
    top, clean = 0, []
    for b in [min(max(v, 0), 90) for v in bounds]:
        top = max(top, b)
        clean.append(top)
    want, size = case.expected(bounds=clean)
    close(case.c, want, sum_bound(case.k, size, False))


@pytest.mark.parametrize("groups", [40, 256, 257, 600])
def test_forward_bad_offsets_of_many_groups(groups):
    """Both walks over the groups, the one that counts the tiles and the one that finds them, clamp alike."""
    case = Forward([3] * groups, 40, 264, torch.bfloat16, seed=groups)
    rows = 3 * groups
    steps = torch.randint(-40, 61, (groups + 1,), generator=torch.Generator().manual_seed(groups))
    bounds = (torch.arange(groups + 1) * rows // groups + steps).tolist()
    case.offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
    case.op()
    torch.cuda.synchronize()
    top, clean = 0, []
    for b in [min(max(v, 0), rows) for v in bounds]:
        top = max(top, b)
        clean.append(top)
    want, size = case.expected(bounds=clean)
    close(case.c, want, sum_bound(case.k, size, False))


def test_forward_special_values_stay_in_their_rows():
    """Infinities and NaN in one group's rows, and in the rows behind it, do not reach another row."""
    case = Forward([20, 20, 20], 96, 64, torch.bfloat16)
    clean, _ = case.expected()
    case.a[25] = float("inf")
    case.a[40, 3] = float("nan")
    case.op()
    torch.cuda.synchronize()
    rows = [r for r in range(60) if r not in (25, 40)]
    want, size = case.expected()
    close(case.c[rows], want[rows], sum_bound(case.k, size[rows], False))
    assert torch.equal(want[rows], clean[rows])
    assert not torch.isfinite(case.c[25]).any() and torch.isnan(case.c[40]).all()


def test_forward_is_repeatable_and_its_buffer_is_reusable():
    """The same bits every time, whatever the buffer held and whether or not Preprocess ran."""
    case = Forward([1, 3, 0, 2], 4096, 256, torch.bfloat16)
    case.op.allocate().fill_(0xAB)
    case.op()
    first = case.c.clone()
    case.op.preprocess()
    for _ in range(3):
        case.c.zero_()
        case.op()
        assert torch.equal(case.c, first)
    case.op.buffer.fill_(0xCD)
    case.op.preprocess()
    case.op()
    assert torch.equal(case.c, first)
    case.check()


def test_wait_failures_are_counted_and_cleared():
    """No wait runs out in a healthy product; a count left in the buffer is reported once and cleared."""
    case = Forward([1, 3], 2048, 256, torch.bfloat16)
    case.op.preprocess()
    case.op()
    assert case.op.wait_failures() == 0
    case.op.buffer[:4].view(torch.int32).fill_(3)
    assert case.op.wait_failures() == 3 and case.op.wait_failures() == 0
    case.check()


def test_two_products_share_a_buffer_in_turn():
    one, two = Forward([1, 2], 2048, 128, torch.bfloat16), Forward([5], 4096, 256, torch.float16, seed=3)
    size = max(one.op.buffer_size(), two.op.buffer_size())
    one.op.buffer = two.op.buffer = torch.empty(size, dtype=torch.uint8, device=DEV)
    one.op.preprocess()
    two.op.preprocess()
    for _ in range(2):
        one.check()
        two.check()


def test_forward_device_scalars():
    case = Forward([40, 9], 64, 48, torch.float16)
    case.op.handle.set_pointer_mode(L.POINTER_MODE_DEVICE)
    alpha, beta = torch.tensor([0.5], device=DEV), torch.tensor([-2.0], device=DEV)
    case.op(alpha, beta)
    torch.cuda.synchronize()
    want, size = case.expected(0.5, -2.0)
    close(case.c, want, sum_bound(case.k, size, False))


def test_forward_few_rows_device_scalars_and_replayed_with_other_offsets():
    case = Forward([1, 2, 0, 4], 512, 320, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    case.op.handle = api.Handle(side)
    case.op.handle.set_pointer_mode(L.POINTER_MODE_DEVICE)
    alpha, beta = torch.tensor([0.5], device=DEV), torch.tensor([0.0], device=DEV)
    case.op.allocate()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        case.op(alpha, beta)
    for bounds, scale in (([0, 1, 3, 3, 7], 0.5), ([0, 7, 7, 7, 7], -1.0), ([0, 0, 0, 5, 7], 2.0)):
        case.offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
        alpha.fill_(scale)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, size = case.expected(scale, bounds=bounds)
        close(case.c, want, sum_bound(case.k, size, False))


@pytest.mark.parametrize("rows", [2, 40])
def test_each_product_sees_the_rows_quantised_just_before_it(rows):
    """Kernels that start while the one before them ends, back to back, over the same few buffers."""
    gen = torch.Generator(device=DEV).manual_seed(15)
    x = torch.randn(30, rows, 1024, generator=gen, device=DEV).bfloat16()
    w, w_scales = A.quantize_rows(torch.randn(512, 1024, generator=gen, device=DEV).bfloat16())
    q, scales = torch.empty(rows, 1024, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    y = torch.empty(30, rows, 512, device=DEV)
    handle, buffer = api.Handle(), None
    steps = []
    for i in range(30):
        product = api.GroupedMM(handle, api.DnMat(rows, 1024, 1024, q), api.DnMat(512, 1024, 1024, w),
                                api.DnMat(rows, 512, 512, y[i]), None, L.OP_T, scales, w_scales)
        product.buffer = buffer = product.allocate() if buffer is None else buffer
        steps.append((api.QuantizeRows(handle, api.DnMat(rows, 1024, 1024, x[i]), api.DnMat(rows, 1024, 1024, q), scales),
                      product))
    torch.cuda.synchronize()
    for quantise, product in steps:
        quantise()
        product()
    torch.cuda.synchronize()
    for i in range(30):
        qi, si = A.quantize_rows(x[i])
        assert torch.equal(y[i], A.int8_mm(qi, w, si, w_scales, out_dtype=torch.float32))


def test_forward_on_another_stream_and_in_a_graph():
    case = Forward([3, 0, 40, 1], 512, 320, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        case.op.handle = api.Handle(side)
        case.op.preprocess()
        case.op()
    side.synchronize()
    want, size = case.expected()
    close(case.c, want, sum_bound(case.k, size, False))
    first = case.c.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        case.op()
    case.op.buffer.fill_(0xEE)      # a replay depends on nothing that the buffer held
    for _ in range(2):
        case.c.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(case.c, first)
    # other rows for the same graph: offsets are read on the device
    case.offsets.copy_(torch.tensor([0, 20, 21, 21, 44], dtype=torch.int32))
    case.bounds = [0, 20, 21, 21, 44]
    graph.replay()
    torch.cuda.synchronize()
    want, size = case.expected()
    close(case.c, want, sum_bound(case.k, size, False))


def test_int8_extremes_are_exact():
    """The longest allowed sum of the largest products: 131071 * 128 * 128 = 2^31 - 2^14."""
    k = 131071
    a = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    a[1] = 127
    w = torch.full((1, 5, k), -128, dtype=torch.int8, device=DEV)
    w[0, 2] = 127
    y = A.int8_mm(a, w, torch.ones(3, device=DEV), torch.ones(1, 5, device=DEV), out_dtype=torch.float32)
    want = (a.double() @ w[0].double().T)
    assert torch.equal(y, want.float())


class Gradient:
    def __init__(self, sizes, m, n, dtype, out=None, order=L.ORDER_ROW, first=0, behind=0, pad=(0, 0, 0), shift=(0, 0, 0),
                 seed=0, batch_pad=0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        out = dtype if out is None else out
        self.bounds = offsets_of(sizes, first)
        rows, groups = self.bounds[-1] + behind, len(sizes)
        self.a = strided(rows, m, m + pad[0], dtype, gen, shift[0])
        self.b = strided(rows, n, n + pad[1], dtype, gen, shift[1])
        outer, inner = (m, n) if order == L.ORDER_ROW else (n, m)
        ld = inner + pad[2]
        stride = outer * ld + batch_pad
        self.store = randn(groups * stride + shift[2], dtype=out, gen=gen)
        self.store0 = self.store.clone()
        view = lambda s: torch.as_strided(s, (groups, outer, inner), (stride, ld, 1), shift[2])  # noqa: E731
        flip = (lambda t: t) if order == L.ORDER_ROW else (lambda t: t.transpose(1, 2))
        self.c, self.c0 = flip(view(self.store)), flip(view(self.store0))
        self.view = view
        self.offsets = torch.tensor(self.bounds, dtype=torch.int32, device=DEV)
        self.op = api.GroupedMMWeightGrad(
            api.Handle(), api.DnMat(rows, m, m + pad[0], self.a), api.DnMat(rows, n, n + pad[1], self.b),
            api.DnMat(m, n, ld, self.store[shift[2]:], order, groups, stride), self.offsets)

    def expected(self, alpha=1.0, beta=0.0):
        want, size, most = [], [], max(self.bounds[g + 1] - self.bounds[g] for g in range(len(self.bounds) - 1))
        for g in range(len(self.bounds) - 1):
            rows = slice(self.bounds[g], self.bounds[g + 1])
            a, b, old = self.a[rows].double(), self.b[rows].double(), beta * self.c0[g].double() if beta else 0.0
            want.append(alpha * (a.T @ b) + old)
            size.append(abs(alpha) * (a.abs().T @ b.abs()) + abs(old))
        return torch.stack(want), torch.stack(size), most

    def check(self, alpha=1.0, beta=0.0):
        self.op(alpha, beta)
        torch.cuda.synchronize()
        want, size, most = self.expected(alpha, beta)
        close(self.c, want, sum_bound(most, size, False))
        # what lies between the rows and the matrices stays
        keep, keep0 = self.store.clone(), self.store0.clone()
        self.view(keep).zero_()
        self.view(keep0).zero_()
        assert torch.equal(keep, keep0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", [L.ORDER_ROW, L.ORDER_COL])
@pytest.mark.parametrize("m,n", [(128, 256), (8, 8), (1, 1), (136, 264), (77, 301), (512, 40)])
def test_gradient_shapes(dtype, order, m, n):
    Gradient(RAGGED, m, n, dtype, order=order).check()


@pytest.mark.parametrize("sizes", [[1], [15], [16], [17], [63], [64], [65], [0], [0, 0], [700], [1] * 40, [300, 0, 513, 31, 32]])
def test_gradient_group_sizes(sizes):
    Gradient(sizes, 144, 272, torch.bfloat16, first=2, behind=3, seed=len(sizes)).check()


@pytest.mark.parametrize("sizes", [[150, 0, 1, 700, 64, 65, 31, 2, 0, 400, 17, 300], [3] * 12, [1000] + [0] * 11])
def test_gradient_many_tiles(sizes):
    """Several tiles per CTA, most of them with rows to cut off, in every stage of the ring."""
    Gradient(sizes, 1280, 1288, torch.bfloat16, first=5, behind=9, seed=sizes[0]).check()


@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                       (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (-0.5, 0.25), (0.0, 2.0)])
def test_gradient_scalars(dtype, out, alpha, beta):
    Gradient([40, 0, 9, 100], 72, 80, dtype, out).check(alpha, beta)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pad,shift", [((8, 16, 24), (0, 0, 0)), ((8, 8, 1), (0, 0, 1)), ((1, 3, 5), (0, 0, 0)),
                                       ((8, 8, 8), (1, 0, 0)), ((8, 8, 8), (0, 1, 0))])
def test_gradient_strides_and_alignment(dtype, pad, shift):
    Gradient([40, 0, 9, 150], 96, 160, dtype, pad=pad, shift=shift, batch_pad=16).check()


def test_gradient_special_values_stay_in_their_group():
    """The rows next to a group's ends hold NaN and infinities: they are not in its sum."""
    case = Gradient([20, 5, 21], 64, 64, torch.bfloat16)
    case.a[20:25] = float("nan")
    case.b[20:25] = float("inf")
    case.op()
    torch.cuda.synchronize()
    want, size, most = case.expected()
    for g in (0, 2):
        close(case.c[g], want[g], sum_bound(most, size[g], False))
    assert torch.isnan(case.c[1]).all()


def test_gradient_bad_offsets_stay_inside():
    case = Gradient([30, 30, 30], 64, 48, torch.bfloat16)
    case.offsets.copy_(torch.tensor([-5, 40, 20, 2 ** 31 - 1], dtype=torch.int32))
    case.op()
    torch.cuda.synchronize()
    a, b = case.a.double(), case.b.double()
    close(case.c[0], a[:40].T @ b[:40], sum_bound(90, a[:40].abs().T @ b[:40].abs(), False))
    assert (case.c[1] == 0).all()


def test_gradient_is_repeatable_and_captures():
    case = Gradient([500, 0, 1200, 3], 96, 64, torch.bfloat16)
    case.op.allocate().fill_(0xAB)
    case.op()
    first = case.c.clone()
    case.op.preprocess()
    for _ in range(3):
        case.op()
        assert torch.equal(case.c, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    case.op.handle = api.Handle(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        case.op()
    case.op.buffer.fill_(0x55)
    case.store.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(case.c, first)


# ---- rows in 8 bits ----

def quantized(x):
    # the product of two fp32 numbers is exact in 64 bits: rounded once
    scale = (x.double().abs().amax(dim=1) * torch.tensor(1 / 127, dtype=torch.float32).double()).float()
    ratio = x.double() / torch.where(scale == 0, torch.ones_like(scale), scale).double()[:, None]
    return torch.where(scale[:, None] == 0, 0.0, torch.round(ratio)).clamp(-127, 127).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,pad,shift", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 64, 8, 8), (64, 1000, 0, 0), (2, 4096, 0, 0),
                                                 (33, 257, 3, 1), (3, 16384, 0, 0), (2, 40000, 0, 0), (300, 48, 16, 0),
                                                 (4, 8192, 0, 1)])
def test_quantize_rows(dtype, rows, cols, pad, shift):
    gen = torch.Generator(device=DEV).manual_seed(cols)
    x = strided(rows, cols, cols + pad, dtype, gen, shift)
    x.mul_(torch.exp(3 * torch.randn(rows, 1, generator=gen, device=DEV)).to(dtype).clamp(max=100))
    store = torch.full((rows * (cols + pad) + shift,), 99, dtype=torch.int8, device=DEV)
    q = store[shift:].view(rows, cols + pad)[:, :cols]
    scales = torch.empty(rows, device=DEV)
    api.QuantizeRows(api.Handle(), api.DnMat(rows, cols, cols + pad, x), api.DnMat(rows, cols, cols + pad, q), scales)()
    want, want_scales = quantized(x)
    assert torch.equal(scales, want_scales)
    assert torch.equal(q, want)
    if pad:
        assert (store[shift:].view(rows, cols + pad)[:, cols:] == 99).all()


def test_quantize_ties_and_near_ties():
    """Quotients on a tie, and so close to one that their fp32 value is the tie itself."""
    scale = torch.tensor([1.0, 1.0 + 2.0 ** -23, 3.0, 0.7, 1.9999999, 1e-30, 2.0 ** -140], device=DEV)
    halves = torch.arange(-126, 127, device=DEV).double() + 0.5
    rows = []
    for s in scale.double():
        near = (halves * s).float()
        up, down = torch.nextafter(near, near.new_tensor(3e38)), torch.nextafter(near, near.new_tensor(-3e38))
        # the row's largest value: one whose scale is s, where there is one
        tops = (127 * s).float().view(torch.int32) + torch.arange(-2, 3, device=DEV, dtype=torch.int32)
        tops = tops.view(torch.float32)
        fits = tops * torch.tensor(1 / 127, device=DEV, dtype=torch.float32) == s.float()
        rows.append(torch.cat([tops[fits][:1] if fits.any() else tops[2:3], near, up, down]))
    x = torch.stack(rows)
    assert (x.abs().amax(dim=1) == x[:, 0]).all()
    q, scales = A.quantize_rows(x)
    want, want_scales = quantized(x)
    ratio = x.double() / want_scales.double()[:, None]
    assert int(((2 * ratio) % 2 == 1).sum()) > 250  # ties, exactly
    assert torch.equal(scales, want_scales) and torch.equal(q, want)


def test_quantize_special_rows():
    x = torch.randn(6, 300, device=DEV)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 299] = float("nan")
    x[3, 0] = float("-inf")
    x[4] = 2.0 ** -149 * 60          # the scale rounds to zero
    x[5] = 3.4028234e38
    q, scales = A.quantize_rows(x)
    assert (q[1:5] == 0).all() and scales[1] == 0 and scales[4] == 0
    assert torch.isinf(scales[2]) and torch.isnan(scales[3])
    assert (q[5] == 127).all()
    y = A.int8_mm(q, torch.ones(1, 8, 300, dtype=torch.int8, device=DEV), scales, torch.ones(8, device=DEV),
                  out_dtype=torch.float32)
    assert torch.isnan(y[2:4]).all() and torch.isfinite(y[[0, 1, 4]]).all()
    empty_q, empty_s = A.quantize_rows(torch.empty(0, 5, device=DEV))
    assert empty_q.shape == (0, 5) and empty_s.shape == (0,)
    no_cols, zero = A.quantize_rows(torch.empty(3, 0, device=DEV))
    assert no_cols.shape == (3, 0) and (zero == 0).all()


# ---- the adapter, and a layer as it is used ----

def plain_grouped(x, w, bounds):
    parts = [x[bounds[g]:bounds[g + 1]] @ w[g].T for g in range(w.shape[0])]
    return torch.cat([x.new_zeros(bounds[0], w.shape[1])] + parts + [x.new_zeros(x.shape[0] - bounds[-1], w.shape[1])])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["plain", "transposed", "expanded", "sliced"])
def test_grouped_mm_gradients_match_the_formula(dtype, layout):
    gen = torch.Generator(device=DEV).manual_seed(5)
    bounds, k, n = [2, 30, 30, 95], 80, 56
    rows, groups = 100, 3
    x = randn(rows, 2 * k, dtype=dtype, gen=gen)[:, :k] if layout == "sliced" else randn(rows, k, dtype=dtype, gen=gen)
    w = {"plain": lambda: randn(groups, n, k, dtype=dtype, gen=gen),
         "sliced": lambda: randn(groups, n + 3, k + 8, dtype=dtype, gen=gen)[:, :n, :k],
         "transposed": lambda: randn(groups, k, n, dtype=dtype, gen=gen).transpose(1, 2),
         "expanded": lambda: randn(1, n, k, dtype=dtype, gen=gen).expand(groups, n, k)}[layout]()
    dy = randn(rows, n, dtype=dtype, gen=gen)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = A.grouped_mm(x, w, offsets)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    y64 = plain_grouped(x64, w64, bounds)
    gx64, gw64 = torch.autograd.grad(y64, (x64, w64), dy.double())
    close(y.detach(), y64.detach(), sum_bound(k, plain_grouped(x.detach().double().abs(), w.detach().double().abs(), bounds), False))
    inside = [slice(bounds[g], bounds[g + 1]) for g in range(groups)]
    size = torch.zeros(rows, k, dtype=torch.float64, device=DEV)
    for g, s in enumerate(inside):
        size[s] = dy[s].double().abs() @ w[g].detach().double().abs()
    close(gx, gx64, sum_bound(n, size, False))
    size = torch.stack([dy[s].double().abs().T @ x[s].detach().double().abs() for s in inside])
    close(gw, gw64, sum_bound(65, size, False))
    assert (y[:2] == 0).all() and (y[95:] == 0).all() and (gx[:2] == 0).all() and (gx[95:] == 0).all()


def test_grouped_mm_gradients_match_differences():
    """Directional differences of a 64-bit loss over the kernel's own fp32 results.

    The product is bilinear, so the central difference has no truncation error in x or w alone; what remains is the
    sums' error (bound as above, on both sides of the difference) and the rounding of the gradients to bf16.
    """
    gen = torch.Generator(device=DEV).manual_seed(6)
    bounds, k, n = [0, 20, 20, 33], 64, 48
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    x, w = randn(33, k, dtype=torch.bfloat16, gen=gen), randn(3, n, k, dtype=torch.bfloat16, gen=gen)
    # steps of one, on the values' own grid: x + d and x - d are exact in bf16 for whole numbers of this size
    x, w = (x * 4).round(), (w * 4).round()
    c = randn(33, n, dtype=torch.bfloat16, gen=gen)
    dx, dw = (torch.randint(-2, 3, t.shape, generator=gen, device=DEV).to(torch.bfloat16) for t in (x, w))
    loss = lambda x, w: (A.grouped_mm(x, w, offsets, out_dtype=torch.float32).double() * c.double()).sum()  # noqa: E731
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(A.grouped_mm(xg, wg, offsets, out_dtype=torch.float32), (xg, wg), c.float())
    whole = 64 * 64 * k * 2.0 ** -23 * 33 * n * 8   # |x|, |w| < 64 and |c| < 8: the sums' error, generously
    for step, diff, grad in ((dx, loss(x + dx, w) - loss(x - dx, w), gx), (dw, loss(x, w + dw) - loss(x, w - dw), gw)):
        along = (grad.double() * step.double()).sum()
        rounding = (grad.double().abs() * step.double().abs()).sum() * 2.0 ** -8
        assert abs(float(diff / 2 - along)) <= float(rounding) + whole


def route(tokens, experts, top, gen):
    """Top-k routing in the library's own formats: a stable sort of the expert numbers and the experts' offsets."""
    scores = torch.randn(tokens, experts, generator=gen, device=DEV)
    gates, chosen = scores.softmax(1).topk(top, dim=1)
    ids = chosen.reshape(-1).to(torch.int32)
    h, lib = api.Handle(), L.lib()
    order = torch.arange(ids.numel(), dtype=torch.int32, device=DEV)
    one_row = torch.tensor([0, ids.numel()], dtype=torch.int32, device=DEV)
    sorted_ids = ids.clone()
    descr = ctypes.c_void_p(None)
    assert lib.aclsparseCreateMatDescr(ctypes.byref(descr)) == L.SUCCESS
    size = ctypes.c_size_t(0)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    assert lib.aclsparseXcsrsort_bufferSizeExt(h.raw, 1, experts, ids.numel(), p(one_row), p(sorted_ids),
                                               ctypes.byref(size)) == L.SUCCESS
    work = torch.empty(max(int(size.value), 64), dtype=torch.uint8, device=DEV)
    assert lib.aclsparseXcsrsort(h.raw, 1, experts, ids.numel(), descr, p(one_row), p(sorted_ids), p(order),
                                 p(work)) == L.SUCCESS
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=DEV)
    assert lib.aclsparseXcoo2csr(h.raw, p(sorted_ids), ids.numel(), experts, p(offsets), L.BASE_ZERO) == L.SUCCESS
    torch.cuda.synchronize()
    lib.aclsparseDestroyMatDescr(descr)
    return gates, order.long(), offsets


@pytest.mark.parametrize("tokens,experts,top", [(1, 4, 2), (37, 8, 2), (200, 5, 3)])
def test_expert_layer_from_routing_to_combination(tokens, experts, top):
    """csrsort and coo2csr sort the routing, two grouped products compute, SpMM takes the gated sum, in bf16."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    k, inner = 64, 96
    x = randn(tokens, k, dtype=torch.bfloat16, gen=gen)
    up, down = randn(experts, inner, k, dtype=torch.bfloat16, gen=gen) / 8, randn(experts, k, inner, dtype=torch.bfloat16, gen=gen) / 8
    gates, order, offsets = route(tokens, experts, top, gen)
    rows = x[order // top]
    hidden = torch.relu(A.grouped_mm(rows, up, offsets))
    out = A.grouped_mm(hidden, down, offsets)
    # C = G * out with G the tokens x slots gate matrix: slot order[i] // top, gate of that choice
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=DEV)
    y = torch.empty(tokens, k, dtype=torch.float32, device=DEV)
    mat = api.CsrMatrix(tokens, order.numel(), torch.arange(0, tokens * top + 1, top, dtype=torch.int32, device=DEV),
                        place.to(torch.int32), gates.reshape(-1).to(torch.bfloat16).contiguous())
    spmm = api.SpMM(api.Handle(), mat, api.DnMat(order.numel(), k, k, out), api.DnMat(tokens, k, k, y))
    spmm.preprocess()
    spmm()
    # every step in 64 bits on that step's own inputs
    bounds = offsets.tolist()
    assert bounds[0] == 0 and bounds[-1] == tokens * top
    for got, a, w in ((hidden, rows, up), (out, hidden, down)):
        a64, w64 = a.double(), w.double()
        want = plain_grouped(a64, w64, bounds)
        close(got, torch.relu(want) if got is hidden else want,
              sum_bound(a.shape[1], plain_grouped(a64.abs(), w64.abs(), bounds), False))
    g64 = gates.to(torch.bfloat16).double()
    picked = out.double()[place].view(tokens, top, k)
    want = (g64[:, :, None] * picked).sum(1)
    close(y, want, 2.0 ** -40 * (g64[:, :, None] * picked.abs()).sum(1))


def test_expert_layer_in_8_bits():
    """Quantised rows and weights through the int8 product, against the same whole numbers in 64 bits."""
    gen = torch.Generator(device=DEV).manual_seed(8)
    x, w = randn(50, 128, dtype=torch.bfloat16, gen=gen), randn(4, 72, 128, dtype=torch.bfloat16, gen=gen)
    offsets = torch.tensor([0, 10, 10, 49, 50], dtype=torch.int32, device=DEV)
    xq, xs = A.quantize_rows(x)
    wq, ws = A.quantize_rows(w.view(-1, 128))
    y = A.int8_mm(xq, wq.view(4, 72, 128), xs, ws, offsets)
    want = plain_grouped(xq.double(), wq.view(4, 72, 128).double(), offsets.tolist()) * xs.double()[:, None]
    for g in range(4):
        want[int(offsets[g]):int(offsets[g + 1])] *= ws.view(4, 72)[g].double()
    close(y, want, 8 * 2.0 ** -24 * want.abs())
    # and how near that is to the product that it stands for: half a step of each operand
    truth = plain_grouped(x.double(), w.double(), offsets.tolist())
    x_off, w_off = xs.double()[:, None] / 2, ws.view(4, 72, 1).double() / 2
    for g in range(4):
        r = slice(int(offsets[g]), int(offsets[g + 1]))
        a, b = x[r].double().abs(), w[g].double().abs()
        bound = (a + x_off[r]) @ (b + w_off[g]).T - a @ b.T
        assert ((want[r] - truth[r]).abs() <= bound + 1e-9).all()


def test_dense_8_bit_product_of_two_dimensions():
    gen = torch.Generator(device=DEV).manual_seed(9)
    xq, wq = randn(7, 96, dtype=torch.int8, gen=gen), randn(40, 96, dtype=torch.int8, gen=gen)
    xs, ws = torch.rand(7, generator=gen, device=DEV), torch.rand(40, generator=gen, device=DEV)
    want = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()
    close(A.int8_mm(xq, wq, xs, ws, out_dtype=torch.float32), want, 8 * 2.0 ** -24 * want.abs())


def test_adapter_checks_its_arguments():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 6, 8, dtype=torch.bfloat16, device=DEV)
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    for bad, error in ((lambda: A.grouped_mm(x, w), ValueError), (lambda: A.grouped_mm(x, w, offsets.long()), TypeError),
                       (lambda: A.grouped_mm(x, w, offsets[:2]), ValueError), (lambda: A.grouped_mm(x, w.half(), offsets), TypeError),
                       (lambda: A.grouped_mm(x[:, :7], w, offsets), ValueError), (lambda: A.grouped_mm(x.float(), w.float(), offsets), TypeError),
                       (lambda: A.grouped_mm(x, w, offsets.cpu()), TypeError),
                       (lambda: A.grouped_mm(x, w, offsets, out_dtype=torch.float16), TypeError),
                       (lambda: A.quantize_rows(x.to(torch.int8)), TypeError), (lambda: A.quantize_rows(x[0]), ValueError)):
        with pytest.raises(error):
            bad()
    assert A.grouped_mm(x[:0], w, offsets).shape == (0, 6)
    assert A.grouped_mm(x, w[:, :0], offsets).shape == (4, 0)
    y = A.grouped_mm(x[:0].requires_grad_(), w.requires_grad_(), offsets)
    gw, = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert gw.shape == w.shape and (gw == 0).all()


def test_gradient_of_a_broadcast_result():
    """dy with strides of zero, as the gradient of a sum has them, and a gradient for one operand only."""
    gen = torch.Generator(device=DEV).manual_seed(12)
    offsets = torch.tensor([0, 7, 20], dtype=torch.int32, device=DEV)
    x, w = randn(20, 24, dtype=torch.bfloat16, gen=gen), randn(2, 16, 24, dtype=torch.bfloat16, gen=gen)
    w1 = w.clone().requires_grad_()
    A.grouped_mm(x, w1, offsets).sum().backward()
    want = torch.stack([x[:7].double().sum(0).expand(16, 24), x[7:].double().sum(0).expand(16, 24)])
    size = torch.stack([x[:7].double().abs().sum(0).expand(16, 24), x[7:].double().abs().sum(0).expand(16, 24)])
    close(w1.grad, want, sum_bound(13, size, False))
    x1 = x.clone().requires_grad_()
    A.grouped_mm(x1, w, offsets).sum().backward()
    want = torch.cat([w[0].double().sum(0).expand(7, 24), w[1].double().sum(0).expand(13, 24)])
    size = torch.cat([w[0].double().abs().sum(0).expand(7, 24), w[1].double().abs().sum(0).expand(13, 24)])
    close(x1.grad, want, sum_bound(16, size, False))


@pytest.mark.parametrize("shift", [1, 8])
def test_shifted_operands_give_the_same(shift):
    """Views that start between two multiples of 16 bytes are computed in the same way as aligned ones."""
    gen = torch.Generator(device=DEV).manual_seed(13)
    offsets = torch.tensor([0, 70, 70, 200], dtype=torch.int32, device=DEV)

    def shifted(t):
        store = torch.empty(t.numel() + shift, dtype=t.dtype, device=DEV)
        return store[shift:].view(t.shape).copy_(t)

    x, w = randn(200, 1040, dtype=torch.bfloat16, gen=gen), randn(3, 96, 1040, dtype=torch.bfloat16, gen=gen)
    dy = randn(200, 96, dtype=torch.bfloat16, gen=gen)
    got = []
    for put in (lambda t: t, shifted):
        a, b = put(x).requires_grad_(), put(w).requires_grad_()
        y = A.grouped_mm(a, b, offsets)
        got.append((y, *torch.autograd.grad(y, (a, b), put(dy))))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,k", [(1, 64), (5, 0), (40, 0), (40, 72), (300, 77)])
def test_one_group_without_offsets(rows, k):
    """Every element is written, whatever the memory held."""
    gen = torch.Generator(device=DEV).manual_seed(14)
    x, w = randn(rows, k, dtype=torch.bfloat16, gen=gen), randn(1, 50, k, dtype=torch.bfloat16, gen=gen)
    full = torch.full((rows, 50), float("nan"), dtype=torch.bfloat16, device=DEV)
    del full  # the allocator hands this memory out again
    y = A.grouped_mm(x, w)
    close(y, x.double() @ w[0].double().T, sum_bound(k, x.double().abs() @ w[0].double().abs().T, False))


def test_training_step_replays_in_a_graph():
    gen = torch.Generator(device=DEV).manual_seed(10)
    offsets = torch.tensor([0, 30, 30, 64], dtype=torch.int32, device=DEV)
    x, w = randn(64, 64, dtype=torch.bfloat16, gen=gen), randn(3, 48, 64, dtype=torch.bfloat16, gen=gen)
    dy = randn(64, 48, dtype=torch.bfloat16, gen=gen)

    def step():
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = A.grouped_mm(a, b, offsets)
        return (y, *torch.autograd.grad(y, (a, b), dy))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(77, 301), (300, 1021), (513, 129)])
def test_gradient_odd_widths_in_aligned_rows(out, m, n):
    """Rows of C that start on multiples of 16 bytes but end between them: what is behind each stays."""
    wide = -(-n // 8) * 8
    Gradient([150, 0, 1, 700, 64, 65], m, n, torch.bfloat16, out, pad=(-m % 8, wide - n, wide - n + 8), first=3, behind=40,
             seed=m, batch_pad=8).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", [L.ORDER_ROW, L.ORDER_COL])
@pytest.mark.parametrize("k,n", [(77, 301), (200, 13), (1033, 130)])
def test_forward_odd_widths_in_aligned_rows(dtype, order, k, n):
    """What lies between the rows of A and B is in no sum, and what lies between those of C stays."""
    pad_b = -(k if order == L.ORDER_ROW else n) % 16
    case = Forward([40, 0, 9, 300], k, n, dtype, order=order, pad=(-k % 16, pad_b, -n % 16), seed=k, batch_pad=-n % 16)
    a, c = (t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1)) for t in (case.a, case.c))
    every = case.w if order == L.ORDER_ROW else case.w.transpose(1, 2)
    w = every.as_strided((*every.shape[:2], every.stride(1)), every.stride())
    poison = 127 if dtype == torch.int8 else float("nan")
    a[:, k:] = poison
    w[:, :, every.shape[2]:] = poison
    c0 = c.clone()
    case.check()
    assert torch.equal(c[:, n:], c0[:, n:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_operands_of_odd_widths_in_aligned_rows(dtype):
    case = Gradient([40, 0, 9, 300], 77, 301, dtype, pad=(3, 3, 3), seed=77)
    for t in (case.a, case.b):
        t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1))[:, t.shape[1]:] = float("nan")
    case.check()


@pytest.mark.parametrize("groups", [31, 33, 300])
def test_forward_and_gradient_of_many_groups(groups):
    sizes = [(7 * g) % 41 if g % 3 else 0 for g in range(groups)]
    Forward(sizes, 72, 1032, torch.bfloat16, first=1, behind=2, seed=groups).check()
    Gradient(sizes, 136, 264, torch.bfloat16, first=1, behind=2, seed=groups).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,k,n", [([1], 16400, 264), ([2, 0, 5], 8208, 40), ([20], 16400, 264), ([18, 0, 5, 30], 8208, 40),
                                       ([300], 12304, 264)])
def test_forward_long_sums_of_few_tiles(dtype, sizes, k, n):
    """Tiles split along the summed index into as many parts as there are CTAs for them, the last one short."""
    Forward(sizes, k, n, dtype, scales=True, seed=k).check()


@pytest.mark.parametrize("extra", [0, 1])
def test_operands_beyond_32_bits(extra):
    """Rows and matrices whose distance times their number passes 2^32 elements, aligned and not."""
    gen = torch.Generator(device=DEV).manual_seed(31)
    rows, k, n, ld = 40, 72, 136, 2 ** 27 + extra
    far = torch.empty((rows - 1) * ld + 160, dtype=torch.bfloat16, device=DEV)
    apart = 2 ** 31 + 8 + extra
    matrices = torch.empty(2 * apart + n * k, dtype=torch.bfloat16, device=DEV)
    x = torch.as_strided(far, (rows, k), (ld, 1))
    w = torch.as_strided(matrices, (3, n, k), (apart, k, 1))
    x0, w0 = randn(rows, k, dtype=torch.bfloat16, gen=gen), randn(3, n, k, dtype=torch.bfloat16, gen=gen)
    x.copy_(x0)
    w.copy_(w0)
    bounds = [0, 11, 11, rows]
    offsets = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    want, size = torch.zeros(rows, n, dtype=torch.float64, device=DEV), torch.zeros(rows, n, dtype=torch.float64, device=DEV)
    for g in range(3):
        part = slice(bounds[g], bounds[g + 1])
        want[part] = x0[part].double() @ w0[g].double().T
        size[part] = x0[part].double().abs() @ w0[g].double().abs().T
    y = A.grouped_mm(x, w, offsets)
    close(y, want, sum_bound(k, size, False))
    # the same rows as the result of a product, and the same matrices as that of a gradient
    c = torch.as_strided(far, (rows, n), (ld, 1))
    api.GroupedMM(api.Handle(), api.DnMat(rows, k, k, x0), api.DnMat(n, k, k, w0, L.ORDER_ROW, 3, n * k),
                  api.DnMat(rows, n, ld, c), offsets, L.OP_T)()
    close(c, want, sum_bound(k, size, False))
    dy = randn(rows, n, dtype=torch.bfloat16, gen=gen)
    api.GroupedMMWeightGrad(api.Handle(), api.DnMat(rows, n, n, dy), api.DnMat(rows, k, k, x0),
                            api.DnMat(n, k, k, matrices, L.ORDER_ROW, 3, apart), offsets)()
    for g in range(3):
        part = slice(bounds[g], bounds[g + 1])
        close(w[g], dy[part].double().T @ x0[part].double(),
              sum_bound(rows, dy[part].double().abs().T @ x0[part].double().abs(), False))
    q, scales = A.quantize_rows(torch.as_strided(far, (rows, n), (ld, 1)))
    want_q, want_scales = quantized(c)
    assert torch.equal(q, want_q) and torch.equal(scales, want_scales)


def test_products_on_two_streams_at_once():
    """Each with its own buffer: a long product and many short ones, split and joined, side by side."""
    long = Forward([3000, 1, 2000], 1024, 2048, torch.bfloat16, seed=1)
    short = Forward([20], 8208, 264, torch.bfloat16, seed=2)
    few = Forward([2, 1], 520, 264, torch.bfloat16, seed=5)
    grad = Gradient([900, 0, 300], 256, 264, torch.bfloat16, seed=3)
    cases = [long, short, grad, few]
    wants = []
    for case in cases:
        case.op()
        torch.cuda.synchronize()
        wants.append(case.c.clone())
    streams = [torch.cuda.Stream() for _ in cases]
    for case, stream in zip(cases, streams):
        case.op.handle = api.Handle(stream)
        case.c.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for case, times in ((long, 1), (short, 5), (grad, 3), (few, 9)):
            for _ in range(times):
                case.op()
    torch.cuda.synchronize()
    for case, want in zip(cases, wants):
        assert torch.equal(case.c, want)
        assert case.op.wait_failures() == 0


def test_eager_and_replayed_products_take_turns_over_one_buffer():
    case = Forward([5, 0, 70], 4104, 264, torch.bfloat16, seed=4)
    case.op.preprocess()
    case.op()
    want = case.c.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eager, handle = case.op.handle, api.Handle(side)
    graph = torch.cuda.CUDAGraph()
    case.op.handle = handle
    with torch.cuda.graph(graph, stream=side):
        case.op()
        case.op()
    case.op.handle = eager
    for turn in range(6):
        case.c.zero_()
        graph.replay() if turn % 2 else case.op()
        assert torch.equal(case.c, want)
