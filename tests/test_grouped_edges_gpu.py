"""Calls of the grouped products that their documentation allows and that went wrong, or could: offsets that do not
ascend, buffers whose memory had another use, products side by side that share nothing but the GPU."""
import numpy as np
import pytest
import torch

from ops_sparse_b200 import _lib as L
from ops_sparse_b200 import api
from ops_sparse_b200 import torch_adapter as A
from tests.test_grouped_gpu import DEV, Forward, Gradient, close, randn, sum_bound

pytestmark = pytest.mark.gpu


def ascending(bounds, rows):
    """Each offset inside the matrix, and none below one before it."""
    top, out = 0, []
    for b in bounds:
        top = max(top, min(max(b, 0), rows))
        out.append(top)
    return out


def check_gradient(case, bounds):
    case.offsets.copy_(torch.tensor(bounds, dtype=torch.int32))
    case.bounds = ascending(bounds, case.a.shape[0])
    case.check()


@pytest.mark.parametrize("shift", [(0, 0, 0), (1, 0, 0)], ids=["tensor cores", "plain"])
@pytest.mark.parametrize("bounds", [[-5, 40, 20, 2 ** 31 - 1], [0, 50, 20, 80], [90, 60, 30, 0], [-7, 10, 10 ** 9, 90],
                                    [2 ** 31 - 1, -2 ** 31, 5, 6], [30, 10, 60, 40]])
def test_gradient_of_bad_offsets_has_every_row_once_at_most(bounds, shift):
    """The groups are those of the forward product, so that the gradient stays its derivative."""
    check_gradient(Gradient([30, 30, 30], 64, 48, torch.bfloat16, pad=(8, 8, 0), shift=shift), bounds)


@pytest.mark.parametrize("shift", [(0, 0, 0), (0, 1, 0)], ids=["tensor cores", "plain"])
@pytest.mark.parametrize("groups", [31, 32, 33, 64, 300])
def test_gradient_of_bad_offsets_of_many_groups(groups, shift):
    case = Gradient([3] * groups, 136, 72, torch.bfloat16, pad=(8, 8, 0), shift=shift, seed=groups)
    rows = 3 * groups
    steps = torch.randint(-40, 61, (groups + 1,), generator=torch.Generator().manual_seed(groups))
    check_gradient(case, (torch.arange(groups + 1) * rows // groups + steps).tolist())


@pytest.mark.parametrize("bounds", [[0, 9000, 3000, 12000], [4000, 100, 11000, 11999], [0, 12000, 5000, 12000]])
def test_gradient_of_bad_offsets_split_along_the_rows(bounds):
    check_gradient(Gradient([4000, 4000, 4000], 136, 264, torch.bfloat16, seed=4), bounds)


def test_gradient_of_bad_offsets_is_the_derivative_of_the_product():
    """Through the adapter: what autograd gets is the formula's gradient for the rows that the product used."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    x, w = randn(90, 64, dtype=torch.bfloat16, gen=gen), randn(3, 48, 64, dtype=torch.bfloat16, gen=gen)
    dy = randn(90, 48, dtype=torch.bfloat16, gen=gen)
    offsets = torch.tensor([0, 50, 20, 80], dtype=torch.int32, device=DEV)
    w1 = w.clone().requires_grad_()
    y = A.grouped_mm(x, w1, offsets, out_dtype=torch.float32)
    gw, = torch.autograd.grad(y, w1, dy.float())
    for g, (first, last) in enumerate([(0, 50), (50, 50), (50, 80)]):
        r = slice(first, last)
        close(y[r].detach(), x[r].double() @ w[g].double().T, sum_bound(64, x[r].double().abs() @ w[g].double().abs().T, False))
        close(gw[g], dy[r].double().T @ x[r].double(), sum_bound(50, dy[r].double().abs().T @ x[r].double().abs(), False))


# ---- buffers ----

def split_product():
    """A product whose tiles are split, so that it lives by the counters in its buffer, and its result."""
    case = Forward([20], 16400, 264, torch.bfloat16)
    case.op.preprocess()
    case.op()
    torch.cuda.synchronize()
    want, size = case.expected()
    close(case.c, want, sum_bound(case.k, size, False))
    return case, case.c.clone()


def again(case):
    return api.GroupedMM(case.op.handle, case.op.a, case.op.b, case.op.c, case.op.offsets, case.op.op_b)


def test_a_buffer_at_the_address_of_an_earlier_one_is_cleared():
    """The result's descriptor remembers a Preprocess by the buffer's address; the memory has had another use since."""
    case, want = split_product()
    address, size, op = case.op.buffer.data_ptr(), case.op.buffer.numel(), again(case)
    case.op = None
    other = torch.empty(size, dtype=torch.uint8, device=DEV).fill_(0xAB)
    assert other.data_ptr() == address
    del other
    case.c.zero_()
    op()
    assert op.buffer.data_ptr() == address and torch.equal(case.c, want)


def test_a_buffer_that_is_handed_over_is_cleared():
    case, want = split_product()
    buffer, op = case.op.buffer, again(case)
    for fresh in (op, case.op):  # another operator's, and the same one's again
        buffer.fill_(0xCD)
        fresh.buffer = buffer
        case.c.zero_()
        fresh()
        assert torch.equal(case.c, want)
    case.op.preprocess()
    case.c.zero_()
    case.op()
    assert torch.equal(case.c, want)


def test_asking_for_the_size_ends_a_preprocess():
    """As a program in C does that frees its buffer, asks for the size again and goes on without a Preprocess."""
    case, want = split_product()
    case.op.buffer.fill_(0xEF)
    case.op.buffer_size()
    case.c.zero_()
    case.op()
    assert torch.equal(case.c, want)


def test_gradient_buffer_at_the_address_of_an_earlier_one_is_cleared():
    case = Gradient([9000], 136, 264, torch.bfloat16)
    case.op.preprocess()
    case.op()
    want, (handle, a, b, c, offsets) = case.c.clone(), (case.op.handle, case.op.a, case.op.b, case.op.c, case.op.offsets)
    address, size = case.op.buffer.data_ptr(), case.op.buffer.numel()
    case.op = None
    other = torch.empty(size, dtype=torch.uint8, device=DEV).fill_(0xAB)
    assert other.data_ptr() == address
    del other
    case.c.zero_()
    op = api.GroupedMMWeightGrad(handle, a, b, c, offsets)
    op()
    assert op.buffer.data_ptr() == address and torch.equal(case.c, want)
    want64, size64, most = case.expected()
    close(case.c, want64, sum_bound(most, size64, False))


def test_plans_of_sparse_products_outlive_any_number_of_grouped_products():
    """A grouped product without Preprocess keeps no plan in its buffer: a thousand buffers push no SpMV plan out."""
    from tests.gpu_util import SpmvCase, random_csr
    row_ptr, col_ind = random_csr(np.random.default_rng(3), [8] * 300, 200)
    sparse = SpmvCase(row_ptr, col_ind, np.ones(2400), np.ones(200), np.zeros(300))
    sparse.run()
    before = api.kernel_launches()
    sparse.run(preprocess=False)
    each = api.kernel_launches() - before
    x, w = torch.randn(2, 64, device=DEV).bfloat16(), torch.randn(1, 32, 64, device=DEV).bfloat16()
    c = torch.empty(2, 32, device=DEV)
    op = api.GroupedMM(api.Handle(), api.DnMat(2, 64, 64, x), api.DnMat(32, 64, 64, w), api.DnMat(2, 32, 32, c), op_b=L.OP_T)
    size = -(-op.buffer_size() // 64) * 64
    many = torch.empty(1100 * size, dtype=torch.uint8, device=DEV)
    for i in range(1100):
        op.buffer = many[i * size:(i + 1) * size]
        op()
    before = api.kernel_launches()
    sparse.run(preprocess=False)
    assert api.kernel_launches() - before == each


# ---- operands cut out of larger ones ----

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 20])
def test_rows_cut_out_of_a_matrix_of_odd_width_are_computed_as_others(dtype, rows):
    """The same kernel, and so the same bits; one row's stride is that of the matrix it was cut out of."""
    gen = torch.Generator(device=DEV).manual_seed(23)
    big = randn(40, 777, dtype=dtype, gen=gen)
    x = big[3:3 + rows, :776]
    w = randn(1, 520, 776, dtype=dtype, gen=gen)
    got = A.grouped_mm(x, w, out_dtype=torch.float32)
    close(got, x.double() @ w[0].double().T, sum_bound(776, x.double().abs() @ w[0].double().abs().T, False))
    if rows == 1:  # more rows of an odd pitch go through the library's own copy
        assert x.stride(0) == 777 and x.data_ptr() % 16 != 0
    assert torch.equal(got, A.grouped_mm(x.contiguous().clone(), w, out_dtype=torch.float32))
    odd = randn(2, 521, 777, dtype=dtype, gen=gen)[1:2, 1:2, :776]  # one row of one matrix, as weights
    assert torch.equal(A.grouped_mm(x, odd, out_dtype=torch.float32),
                       A.grouped_mm(x.contiguous().clone(), odd.contiguous().clone(), out_dtype=torch.float32))


def test_one_int8_row_cut_out_of_a_matrix_of_odd_width():
    gen = torch.Generator(device=DEV).manual_seed(24)
    x, w = randn(5, 777, dtype=torch.int8, gen=gen)[2:3, :768], randn(264, 768, dtype=torch.int8, gen=gen)
    one, scales = torch.ones(1, device=DEV), torch.ones(264, device=DEV)
    assert x.data_ptr() % 16 != 0
    assert torch.equal(A.int8_mm(x, w, one, scales, out_dtype=torch.float32).double(), x.double() @ w.double().T)


# ---- side by side ----

def test_prepared_products_side_by_side_reuse_their_counters():
    """Four streams, each with a buffer that is cleared once: split tiles leave their counters at zero for the next product,
    with others' tiles on the same SMs, and no wait runs out in any of them."""
    long = Forward([3000, 1, 2000], 1024, 2048, torch.bfloat16, seed=1)
    split = Forward([20], 16400, 264, torch.bfloat16, seed=2)
    int8 = Forward([40, 9], 8208, 264, torch.int8, seed=5)
    grad = Gradient([9000, 0, 3000], 256, 264, torch.bfloat16, seed=3)
    turns = ((long, 1), (split, 5), (grad, 3), (int8, 9))
    wants = []
    for case, _ in turns:
        case.check()
        wants.append(case.c.clone())
    for case, _ in turns:
        case.op.handle = api.Handle(torch.cuda.Stream())
        case.c.zero_()
    torch.cuda.synchronize()
    before = api.grouped_wait_failures()
    for case, _ in turns:
        case.op.preprocess()
    launches = api.kernel_launches()
    for _ in range(20):
        for case, times in turns:
            for _ in range(times):
                case.op()
    assert api.kernel_launches() - launches == 20 * sum(times for _, times in turns)  # nobody cleared anything again
    torch.cuda.synchronize()
    for (case, _), want in zip(turns, wants):
        assert torch.equal(case.c, want)
        assert case.op.wait_failures() == 0
    assert api.grouped_wait_failures() == before


def test_a_buffer_stays_its_streams_own_until_the_product_has_run():
    """An operator on a stream of its own, dropped while its product waits there: nobody else gets the buffer before."""
    case, want = split_product()
    side = torch.cuda.Stream()
    handle = api.Handle(side)
    op = api.GroupedMM(handle, case.op.a, case.op.b, case.op.c, case.op.offsets, case.op.op_b)
    case.c.zero_()
    torch.cuda.synchronize()
    op.preprocess()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # a tenth of a second
    op()
    size = op.buffer.numel()
    del op  # the handle lives on: destroying it would wait for the stream
    others = [torch.full((size,), 0xAB, dtype=torch.uint8, device=DEV) for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(case.c, want)
    del others, handle


def test_a_product_without_results_leaves_no_count_of_failures():
    """Nothing is launched for it, and whatever its buffer's memory held is no count."""
    for case in (Forward([0, 0], 64, 48, torch.bfloat16), Gradient([5], 64, 0, torch.bfloat16)):
        case.op.allocate().fill_(0xAB)
        case.op()
        assert case.op.wait_failures() == 0
