"""Long sums of the low-rank adapters are rounded, not cut off.

The matrix unit cuts off what an addition shifts out of its sum, by up to 2^-22 of it, always toward zero: over a long sum
of terms of one sign that adds up to an error in one direction.  The kernels leave it few additions in a row and add its sums up
by additions that round.  Those are off either way, so the mean relative error over many results shows the cut additions
alone: at most CHAIN of them of every product's sum, and what the split factors leave out, 2^-21."""

import pytest
import torch

from aihwkit_b200 import _cabi
from tests.test_digital_gpu import IDS, TYPES

pytestmark = pytest.mark.gpu

CUT, LEFT_OUT = 2.0 ** -22, 2.0 ** -21
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def positive(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(shape, device="cuda", generator=g) + 0.5).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def mean_error(got, want):
    return abs(float((got.double() / want - 1).mean()))


def apply(x, a, b, y, v, starts=None):
    rows, rank = x.size(0), a.size(1)
    ids = ints(0) if starts is not None else torch.zeros(rows, dtype=torch.int32, device="cuda")
    scale = torch.ones(1, device="cuda")
    ptr = lambda t: None if t is None else t.data_ptr()
    n = 8 if b is None else b.size(2)
    _cabi.check(_cabi.lib().ab200_low_rank_apply(
        ptr(x), x.size(1), None, 0, ptr(y), n, ptr(a), ptr(b), ptr(scale), ptr(ids), ptr(starts),
        ids.numel(), rows, x.size(1), n, rank, 1, CODE[x.dtype], ptr(v), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("k", [16384, 16381])
@pytest.mark.parametrize("rank", [8, 16, 32, 64])
@pytest.mark.parametrize("single", [False, True], ids=["long", "single"])
def test_first_product(single, rank, k, dtype):
    rows = 1024
    x, a = positive((rows, k), dtype, 1), positive((1, rank, k), dtype, 2)
    v = torch.zeros(rows, rank, device="cuda")
    apply(x, a, None, None, v, None if single else ints(0, rows))
    # additions to a sum of full size in a step of 64 bytes: of 16-bit types its two halves; of fp32 the largest of the first half's
    # three terms (the two before it make sums 2^-11 of that) and the second half's three
    chain = 4 if dtype == torch.float32 else 2
    assert mean_error(v, x.double() @ a[0].double().t()) <= chain * CUT + LEFT_OUT


@pytest.mark.parametrize("single", [False, True], ids=["long", "single"])
@pytest.mark.parametrize("rank", [64, 256])
def test_second_product(single, rank):
    """fp32, whose results are not rounded further.  Sixteen ranks in a sum: the smaller terms first, then two of full size; v has
    its own error."""
    rows, k, n = 256, 16, 4096
    x, a, b = positive((rows, k), torch.float32, 1), positive((1, rank, k), torch.float32, 2), positive((1, rank, n), torch.float32, 3)
    y = torch.zeros(rows, n, device="cuda")
    apply(x, a, b, y, None, None if single else ints(0, rows))
    want = (x.double() @ a[0].double().t()) @ b[0].double()
    assert mean_error(y, want) <= (3 + 3) * CUT + 2 * LEFT_OUT


@pytest.mark.parametrize("width", [4096, 4095])
@pytest.mark.parametrize("rank", [16, 32, 64])
def test_gradient(rank, width):
    """fp32 again.  Sums over 65536 rows, in chunks of 2048."""
    import ctypes as C

    rows = 65536
    lib = _cabi.lib()
    x, u = positive((rows, width), torch.float32, 1), positive((rows, rank), torch.float32, 2)
    grad = torch.zeros(1, rank, width, device="cuda")
    size = C.c_longlong()
    _cabi.check(lib.ab200_low_rank_grad_workspace(rows, 1, 0, width, 0, rank, C.byref(size)))
    work = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    ids, starts = ints(0), ints(0, rows)
    _cabi.check(lib.ab200_low_rank_grad(x.data_ptr(), width, u.data_ptr(), grad.data_ptr(), width, None, 0, None, None, 0,
                                        ids.data_ptr(), starts.data_ptr(), 1, rows, rank, 1, 0, work.data_ptr(),
                                        torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    want = sum(u[r:r + 8192].double().t() @ x[r:r + 8192].double() for r in range(0, rows, 8192))
    assert mean_error(grad[0], want) <= 3 * CUT + LEFT_OUT
