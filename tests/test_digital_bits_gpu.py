"""What the low-rank adapters keep of their factors between the two products, at values where every sum is exact.

A dot product of 1, 2^-10 and 2^-20 has 21 significant bits.  Two such values that differ in the last of them alone meet with
opposite signs, so the result is that last bit, or nothing where fewer bits were kept.  All terms are powers of two within
2^21 of each other, sums of them have at most 22 bits, and the results are powers of two: equality, no tolerance."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import IDS, TYPES

pytestmark = pytest.mark.gpu

BITS = [1.0, 2.0 ** -10, 2.0 ** -20]
FEWER = [1.0, 2.0 ** -10, 0.0]


def tables(rows, single):
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return (as_int([0] * rows), None) if single else (as_int([0]), as_int([0, rows]))


def filled(shape, *rows_of, dtype):
    """Zeros with the values of ``rows_of`` at the start of rows 0, 1, ... of the last but one dimension, in turn."""
    t = torch.zeros(shape, dtype=dtype, device="cuda")
    for r in range(shape[-2]):
        values = rows_of[r % len(rows_of)]
        t[..., r, :len(values)] = torch.tensor(values, dtype=torch.float64).to(dtype)
    return t


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("single", [False, True], ids=["long", "single"])
@pytest.mark.parametrize("rows, k, n, rank", [(64, 64, 64, 2), (40, 33, 17, 2), (80, 96, 128, 8), (70, 64, 64, 20), (48, 64, 64, 40)])
def test_first_product_keeps_all_bits(rows, k, n, rank, single, dtype):
    ids, starts = tables(rows, single)
    x = filled((rows, k), BITS, dtype=dtype)
    a = filled((1, rank, k), [1.0, 1.0, 1.0], [1.0, 1.0, 0.0], dtype=dtype)
    b = torch.zeros(1, rank, n, dtype=dtype, device="cuda")
    b[0, 0], b[0, 1] = 1.0, -1.0
    a[0, 2:] = 0
    scale = torch.ones(1, device="cuda")
    base = torch.zeros(rows, n, dtype=dtype, device="cuda")
    y = digital.low_rank_add(base, x, a, b, scale, ids, starts)
    assert (y.double() == 2.0 ** -20).all()
    # the gradient of x is the same product on other factors
    leaf = torch.zeros(rows, n, dtype=dtype, device="cuda").requires_grad_()
    out = digital.low_rank_add(torch.zeros_like(x), leaf, b, a, scale, ids, starts)
    dx, = torch.autograd.grad(out, leaf, x)
    assert (dx.double() == 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("single", [False, True], ids=["long", "single"])
@pytest.mark.parametrize("rows, k, n, rank", [(64, 64, 64, 1), (40, 33, 17, 3), (70, 64, 64, 20), (48, 64, 64, 40)])
def test_gradients_of_the_factors_keep_all_bits(rows, k, n, rank, single, dtype):
    """da = u^T x with u in turn with and without its last bit, and x in turn 1 and -1: a half of the rows times 2^-20."""
    ids, starts = tables(rows, single)
    one = filled((1, rank, k), [1.0] * 3, dtype=dtype)
    b = filled((1, rank, n), [1.0] * 3, dtype=dtype)
    scale = torch.ones(1, device="cuda")
    sign = torch.ones(rows, 1, dtype=dtype, device="cuda")
    sign[1::2] = -1
    want = rows // 2 * 2.0 ** -20
    b_leaf, a_leaf = b.clone().requires_grad_(), one.clone().requires_grad_()
    base = torch.zeros(rows, n, dtype=dtype, device="cuda")
    out = digital.low_rank_add(base, sign.expand(rows, k).contiguous(), a_leaf, b, scale, ids, starts)
    da, = torch.autograd.grad(out, a_leaf, filled((rows, n), BITS, FEWER, dtype=dtype))
    assert (da.double() == want).all()
    out = digital.low_rank_add(base, filled((rows, k), BITS, FEWER, dtype=dtype), one, b_leaf, scale, ids, starts)
    db, = torch.autograd.grad(out, b_leaf, sign.expand(rows, n).contiguous())
    assert (db.double() == want).all()
