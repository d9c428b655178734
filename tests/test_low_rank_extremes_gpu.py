"""Low-rank adapters at the largest finite values: finite products and sums stay finite."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import F, adapters_exact, rand, unit, within

pytestmark = pytest.mark.gpu


def tables(rows, single):
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return (as_int([0] * rows), None) if single else (as_int([0]), as_int([0, rows]))


@pytest.mark.parametrize("single", [False, True], ids=["long", "single"])
def test_largest_finite_values_fp32(single):
    """The lowest value of the type in x and in the factors: finite products stay finite."""
    rows, k, n, rank = 40, 64, 48, 8
    low = torch.finfo(torch.float32).min
    ids, starts = tables(rows, single)
    scale = torch.ones(1, device="cuda")
    per_row = torch.zeros(rows, device="cuda")
    x, base = rand((rows, k), torch.float32, 1, 2.0 ** -4), rand((rows, n), torch.float32, 2)
    a, b = rand((1, rank, k), torch.float32, 3, 2.0 ** -20), rand((1, rank, n), torch.float32, 4, 2.0 ** -20)
    for place in ("x", "a", "b"):
        t = dict(x=x.clone(), a=a.clone(), b=b.clone())
        if place == "x":
            t["x"][::3, 5], t["x"][1::3, 7] = low, -low
        else:
            t[place][0, 2, 5], t[place][0, 3, 7] = low, -low
        y64, off, _, _ = adapters_exact(t["x"], base, t["a"], t["b"], scale, per_row)
        y = digital.low_rank_add(base, t["x"], t["a"], t["b"], scale, ids, starts)
        within(y, y64, F * y64.abs() + off, place)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("single", [False, True], ids=["long", "single"])
def test_largest_finite_values_between_the_products(single, dtype):
    """v = (2 - 2^-9) 2^127 lies above the largest bf16 value and below the largest fp32 one; its product with b is finite."""
    rows, k, n, rank = 40, 64, 64, 8
    ids, starts = tables(rows, single)
    scale = torch.ones(1, device="cuda")
    for sign in (1.0, -1.0):
        x, a = torch.zeros(rows, k, dtype=dtype, device="cuda"), torch.zeros(1, rank, k, dtype=dtype, device="cuda")
        x[:, :2] = sign * 2.0 ** 100
        a[0, 0, 0], a[0, 0, 1] = (2 - 2.0 ** -7) * 2.0 ** 27, 1.5 * 2.0 ** -8 * 2.0 ** 27
        b = torch.full((1, rank, n), 2.0 ** -30, dtype=dtype, device="cuda")
        b[0, 1:] = 0
        base = torch.zeros(rows, n, dtype=dtype, device="cuda")
        y = digital.low_rank_add(base, x, a, b, scale, ids, starts)
        want = torch.tensor(sign * (2 - 2.0 ** -7 + 1.5 * 2.0 ** -8) * 2.0 ** 97, dtype=torch.float64).to(dtype)
        assert (y == want.cuda()).all()
        # u of the gradient of a factor: the same value, from gy and b
        leaf = torch.zeros(1, rank, n, dtype=dtype, device="cuda").requires_grad_()
        small = torch.full((rows, n), 2.0 ** -30, dtype=dtype, device="cuda")
        out = digital.low_rank_add(torch.zeros(rows, k, dtype=dtype, device="cuda"), small, leaf, a, scale, ids, starts)
        grad, = torch.autograd.grad(out, leaf, x)
        v = sign * (2 - 2.0 ** -7 + 1.5 * 2.0 ** -8) * 2.0 ** 97 * rows
        # forty equal terms of three parts each, every addition off by 2^-22 at most, then one rounding
        assert ((grad[0, 0].double() / v - 1).abs() <= 200 * 2.0 ** -22 + unit(dtype)).all() and (grad[0, 1:] == 0).all()
