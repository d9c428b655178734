"""Gradients of low-rank adapters on the widest rows that the calls take."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import rand, unit, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradient_of_the_widest_rows(dtype):
    """Widths whose columns are more blocks than a grid takes in its second dimension (65535)."""
    k = 1 << 24
    rows, n = 20, 8
    x = rand((rows, k), dtype, 1).requires_grad_()
    a, b = rand((1, 1, k), dtype, 2, 2.0 ** -12).requires_grad_(), rand((1, 1, n), dtype, 3)
    base, gy = torch.zeros(rows, n, dtype=dtype, device="cuda"), rand((rows, n), dtype, 4)
    ids, starts = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0], [0, rows]))
    y = digital.low_rank_add(base, x, a, b, torch.ones(1, device="cuda"), ids, starts)
    dx, da = torch.autograd.grad(y, [x, a], gy)
    u = gy.double() @ b[0].double().t()
    u_mag = gy.double().abs() @ b[0].double().abs().t()
    for part in range(0, k, 1 << 20):
        cols = slice(part, part + (1 << 20))
        xs = x.detach()[:, cols].double()
        want = (u * xs).sum(0)
        # two sums, of 8 and of 20 terms, whose additions are off by 2^-22 at most, products of split factors by 2^-21
        bound = unit(dtype) * want.abs() + (u_mag * xs.abs()).sum(0) * (40 * 2.0 ** -22 + 2 * 2.0 ** -21)
        within(da[0, 0, cols], want, bound, "da")
        want = u * a.detach()[0, :, cols].double()
        within(dx[:, cols], want, unit(dtype) * want.abs() + u_mag * a.detach()[0, :, cols].double().abs() * 40 * 2.0 ** -21, "dx")
