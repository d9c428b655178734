"""A converted pool of adapters in use."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_converted_pool(dtype):
    pool = digital.LowRankAdapters(2, 64, 96, 8, scale=1.0 / 3.0)
    with torch.no_grad():
        pool.b.copy_(rand(pool.b.shape, torch.float32, 1))
    a, b = pool.a.detach().to(dtype), pool.b.detach().to(dtype)
    pool.to(dtype)
    x, base = rand((20, 64), dtype, 2), rand((20, 96), dtype, 3)
    ids = torch.arange(20, dtype=torch.int32, device="cuda") % 2
    want = digital.low_rank_add(base, x, a, b, torch.full((2,), 1.0 / 3.0, device="cuda"), ids)
    got = pool(base, x, ids)
    assert torch.equal(got, want)
    got.float().sum().backward()
    assert pool.a.grad.dtype == pool.b.grad.dtype == dtype
