"""Single rows of one adapter, which share the tiles of the low-rank adapters."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import IDS, TYPES, adapters_exact, rand, unit, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_lists_of_single_rows_repeat(dtype):
    """Single rows of one adapter share tiles, among requests of two to twelve rows: the same bits in each of many calls, in
    which blocks come and go in other orders."""
    rng = torch.Generator().manual_seed(4)
    lengths = torch.randint(0, 4, (700,), generator=rng)
    lengths[::9] = torch.randint(2, 13, (lengths[::9].numel(),), generator=rng)
    starts = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)]).int().cuda()
    ids = torch.randint(-1, 5, (700,), generator=rng).int().cuda()
    rows, k, n = int(lengths.sum()), 128, 160
    x, base = rand((rows, k), dtype, 1), rand((rows, n), dtype, 2)
    a, b, scale = rand((5, 8, k), dtype, 3, k ** -0.5), rand((5, 8, n), dtype, 4, 0.35), torch.rand(5, device="cuda") + 0.5
    per_row = torch.repeat_interleave(ids.long(), lengths.cuda())
    y64, off, _, _ = adapters_exact(x, base, a, b, scale, per_row)
    first = digital.low_rank_add(base, x, a, b, scale, ids, starts)
    within(first, y64, unit(dtype) * y64.abs() + off, "y")
    for _ in range(50):
        assert torch.equal(digital.low_rank_add(base, x, a, b, scale, ids, starts), first)
