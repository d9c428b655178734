"""Results of the low-rank adapters in a tensor that takes part in a graph."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import adapters_case, rand

pytestmark = pytest.mark.gpu


def test_out_with_a_history_is_refused():
    """It would keep its history: the gradient of what was written over it would go to what it was made from."""
    x, base, a, b, scale, ids, starts, _ = adapters_case(90, 4, 2, 64, 96, 8, torch.float32, 3)
    leaf = rand(base.shape, torch.float32, 1).requires_grad_()
    for out in (leaf, leaf * 2.0):
        before = out.detach().clone()
        with pytest.raises(RuntimeError, match="without gradients"):
            digital.low_rank_add(base, x, a, b, scale, ids, starts, out=out)
        assert torch.equal(out, before)
    want = digital.low_rank_add(base, x, a, b, scale, ids, starts)
    out = torch.empty_like(base)
    assert digital.low_rank_add(base, x, a, b, scale, ids, starts, out=out) is not None and torch.equal(out, want)
    with torch.no_grad():  # as torch's own operations with out=
        digital.low_rank_add(base, x, a, b, scale, ids, starts, out=leaf)
    assert torch.equal(leaf, want)
