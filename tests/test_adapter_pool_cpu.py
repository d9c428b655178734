"""A pool of adapters under the conversions of a module."""

import copy

import pytest
import torch

from aihwkit_b200 import digital


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_scale_stays_in_fp32(dtype):
    pool = digital.LowRankAdapters(2, 10, 6, 4, scale=1.0 / 3.0, device="cpu")
    model = torch.nn.Sequential(pool).to(dtype)
    assert model[0] is pool and pool.a.dtype == pool.b.dtype == dtype
    assert pool.scale.dtype == torch.float32 and pool.scale.tolist() == [torch.tensor(1.0 / 3.0).item()] * 2
    pool.set_adapter(1, torch.ones(2, 10), torch.ones(6, 2), 0.1)
    assert pool.scale[1].item() == torch.tensor(0.1).item()
    other = copy.deepcopy(pool).half()
    assert other.scale.dtype == torch.float32 and torch.equal(other.scale, pool.scale)
    state = pool.state_dict()
    assert state["scale"].dtype == torch.float32 and "scale" in dict(pool.named_buffers())
    other.load_state_dict(state)


def test_conversion_without_values():
    pool = digital.LowRankAdapters(2, 10, 6, 4, device="cpu").to("meta").half()
    assert pool.scale.is_meta and pool.scale.dtype == torch.float32
    pool = pool.to_empty(device="cpu").half()
    assert pool.scale.device.type == "cpu" and pool.scale.dtype == torch.float32
