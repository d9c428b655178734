"""Forward-mode differentiation and tracing of the digital operators are refused before anything else is looked at: host
tensors, which the operators do not compute, show it."""

import pytest
import torch
import torch.autograd.forward_ad as ad

from aihwkit_b200 import digital

IDS = torch.zeros(2, dtype=torch.int32)
CALLS = {
    "dropout": (lambda x, r: digital.dropout(x, 0.5, residual=r), 2),
    "layer_norm": (lambda x, w, b: digital.layer_norm(x, w, b), 3),
    "add_layer_norm": (lambda x, r, w, b: digital.add_layer_norm(x, r, w, b), 4),
    "low_rank_add": (lambda base, x, a, b, scale: digital.low_rank_add(base, x, a, b, scale, IDS), 5),
    "low_rank_add in place": (lambda base, x, a, b, scale: digital.low_rank_add(x, x, a, b, scale, IDS, out=base), 5)}


@pytest.mark.parametrize("name", CALLS)
def test_dual_tensors_are_refused(name):
    fn, n = CALLS[name]
    for i in range(n):
        with ad.dual_level():
            args = [torch.ones(2, 8) for _ in range(n)]
            args[i] = ad.make_dual(args[i], torch.ones(2, 8))
            with pytest.raises(RuntimeError, match="forward-mode"):
                fn(*args)
            with ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="no CPU compute path"):
                fn(*args)


@pytest.mark.parametrize("name", CALLS)
def test_tracing_is_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, n = CALLS[name]
    args = tuple(torch.ones(2, 8) for _ in range(n))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(fn, args, check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(fn)(*args)
    with pytest.raises(RuntimeError, match="no CPU compute path"):  # and nothing of it stays behind
        fn(*args)
