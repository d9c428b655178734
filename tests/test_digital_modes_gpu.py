"""Modes of torch in which the digital operators would lose something without a word: forward-mode differentiation and tracing."""

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import adapters_case, rand

pytestmark = pytest.mark.gpu


def calls():
    """name, function of the tensors by their names, those tensors."""
    x, base, a, b, scale, ids, starts, _ = adapters_case(90, 4, 2, 64, 64, 8, torch.float32, 3)
    w, bias = rand((64,), torch.float32, 6), rand((64,), torch.float32, 7)
    return [
        ("dropout", lambda x, residual: digital.dropout(x, 0.3, 1, 2, residual), dict(x=x, residual=base)),
        ("layer_norm", lambda x, weight, bias: digital.layer_norm(x, weight, bias), dict(x=x, weight=w, bias=bias)),
        ("add_layer_norm", lambda x, residual, weight, bias: digital.add_layer_norm(x, residual, weight, bias, p=0.3),
         dict(x=x, residual=base, weight=w, bias=bias)),
        ("low_rank_add", lambda base, x, a, b, scale: digital.low_rank_add(base, x, a, b, scale, ids, starts),
         dict(base=base, x=x, a=a, b=b, scale=scale))]


@pytest.mark.parametrize("no_grad", [False, True], ids=["grad", "no_grad"])
def test_forward_mode_is_refused(no_grad):
    """A result without its tangent would read as a derivative of zero."""
    import torch.autograd.forward_ad as ad

    for _, fn, tensors in calls():
        for name, t in tensors.items():
            with ad.dual_level(), torch.set_grad_enabled(not no_grad):
                dual = ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(**{**tensors, name: dual})
                with ad._set_fwd_grad_enabled(False):  # tangents are not wanted here
                    fn(**{**tensors, name: dual})
            with pytest.raises(RuntimeError):
                torch.func.jvp(lambda v: fn(**{**tensors, name: v}), (t,), (torch.ones_like(t),))
        fn(**tensors)


def test_forward_mode_of_the_result_in_place_is_refused():
    import torch.autograd.forward_ad as ad

    x, base, a, b, scale, ids, starts, _ = adapters_case(90, 4, 2, 64, 64, 8, torch.float32, 3)
    with torch.no_grad(), ad.dual_level():
        out = ad.make_dual(base.clone(), torch.ones_like(base))
        with pytest.raises(RuntimeError, match="forward-mode"):
            digital.low_rank_add(base, x, a, b, scale, ids, starts, out=out)


def test_tracing_is_refused():
    """A trace would hold the allocation of the result and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    for _, fn, tensors in calls():
        first, *others = tensors.values()
        of_tensors = lambda *v: fn(**dict(zip(tensors, v)))
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(of_tensors, tuple(tensors.values()), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(of_tensors)(*tensors.values())
