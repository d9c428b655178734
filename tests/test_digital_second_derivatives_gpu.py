"""The digital operators' gradients inside a recorded backward pass: what they are tied to, and the callers' tensors afterwards."""

import itertools

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import adapters_case, rand

pytestmark = pytest.mark.gpu

NAMES = ("x", "a", "b")


@pytest.mark.parametrize("graded, probed", list(itertools.permutations(NAMES, 2)))
@pytest.mark.parametrize("others", [False, True], ids=["alone", "all"])
def test_low_rank_gradients_are_not_differentiable_again(graded, probed, others):
    """dx = scale gy b^T a, da = scale (gy b^T)^T x and db = scale (x a^T)^T gy: each depends on two of x, a and b, whether or not
    the third has a gradient.  A loss that is linear in y leaves gy without a history."""
    x, base, a, b, scale, ids, starts, _ = adapters_case(90, 4, 2, 64, 96, 8, torch.float32, 5)
    t = dict(x=x, a=a, b=b)
    for name in NAMES if others else (graded, probed):
        t[name].requires_grad_()
    y = digital.low_rank_add(base, t["x"], t["a"], t["b"], scale, ids, starts)
    g, = torch.autograd.grad(y.sum(), [t[graded]], create_graph=True)
    loss = (g * g).sum() + (t[probed] * t[probed]).sum()
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(loss, [t[probed]])


def test_norm_gradients_are_not_differentiable_again():
    x, res = rand((6, 64), torch.float32, 1), rand((6, 64), torch.float32, 2)
    w, b = rand((64,), torch.float32, 3), rand((64,), torch.float32, 4)
    for dtype in (torch.float32, torch.bfloat16):
        for graded, probed in (("x", "w"), ("x", "res"), ("res", "x"), ("res", "w"), ("w", "x"), ("w", "res"), ("x", "x")):
            t = dict(x=x.to(dtype), res=res.to(dtype), w=w.clone(), b=b.clone())
            for name in (graded, probed):
                t[name].requires_grad_()
            y, _ = digital.add_layer_norm(t["x"], t["res"], t["w"], t["b"], p=0.25, seed=1, call=2)
            g, = torch.autograd.grad(y.sum(), [t[graded]], create_graph=True)
            with pytest.raises(RuntimeError, match="not differentiable again"):
                torch.autograd.grad((g * g).sum() + (t[probed] * t[probed]).sum(), [t[probed]])


def test_gradients_without_a_history_carry_none():
    """What a gradient does not depend on is not tied to it: the bias takes no part in any, x none in dropout's."""
    x, w, b = (rand(s, torch.float32, i).requires_grad_() for i, s in ((1, (6, 64)), (2, (64,)), (3, (64,))))
    g, = torch.autograd.grad(digital.dropout(x, 0.3).sum(), [x], create_graph=True)
    again, = torch.autograd.grad(g.sum() * 0.0 + (x * x).sum() if g.requires_grad else (x * x).sum(), [x])
    assert not g.requires_grad and torch.equal(again, 2 * x)
    g, = torch.autograd.grad(digital.layer_norm(x.detach(), w, b).sum(), [b], create_graph=True)
    assert not g.requires_grad and (g == 6).all()


def test_callers_gradient_keeps_its_history():
    """The gradient of h alone passes through the sum: the tensor that the caller handed over comes back as it was."""
    for p in (0.0, 0.5):
        x, res = (rand((6, 64), torch.float32, i).requires_grad_() for i in (1, 2))
        _, h = digital.add_layer_norm(x, res, p=p, seed=3, call=4)
        gh = rand((6, 64), torch.float32, 5)
        dx, dres = torch.autograd.grad([h], [x, res], [gh], create_graph=True)
        assert not gh.requires_grad and gh.grad_fn is None
        assert torch.equal(dres, gh) and not dres.requires_grad and not dx.requires_grad
        gh.requires_grad_()
        _, h = digital.add_layer_norm(x, res, p=p, seed=3, call=4)
        dx, dres = torch.autograd.grad([h], [x, res], [gh], create_graph=True)
        assert gh.is_leaf and torch.equal(torch.autograd.grad(dres.sum(), [gh], retain_graph=True)[0], torch.ones_like(gh))
        if p > 0:
            with pytest.raises(RuntimeError, match="not differentiable again"):
                torch.autograd.grad(dx.sum(), [gh])
