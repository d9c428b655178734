"""The norm's backward pass on long 16-bit rows, which fetches rows ahead into shared memory: every number of tensors that it
can read (gy and x; with the residual; with the gradient of h; both), at widths on both sides of its shapes, several rows to a
block.  Bounds as in test_digital_gpu: F = 2^-24 an fp32 rounding, sums at most 68 additions deep, one rounding of the result
at the end."""

import os
import subprocess
import sys

import pytest
import torch

from aihwkit_b200 import digital
from tests.test_digital_gpu import F, IDS, TYPES, kept, norm_case, norm_exact, rand, unit, within

pytestmark = pytest.mark.gpu

CASES = [  # columns, with a residual, results that have a gradient
    (3080, False, "y"), (4096, False, "y"), (5640, False, "y"), (6144, False, "y"), (8192, False, "y"), (8200, False, "y"),
    (3592, True, "y"), (4096, True, "y"), (6144, True, "y"), (8192, True, "y"), (4096, True, "yh"), (8192, True, "yh")]


@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("cols, residual, results", CASES)
def test_gradients_on_long_rows(cols, residual, results, dtype):
    rows, p = 700, 0.1 if residual else 0.0
    x, res, w, b = norm_case(rows, cols, dtype, residual, p)
    leaves = [t.requires_grad_() for t in (x, res, w, b) if t is not None]
    out = digital.add_layer_norm(*leaves, p=p, seed=7, call=5) if residual else (digital.layer_norm(*leaves),)
    gy, gh = rand((rows, cols), dtype, 8), rand((rows, cols), dtype, 9)
    grads = torch.autograd.grad(out[:len(results)], leaves, [gy, gh][:len(results)])
    with torch.no_grad():
        keep = kept(rows, cols, p, 7, 5) if p > 0 else None
        d, xhat, rstd, _, _, e, w64 = norm_exact(x, res, w, b, 1e-5, keep, p)
        g = gy.double()
        t = g * w64
        m1, m2 = t.mean(1, keepdim=True), (t * xhat).mean(1, keepdim=True)
        dh = rstd * (t - m1 - xhat * m2)
        off = rstd * (m2.abs() * e + xhat.abs() * ((t.abs() * e).mean(1, keepdim=True) + 68 * F * (t * xhat).abs().mean(1, keepdim=True))
                      + 68 * F * t.abs().mean(1, keepdim=True) + 8 * F * (t.abs() + (xhat * m2).abs())) + 160 * F * dh.abs()
        if len(results) == 2:
            dh = dh + gh.double()
            off = off + 2 * F * dh.abs()
        scale = 1.0 if keep is None else keep.double() / (1 - p)
        u = unit(dtype)
        within(grads[0], dh * scale, u * (dh * scale).abs() + (off + 3 * F * dh.abs()) * scale, "dx")
        if residual:
            within(grads[1], dh, u * dh.abs() + off, "dresidual")
        dw, db = (g * xhat).sum(0), g.sum(0)
        within(grads[-2], dw, (g.abs() * e).sum(0) + 68 * F * (g * xhat).abs().sum(0) + F * dw.abs(), "dweight")
        within(grads[-1], db, 68 * F * g.abs().sum(0) + F * db.abs(), "dbias")


@pytest.mark.parametrize("case", ["6144-False-y-f16", "6144-False-y-bf16", "4096-True-y-f16", "4096-True-y-bf16"])
def test_first_call_of_a_process(case):
    """These take 48 KB of rows ahead, and a launch may not rest on an earlier one having asked for more."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-p", "no:cacheprovider",
                          f"{__file__}::test_gradients_on_long_rows[{case}]"], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "1 passed" in run.stdout, run.stdout[-2000:] + run.stderr[-500:]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("residual", [False, True], ids=["norm", "sum"])
@pytest.mark.parametrize("which", ["weight", "bias"])
def test_gradient_with_one_of_the_parameters(which, residual, dtype):
    """The missing one counts as 1 or 0: the others' gradients are those of a call that names it."""
    rows, cols = 40, 300
    x, res, w, b = norm_case(rows, cols, dtype, residual, 0.0)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    gy = rand((rows, cols), dtype, 8)

    def grads(weight, bias, wanted):
        front = [t.detach().requires_grad_() for t in (x, res) if t is not None]
        params = [None if t is None else t.detach().requires_grad_() for t in (weight, bias)]
        y = digital.add_layer_norm(*front, *params)[0] if residual else digital.layer_norm(*front, *params)
        return torch.autograd.grad(y, front + [params[wanted]], gy)

    i = ("weight", "bias").index(which)
    got = grads(w if i == 0 else None, b if i == 1 else None, i)
    want = grads(w if i == 0 else one, b if i == 1 else zero, i)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
