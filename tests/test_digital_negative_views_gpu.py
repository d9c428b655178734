"""Views whose sign torch keeps apart from their memory: the imaginary part of a conjugated tensor.  Of one column they need no
copy to be read as rows."""

import pytest
import torch

from aihwkit_b200 import digital

pytestmark = pytest.mark.gpu


def negative(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    view = torch.view_as_complex(torch.randn(*shape, 2, device="cuda", generator=g)).conj().imag
    assert view.is_neg()
    return view


@pytest.mark.parametrize("cols", [1, 6])
def test_inputs_and_gradients(cols):
    x, res, gy = (negative((5, cols), s) for s in (1, 2, 3))
    w, b = negative((cols,), 4), negative((cols,), 5)
    plain = lambda t: t.clone().resolve_neg()
    assert torch.equal(digital.dropout(x, 0.3, 1, 2, residual=res), digital.dropout(plain(x), 0.3, 1, 2, residual=plain(res)))
    for got, want in zip(digital.add_layer_norm(x, res, w, b), digital.add_layer_norm(plain(x), plain(res), plain(w), plain(b))):
        assert torch.equal(got, want)
    for fn in (lambda t: digital.dropout(t, 0.3, 1, 2), lambda t: digital.layer_norm(t, plain(w), plain(b))):
        leaf = plain(x).requires_grad_()
        got, = torch.autograd.grad(fn(leaf), leaf, gy)
        want, = torch.autograd.grad(fn(leaf), leaf, plain(gy))
        assert torch.equal(got, want)


def test_low_rank_adapters():
    x, base = negative((5, 1), 1), negative((5, 1), 2)
    a, b, scale = torch.randn(2, 3, 1, device="cuda"), torch.randn(2, 3, 1, device="cuda"), torch.ones(2, device="cuda")
    ids = torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32, device="cuda")
    plain = lambda t: t.clone().resolve_neg()
    want = digital.low_rank_add(plain(base), plain(x), a, b, scale, ids)
    assert torch.equal(digital.low_rank_add(base, x, a, b, scale, ids), want)
    one = negative((1, 1, 1), 3)
    for call in (lambda: digital.low_rank_add(base, x, a, b, scale, ids, out=negative((5, 1), 4)),
                 lambda: digital.low_rank_add(base, x, one, one.clone().resolve_neg(), scale[:1], ids),
                 lambda: digital.low_rank_add(base, x, one.clone().resolve_neg(), one, scale[:1], ids),
                 lambda: digital.low_rank_add(base, x, a[:1], b[:1], negative((1,), 5), ids)):
        with pytest.raises(RuntimeError):
            call()
