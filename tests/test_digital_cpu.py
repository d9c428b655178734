"""Refusals of the digital operators that need no device: the C entry points check sizes, types and missing pointers before
they touch CUDA, and the Python calls refuse host tensors."""

import ctypes as C

import pytest
import torch

from aihwkit_b200 import _cabi, digital

P = 4096  # an address that no refused call looks at


def refused(name, args, match):
    lib = _cabi.lib()
    assert getattr(lib, name)(*args) != 0
    assert match in lib.ab200_last_error().decode()


def dropout_args(**kw):
    d = dict(x=P, xs=8, r=None, rs=0, y=P, ys=8, rows=1, cols=8, dtype=0, p=0.1, seed=0, call=0, stream=None)
    d.update(kw)
    return list(d.values())


def norm_args(**kw):
    d = dict(x=P, xs=8, r=None, rs=0, w=None, b=None, y=P, ys=8, h=None, hs=0, mean=None, rstd=None, rows=1, cols=8, dtype=0,
             pdtype=0, eps=1e-5, p=0.0, seed=0, call=0, stream=None)
    d.update(kw)
    return list(d.values())


def norm_grad_args(**kw):
    d = dict(gy=P, gs=8, gh=None, ghs=0, x=P, xs=8, r=None, rs=0, w=None, mean=P, rstd=P, dh=P, dhs=8, dx=None, dxs=0, dw=None, db=None,
             work=None, rows=1, cols=8, dtype=0, pdtype=0, p=0.0, seed=0, call=0, stream=None)
    d.update(kw)
    return list(d.values())


def low_rank_args(**kw):
    d = dict(x=P, xs=8, base=None, bs=0, y=P, ys=8, a=P, b=P, scale=P, ids=P, starts=None, n_req=1, rows=1, k=8, n=8, rank=4,
             adapters=1, dtype=0, v=None, stream=None)
    d.update(kw)
    return list(d.values())


def grad_args(**kw):
    d = dict(x=P, xs=8, u=P, da=P, k=8, gy=P, gs=8, v=P, db=P, n=8, ids=P, starts=None, n_req=1, rows=1, rank=4, adapters=1,
             dtype=0, work=P, stream=None)
    d.update(kw)
    return list(d.values())


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=3), "unknown element type"), (dict(rows=-1), "number of rows"), (dict(rows=1 << 31), "number of rows"),
    (dict(cols=0), "1 to"), (dict(x=None), "x is null"), (dict(y=None), "y is null"), (dict(p=-0.1), "probability"),
    (dict(p=1.5), "probability"), (dict(p=float("nan")), "probability"), (dict(xs=-8), "strides"), (dict(rs=-1), "strides"),
    (dict(rows=2, ys=7), "at least its row"), (dict(rows=2, ys=0), "at least its row")])
def test_dropout_refuses(kw, match):
    refused("ab200_dropout", dropout_args(**kw), match)


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=-1), "unknown element type"), (dict(pdtype=7), "unknown element type"), (dict(cols=16385), "1 to 16384"),
    (dict(cols=0), "1 to 16384"), (dict(rows=-1), "number of rows"), (dict(x=None), "x is null"), (dict(y=None), "y is null"),
    (dict(mean=P), "together"), (dict(p=2.0), "probability"), (dict(xs=-1), "strides"), (dict(rows=3, ys=4), "at least its row"),
    (dict(rows=3, h=P, hs=4), "at least its row")])
def test_layer_norm_refuses(kw, match):
    refused("ab200_layer_norm_forward", norm_args(**kw), match)


@pytest.mark.parametrize("kw, match", [
    (dict(gy=None), "gy is null"), (dict(x=None), "x is null"), (dict(mean=None), "mean is null"),
    (dict(rstd=None), "rstd is null"), (dict(dw=P), "workspace is null"), (dict(cols=20000), "1 to 16384"),
    (dict(dtype=9), "unknown element type"), (dict(gs=-8), "strides"), (dict(rows=2, dhs=1), "at least its row")])
def test_layer_norm_backward_refuses(kw, match):
    refused("ab200_layer_norm_backward", norm_grad_args(**kw), match)


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=3), "unknown element type"), (dict(n_req=2), "one request per row"), (dict(n_req=-1), "number of requests"),
    (dict(ids=None), "adapter_ids is null"), (dict(rank=0), "rank"), (dict(rank=257), "rank"), (dict(adapters=0), "adapters"),
    (dict(adapters=70000), "adapters"), (dict(k=0), "elements"), (dict(n=0), "elements"), (dict(x=None), "x is null"),
    (dict(a=None), "a is null"), (dict(b=None), "b is null"), (dict(scale=None), "scale is null"), (dict(y=None), "neither"),
    (dict(base=P, bs=16), "row stride"), (dict(xs=-1), "strides"),
    (dict(rows=2, n_req=2, ys=7), "at least its row"), (dict(rows=-1, n_req=-1), "number of")])
def test_low_rank_refuses(kw, match):
    refused("ab200_low_rank_apply", low_rank_args(**kw), match)


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=3), "unknown element type"), (dict(rank=300), "rank"), (dict(k=0), "elements"), (dict(gy=None), "gy is null"),
    (dict(u=None), "u is null"), (dict(v=None), "v is null"), (dict(work=None), "workspace is null"),
    (dict(n_req=3), "one request per row"), (dict(gs=-2), "strides")])
def test_low_rank_grad_refuses(kw, match):
    refused("ab200_low_rank_grad", grad_args(**kw), match)


def test_empty_calls_return_at_once():
    """No rows: nothing is launched, so the calls succeed without a device."""
    lib = _cabi.lib()
    assert lib.ab200_dropout(*dropout_args(rows=0, x=None, y=None)) == 0
    assert lib.ab200_layer_norm_forward(*norm_args(rows=0, x=None, y=None)) == 0
    assert lib.ab200_layer_norm_backward(*norm_grad_args(rows=0)) == 0
    assert lib.ab200_low_rank_apply(*low_rank_args(rows=0, n_req=0, x=None, y=None, ids=None)) == 0
    floats, size = C.c_longlong(7), C.c_longlong(7)
    assert lib.ab200_layer_norm_workspace(0, 8, C.byref(floats)) == 0 and floats.value == 0
    assert lib.ab200_low_rank_grad_workspace(0, 0, 0, 8, 8, 4, C.byref(size)) == 0 and size.value == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    ids = torch.zeros(2, dtype=torch.int32)
    for fn in (lambda: digital.dropout(x), lambda: digital.layer_norm(x), lambda: digital.add_layer_norm(x, x),
               lambda: digital.low_rank_add(x, x, torch.zeros(1, 2, 8), torch.zeros(1, 2, 8), torch.ones(1), ids)):
        with pytest.raises(RuntimeError, match="no CPU compute path"):
            fn()
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        digital.layer_norm(x.double())


def test_pool_of_adapters_on_the_host():
    """Layout and bounds of the pool; the products need a device."""
    pool = digital.LowRankAdapters(3, 10, 6, 4, device="cpu", generator=torch.Generator().manual_seed(1))
    assert pool.a.shape == (3, 4, 10) and pool.b.shape == (3, 4, 6) and not pool.b.any()
    a, b = torch.randn(2, 10), torch.randn(6, 2)
    pool.set_adapter(1, a, b, 0.5)
    assert torch.equal(pool.b[1].t() @ pool.a[1], b @ a) and pool.scale.tolist() == [1.0, 0.5, 1.0]
    for bad in (lambda: pool.set_adapter(3, a, b), lambda: pool.set_adapter(-1, a, b), lambda: pool.set_adapter(0, a, b.t()),
                lambda: pool.set_adapter(0, torch.zeros(5, 10), torch.zeros(6, 5)),
                lambda: digital.LowRankAdapters(1, 8, 8, 257, device="cpu"),
                lambda: digital.LowRankAdapters(0, 8, 8, 4, device="cpu"),
                lambda: digital.LowRankAdapters(1, 8, 8, 4, device="cpu", dtype=torch.float64)):
        with pytest.raises(RuntimeError):
            bad()
