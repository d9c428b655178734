"""Digital operators against the formulas in 64 bits.

Tolerances. U = eps / 2 of the result's type is the one rounding at the end; F = 2^-24 is a rounding of an fp32 operation.
Norm: a row's sums are 8 * spans + 5 + warps additions deep, at most 64, so mean and variance are off by 64 F of the sums of
absolute values; the root and the products add a few F more.  Adapters: a sum along k is split over at least 8 warps of
16-bit (4 of fp32) steps of 32 (16) elements, so an accumulator takes k / 64 additions and up to 24 joins after that; each
addition of the matrix unit may truncate, off by up to 2^-22 of the absolute sum with the alignment of its terms; products of
split fp32 factors leave out at most 2^-21.  Each bound below multiplies those by the sums of absolute values in 64 bits.
"""

import math

import numpy as np
import pytest
import torch

from aihwkit_b200 import digital

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rand(shape, dtype, seed, scale=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale + mean).to(dtype)


def within(got, want, bound, what):
    # the smallest normal of the type covers results that round to subnormals
    bound = bound + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    bad = off > bound
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.3g} of the bound"


# ---- dropout ---------------------------------------------------------------------------------------------------------


def philox(blocks, call, tag, seed):
    """Philox4x32-10 of 64-bit block numbers, as eight half-words per block."""
    m = np.uint64(0xFFFFFFFF)
    c = [blocks & m, blocks >> np.uint64(32), np.full_like(blocks, call), np.full_like(blocks, tag)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).astype("<u4").view("<u2").astype(np.int64)


def kept(rows, cols, p, seed, call, first_row=0):
    per = -(-cols // 8)
    blocks = np.arange(first_row * per, (first_row + rows) * per, dtype=np.uint64)
    word = (philox(blocks, call, 0xB0000000, seed) << 16) + philox(blocks, call, 0xB0000001, seed)
    return torch.from_numpy((word >= int(math.floor(p * 2.0 ** 32 + 0.5))).reshape(rows, per * 8)[:, :cols].copy()).cuda()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 7), (3, 8), (5, 33), (64, 256), (17, 257), (300, 785), (1000, 64)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.7331, 1.0])
def test_dropout_against_the_generator(rows, cols, p, dtype):
    x, res = rand((rows, cols), dtype, 1), rand((rows, cols), dtype, 2)
    seed, call = 0x1234567890ABCDEF, 4000000001
    keep = kept(rows, cols, p, seed, call)
    scale = 1.0 / (1.0 - p) if p < 1 else 0.0
    want = torch.where(keep, x.double() * scale, 0.0)
    y = digital.dropout(x, p, seed, call)
    within(y, want, want.abs() * (unit(dtype) + 3 * F), "y")
    assert torch.equal(y != 0, keep & (x != 0)), "another set of elements"
    both = want + res.double()
    yr = digital.dropout(x, p, seed, call, residual=res)
    within(yr, both, both.abs() * unit(dtype) + 4 * F * (want.abs() + both.abs()), "y with residual")


def test_dropout_threshold_uses_all_32_bits():
    """Probabilities between two multiples of 2^-16 differ where a high half-word ties: at 2^23 elements about 128 do."""
    rows, cols, seed = 2048, 4096, 99
    x = torch.ones(rows, cols, device="cuda")
    high = (philox(np.arange(rows * cols // 8, dtype=np.uint64), 5, 0xB0000000, seed) == 6000).sum()
    assert high > 50
    sums = []
    for p in (6000 / 65536, 6000.25 / 65536, 6000.5 / 65536, 6001 / 65536):
        y = digital.dropout(x, p, seed, 5)
        assert torch.equal(y != 0, kept(rows, cols, p, seed, 5))
        sums.append(int((y != 0).sum()))
    assert sums[0] > sums[1] > sums[2] > sums[3] and sums[0] - sums[3] == high


def test_dropout_rate_and_independence():
    x = torch.ones(4096, 4096, device="cuda")
    for p in (0.1, 0.5):
        a, b, c = (digital.dropout(x, p, s, k) != 0 for s, k in ((1, 0), (1, 1), (2, 0)))
        n = x.numel()
        sd = math.sqrt(p * (1 - p) * n)
        assert abs(int(a.sum()) - (1 - p) * n) < 6 * sd
        for other in (b, c):  # two draws agree as often as independent ones do
            q = (1 - p) ** 2 + p ** 2
            assert abs(int((a == other).sum()) - q * n) < 6 * math.sqrt(q * (1 - q) * n)


def test_dropout_of_non_finite_values_and_its_gradient():
    x = rand((33, 72), torch.float32, 3)
    keep = kept(33, 72, 0.4, 8, 2)
    x[~keep] = float("nan")
    x[~keep & (torch.arange(72, device="cuda") % 2 == 0)] = float("inf")
    y = digital.dropout(x, 0.4, 8, 2)
    assert torch.isfinite(y).all() and (y[~keep] == 0).all()
    x = rand((33, 72), torch.float32, 3).requires_grad_()
    res = rand((33, 72), torch.float32, 4).requires_grad_()
    gy = rand((33, 72), torch.float32, 5)
    dx, dres = torch.autograd.grad(digital.dropout(x, 0.4, 8, 2, residual=res), [x, res], gy)
    within(dx, torch.where(keep, gy.double() / 0.6, 0.0), gy.double().abs() / 0.6 * 3 * F, "dx")
    assert torch.equal(dres, gy)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_dropout_of_views(dtype):
    """Strided rows, a start between two aligned addresses, transposed and three-dimensional tensors draw the same
    elements as the compact ones."""
    big = rand((40, 3, 96), dtype, 6)
    for view in (big[:, 1], big[:, :, 5:69], big.transpose(0, 1), big.permute(2, 0, 1), big[::2, 1, 3:],
                 big[:1, :1].expand(40, 3, 96)):
        assert torch.equal(digital.dropout(view, 0.3, 1, 2), digital.dropout(view.contiguous(), 0.3, 1, 2))
        assert torch.equal(digital.dropout(view, 0.3, 1, 2, residual=view), digital.dropout(view.contiguous(), 0.3, 1, 2,
                                                                                             residual=view.contiguous()))


def test_dropout_behind_32_bit_offsets():
    """Rows whose offsets and element numbers pass 2^31 and 2^32."""
    rows, cols = (1 << 20) + 3, 4104
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    y = digital.dropout(x, 0.25, 11, 3)
    tail = kept(64, cols, 0.25, 11, 3, rows - 64)
    assert torch.equal(y[-64:] != 0, tail)
    wide = x[:, :4097]  # the way without wide accesses
    assert torch.equal(digital.dropout(wide, 0.25, 11, 3)[-64:] != 0, kept(64, 4097, 0.25, 11, 3, rows - 64))


# ---- layer norm ------------------------------------------------------------------------------------------------------


def norm_case(rows, cols, dtype, residual, p, seed=0, wdtype=torch.float32, loud=True):
    x = rand((rows, cols), dtype, seed + 1)
    res = rand((rows, cols), dtype, seed + 2, 2.0, 0.5) if residual else None
    if residual and loud:
        res[:, :: max(1, cols // 3)] *= 8
    w, b = rand((cols,), wdtype, seed + 3, 0.3, 1.0), rand((cols,), wdtype, seed + 4, 0.2)
    return x, res, w, b


def norm_exact(x, res, w, b, eps, keep, p):
    d = x.double()
    if keep is not None:
        d = torch.where(keep, d / (1 - p) if p < 1 else 0 * d, 0.0)
    parts = d.abs()
    if res is not None:
        parts = parts + res.double().abs()
        d = d + res.double()
    mean = d.mean(1, keepdim=True)
    rstd = ((d - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    xhat = (d - mean) * rstd
    w64 = torch.ones_like(d[0]) if w is None else w.double()
    b64 = torch.zeros_like(d[0]) if b is None else b.double()
    off_h = 4 * F * parts  # of the fp32 sum h
    off_x = rstd * (off_h + 64 * F * d.abs().mean(1, keepdim=True) + off_h.mean(1, keepdim=True)) + xhat.abs() * 160 * F
    return d, xhat, rstd, xhat * w64 + b64, off_h, off_x, w64


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, cols, residual, p", [
    (1, 1, False, 0.0), (1, 768, True, 0.0), (3, 7, True, 0.3), (9, 256, False, 0.0), (6, 257, True, 0.1), (130, 785, True, 0.2),
    (5, 1024, True, 0.0), (7, 1032, True, 0.25), (700, 64, False, 0.0), (33, 2304, False, 0.0), (4, 4096, True, 0.1),
    (2, 8192, True, 0.0), (3, 8200, True, 0.5), (2, 16384, False, 0.0), (2, 16383, True, 0.1), (2, 40, True, 1.0)])
def test_layer_norm_forward_and_backward(rows, cols, residual, p, dtype):
    eps = 1e-5
    x, res, w, b = norm_case(rows, cols, dtype, residual, p)
    keep = kept(rows, cols, p, 77, 5) if p > 0 else None
    leaves = [t.requires_grad_() for t in (x, res, w, b) if t is not None]
    if residual:
        y, h = digital.add_layer_norm(x, res, w, b, eps, p=p, seed=77, call=5)
    else:
        y, h = digital.layer_norm(x, w, b, eps), None
    x, res, w, b = (None if t is None else t.detach() for t in (x, res, w, b))
    d, xhat, rstd, want, off_h, off_x, w64 = norm_exact(x, res, w, b, eps, keep, p)
    u = unit(dtype)
    within(y, want, u * want.abs() + w64.abs() * off_x + 4 * F * (want.abs() + (xhat * w64).abs()), "y")
    if residual:
        within(h, d, u * d.abs() + off_h, "h")
    gy = rand((rows, cols), dtype, 8)
    gh = rand((rows, cols), dtype, 9) if residual else None
    grads = torch.autograd.grad([y, h] if residual else [y], leaves, [gy, gh] if residual else [gy])
    g = gy.double()
    t = g * w64
    m1, m2 = t.mean(1, keepdim=True), (t * xhat).mean(1, keepdim=True)
    dh = rstd * (t - m1 - xhat * m2)
    e = off_x  # the backward pass sums h again: nothing is lost to the rounding of the stored one
    off = rstd * (m2.abs() * e + xhat.abs() * ((t.abs() * e).mean(1, keepdim=True) + 68 * F * (t * xhat).abs().mean(1, keepdim=True))
                  + 68 * F * t.abs().mean(1, keepdim=True) + 8 * F * (t.abs() + (xhat * m2).abs())) + 160 * F * dh.abs()
    if residual:
        dh = dh + gh.double()
        off = off + 2 * F * dh.abs()
        within(grads[1], dh, u * dh.abs() + off, "dresidual")
    scale = 1.0 if keep is None else torch.where(keep, 1 / (1 - p) if p < 1 else 0.0, 0.0).double()
    dx = dh * scale
    within(grads[0], dx, u * dx.abs() + (off + 3 * F * dh.abs()) * scale, "dx")
    depth = 64 + rows / 256
    dw, db = (g * xhat).sum(0), g.sum(0)
    within(grads[-2], dw, (g.abs() * e).sum(0) + depth * F * (g * xhat).abs().sum(0) + unit(w.dtype) * dw.abs(), "dweight")
    within(grads[-1], db, depth * F * g.abs().sum(0) + unit(b.dtype) * db.abs(), "dbias")
    # without gradients: the same bits
    with torch.no_grad():
        again = digital.add_layer_norm(x, res, w, b, eps, p=p, seed=77, call=5) if residual else (digital.layer_norm(x, w, b, eps),)
        assert torch.equal(again[0], y) and (not residual or torch.equal(again[1], h))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS[1:])
def test_layer_norm_parameters_of_the_input_type(dtype):
    x, _, w, b = norm_case(50, 96, dtype, False, 0.0, wdtype=dtype)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = digital.layer_norm(x, w, b)
    gy = rand((50, 96), dtype, 5)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], gy)
    assert dw.dtype == db.dtype == dtype
    _, xhat, _, want, _, off_x, w64 = norm_exact(x.detach(), None, w.detach(), b.detach(), 1e-5, None, 0)
    within(y, want, unit(dtype) * want.abs() + w64.abs() * off_x + 4 * F * (want.abs() + (xhat * w64).abs()), "y")
    g = gy.double()
    within(dw, (g * xhat).sum(0), (unit(dtype) * (g * xhat).sum(0)).abs() + (g.abs() * off_x).sum(0)
           + 65 * F * (g * xhat).abs().sum(0), "dweight")
    within(db, g.sum(0), (unit(dtype) * g.sum(0)).abs() + 65 * F * g.abs().sum(0), "dbias")


def test_layer_norm_special_rows():
    """Constant rows (variance 0), a large offset, no parameters, one row of NaN among others, no rows at all."""
    x = torch.full((4, 512), 3.25, device="cuda")
    x[1] = 1e4 + rand((512,), torch.float32, 1, 0.5)
    x[2, 100] = float("nan")
    y = digital.layer_norm(x)
    assert (y[0] == 0).all() and (y[3] == 0).all() and torch.isnan(y[2]).all()
    d = x[1].double()
    want = (d - d.mean()) / ((d - d.mean()).square().mean() + 1e-5).sqrt()
    # 64 F of the mean of |x| = 1e4 against a deviation of 0.5
    assert float((y[1].double() - want).abs().max()) <= 64 * F * 1e4 / 0.4 + 200 * F * float(want.abs().max())
    e = torch.empty(0, 512, device="cuda", requires_grad=True)
    w = torch.ones(512, device="cuda", requires_grad=True)
    out = digital.layer_norm(e, w)
    de, dw = torch.autograd.grad(out, [e, w], torch.empty(0, 512, device="cuda"))
    assert out.shape == de.shape == (0, 512) and (dw == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_layer_norm_of_views(dtype):
    big = rand((20, 3, 1024), dtype, 6)
    w, b = rand((1024,), torch.float32, 7), rand((1024,), torch.float32, 8)
    for view in (big[:, 1], big[:, :, 5:800], big.transpose(0, 1), big[::2, 1, 3:], big[0, 0], big[:1, :1].expand(20, 3, 1024)):
        n = view.size(-1)
        got = digital.add_layer_norm(view, view, w[:n], b[:n], p=0.2, seed=1, call=2)
        flat = view.contiguous()
        want = digital.add_layer_norm(flat, flat, w[:n].clone(), b[:n].clone(), p=0.2, seed=1, call=2)
        for q, r in zip(got, want):
            # another layout sums in another order
            assert torch.allclose(q.float(), r.float(), rtol=4 * unit(dtype) + 1e-5, atol=1e-5)


def test_layer_norm_sums_repeat_bit_for_bit():
    x, res, w, b = norm_case(5000, 768, torch.float32, True, 0.1)
    gy = rand((5000, 768), torch.float32, 3)
    outs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (x, res, w, b)]
        y, h = digital.add_layer_norm(*leaves, p=0.1, seed=3, call=4)
        outs.append(torch.autograd.grad([y], leaves, [gy]))
    for other in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], other))


def test_layer_norm_gradient_of_one_result_only():
    x, res, w, b = norm_case(6, 64, torch.float32, True, 0.1)
    leaves = [t.requires_grad_() for t in (x, res, w, b)]
    gh = rand((6, 64), torch.float32, 3)
    y, h = digital.add_layer_norm(*leaves, p=0.5, seed=3, call=4)
    dx, dres = torch.autograd.grad([h], leaves[:2], [gh])
    keep = kept(6, 64, 0.5, 3, 4)
    assert torch.equal(dres, gh) and torch.equal(dx, torch.where(keep, gh * 2, 0.0))
    y, h = digital.add_layer_norm(*leaves, p=0.0)
    dres, = torch.autograd.grad([y.sum() + (h * gh).sum()], [leaves[1]])
    assert torch.isfinite(dres).all()


def test_layer_norm_gradient_against_differences():
    """The gradient's dot with a direction against the difference of the forward pass in steps of 2^-6: the third derivative
    of a row's norm (deviation about 1) times step^2 is below 1e-2 of it, and the fp32 noise of the sums 1e-3."""
    x, res, w, b = norm_case(4, 96, torch.float32, True, 0.0, loud=False)
    leaves = [t.requires_grad_() for t in (x, res, w, b)]
    gy, gh = rand((4, 96), torch.float32, 20), rand((4, 96), torch.float32, 21)

    def f(*a):
        y, h = digital.add_layer_norm(*a, p=0.25, seed=5, call=6)
        return float((y.double() * gy.double()).sum() + (h.double() * gh.double()).sum())

    y, h = digital.add_layer_norm(*leaves, p=0.25, seed=5, call=6)
    grads = torch.autograd.grad([y, h], leaves, [gy, gh])
    with torch.no_grad():
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            way = rand(leaf.shape, torch.float32, 30 + i)
            s = 2.0 ** -6
            plus, minus = ([q + s * k * way if j == i else q for j, q in enumerate(leaves)] for k in (1, -1))
            slope = (f(*plus) - f(*minus)) / (2 * s)
            dot = float((grad.double() * way.double()).sum())
            size = float(grad.double().norm() * way.double().norm())
            assert abs(slope - dot) <= 1.1e-2 * size


# ---- low-rank adapters -----------------------------------------------------------------------------------------------


def adapters_case(rows, requests, adapters, k, n, rank, dtype, seed=0, ragged=True):
    rng = np.random.default_rng(seed)
    if ragged:
        starts = np.sort(rng.integers(rows // 20, rows - rows // 20 + 1, requests + 1))
        if requests > 2:
            starts[1] = starts[2]  # a request without rows
    else:
        starts = None
    ids = rng.integers(0, adapters, requests)
    if requests > 3:
        ids[requests // 2], ids[requests - 1] = -1, adapters + 3
    per_row = np.full(rows, -1)
    for j, i in enumerate(ids):
        s, e = (starts[j], starts[j + 1]) if ragged else (j, j + 1)
        per_row[s:e] = i if 0 <= i < adapters else -1
    x, base = rand((rows, k), dtype, seed + 1), rand((rows, n), dtype, seed + 2)
    a, b = rand((adapters, rank, k), dtype, seed + 3, k ** -0.5), rand((adapters, rank, n), dtype, seed + 4, rank ** -0.5)
    scale = torch.rand(adapters, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) + 0.5
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return x, base, a, b, scale, as_int(ids), None if starts is None else as_int(starts), torch.tensor(per_row, device="cuda")


def product(x, f, c):
    """x f^T in 64 bits and how far the kernel's sum of width c.. may be off."""
    return x @ f.t(), x.abs() @ f.abs().t()


def adapters_exact(x, base, a, b, scale, per_row):
    """y, its bound, v = scale x a^T and its bound, in 64 bits."""
    k, rank = a.size(2), a.size(1)
    split = 2.0 ** -21  # left out of a product of split fp32 factors
    step = 2.0 ** -22
    y, off = base.double().clone(), torch.zeros_like(base, dtype=torch.float64)
    v, v_off = torch.zeros(x.size(0), rank, dtype=torch.float64, device="cuda"), torch.zeros(x.size(0), rank, dtype=torch.float64, device="cuda")
    for i in range(a.size(0)):
        rows = (per_row == i).nonzero().flatten()
        ai, bi, s = a[i].double(), b[i].double(), float(scale[i])
        vi, mag = product(x[rows].double(), ai, k)
        vo = s * mag * ((k / 64 + 24) * step + split)
        vi = vi * s
        v[rows], v_off[rows] = vi, vo
        d = vi @ bi
        y[rows] += d
        off[rows] = vo @ bi.abs() + (vi.abs() @ bi.abs()) * ((rank + 8) * step + split) + 2 * F * (d.abs() + base[rows].double().abs())
    return y, off, v, v_off


SHAPES = [  # rows, requests, adapters, k, n, rank, ragged
    (1, 1, 1, 8, 8, 1, False), (1, 1, 4, 768, 2304, 8, False), (7, 7, 3, 33, 17, 3, False), (40, 40, 5, 256, 512, 16, False),
    (150, 150, 8, 96, 64, 64, False), (20, 2, 2, 64, 64, 8, True), (300, 4, 2, 128, 256, 16, True), (515, 9, 3, 785, 461, 5, True),
    (1100, 5, 2, 1024, 320, 32, True), (260, 6, 3, 200, 72, 33, True), (200, 3, 2, 512, 384, 64, True),
    (130, 5, 2, 160, 224, 100, True), (70, 4, 2, 96, 130, 256, True), (64, 70, 4, 64, 32, 4, True), (5000, 3, 2, 64, 48, 8, True)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, requests, adapters, k, n, rank, ragged", SHAPES)
def test_low_rank_forward_and_backward(rows, requests, adapters, k, n, rank, ragged, dtype):
    x, base, a, b, scale, ids, starts, per_row = adapters_case(rows, requests, adapters, k, n, rank, dtype, rows, ragged)
    y64, off, v, v_off = adapters_exact(x, base, a, b, scale, per_row)
    u = unit(dtype)
    y = digital.low_rank_add(base, x, a, b, scale, ids, starts)
    within(y, y64, u * y64.abs() + off, "y")
    none = per_row < 0
    assert torch.equal(y[none], base[none])
    inplace = base.clone()
    digital.low_rank_add(inplace, x, a, b, scale, ids, starts, out=inplace)
    assert torch.equal(inplace, y)
    gy = rand((rows, n), dtype, 50)
    leaves = [t.requires_grad_() for t in (base, x, a, b)]
    out = digital.low_rank_add(base, x, a, b, scale, ids, starts)
    assert torch.equal(out, y)
    dbase, dx, da, db = torch.autograd.grad(out, leaves, gy)
    assert torch.equal(dbase, gy)
    x, a, b = x.detach(), a.detach(), b.detach()
    dx64, dx_off, w, w_off = adapters_exact(gy, torch.zeros_like(x), b, a, scale, per_row)
    within(dx, dx64, u * dx64.abs() + dx_off, "dx")
    assert (dx[none] == 0).all()
    step, split = 2.0 ** -22, 2.0 ** -21
    for i in range(adapters):
        m = (per_row == i).nonzero().flatten()
        for got, left, left_off, right, what in ((da, w, w_off, x, "da"), (db, v, v_off, gy, "db")):
            l, r = left[m], right[m].double()
            want = l.t() @ r
            count = 3 * len(m) / 8 + requests + 16
            bound = left_off[m].t() @ r.abs() + (l.abs().t() @ r.abs()) * (count * step + split)
            within(got[i], want, u * want.abs() + bound, what)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_low_rank_rows_without_an_adapter_are_left_alone(dtype):
    """NaN and infinities in rows of no request, or of one without an adapter, stay where they are: in place nothing is
    written there, and no gradient of an adapter sees them."""
    x, base, a, b, scale, ids, starts, per_row = adapters_case(200, 5, 2, 96, 128, 8, dtype, 3)
    none = per_row < 0
    assert none.any() and (~none).any()
    clean = digital.low_rank_add(base, x, a, b, scale, ids, starts)
    gy = rand((200, 128), dtype, 9)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(digital.low_rank_add(base, *leaves, scale, ids, starts), leaves, gy)
    x2, base2, gy2 = x.clone(), base.clone(), gy.clone()
    x2[none], base2[none], gy2[none] = float("nan"), float("-inf"), float("inf")
    y2 = digital.low_rank_add(base2, x2, a, b, scale, ids, starts)
    assert torch.equal(y2[~none], clean[~none]) and (y2[none] == float("-inf")).all()
    leaves = [t.clone().requires_grad_() for t in (x2, a, b)]
    other = torch.autograd.grad(digital.low_rank_add(base2, *leaves, scale, ids, starts), leaves, gy2)
    for p, q in zip(grads, other):
        assert torch.equal(p, q)


def test_low_rank_bad_tables_stay_in_bounds():
    """Borders that run backwards or past the rows and ids past the adapters: the call ends, nothing outside the buffers is
    touched, and rows that no tile covers keep what they held."""
    rows, k, n = 100, 64, 96
    x, base, a, b, scale, _, _, _ = adapters_case(rows, 4, 2, k, n, 8, torch.float32, 3)
    guard = torch.full((rows + 64, n), 7.0, device="cuda")
    for starts in ([0, 500, 20, 1 << 30, 90], [-7, -3, 50, 40, 30], [90, 60, 30, 10, 0], [2 ** 31 - 1] * 5, [-2 ** 31] * 5):
        s = torch.tensor(starts, dtype=torch.int32, device="cuda")
        for ids in ([0, 1, 0, 1], [5, -1, 2 ** 31 - 1, -2 ** 31]):
            i = torch.tensor(ids, dtype=torch.int32, device="cuda")
            guard.fill_(7.0)
            out = guard[32:32 + rows]
            out.copy_(base)
            digital.low_rank_add(out, x, a, b, scale, i, s, out=out)
            assert (guard[:32] == 7.0).all() and (guard[32 + rows:] == 7.0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_low_rank_views_and_layouts(dtype):
    x3, base3 = rand((6, 50, 160), dtype, 1), rand((6, 50, 192), dtype, 2)
    a, b = rand((3, 16, 96), dtype, 3, 0.1), rand((3, 16, 128), dtype, 4, 0.25)
    scale = torch.ones(3, device="cuda")
    ids = torch.tensor([2, -1, 1, 0], dtype=torch.int32, device="cuda")
    starts = torch.tensor([3, 60, 90, 200, 290], dtype=torch.int32, device="cuda")
    for xs, bs in (((0, 96), (0, 128)), ((32, 128), (64, 192)), ((1, 97), (3, 131)), ((8, 104), (8, 136))):
        x, base = x3[:, :, xs[0]:xs[1]], base3[:, :, bs[0]:bs[1]]
        want = digital.low_rank_add(base.contiguous(), x.contiguous(), a, b, scale, ids, starts)
        got = digital.low_rank_add(base, x, a, b, scale, ids, starts)
        assert torch.equal(got, want)  # the same sums, whatever way the elements came
        held = base3.clone()
        part = held[:, :, bs[0]:bs[1]]
        digital.low_rank_add(part, x, a, b, scale, ids, starts, out=part)
        assert torch.equal(part, want)
        part.copy_(base)
        assert torch.equal(held, base3)
    # one row for all
    got = digital.low_rank_add(base3[:, :, :128], x3[:1, :1, :96].expand(6, 50, 96), a, b, scale, ids, starts)
    want = digital.low_rank_add(base3[:, :, :128], x3[:1, :1, :96].expand(6, 50, 96).contiguous(), a, b, scale, ids, starts)
    assert torch.equal(got, want)


def test_low_rank_behind_32_bit_offsets():
    """Rows two gigabytes apart."""
    ld = (1 << 30) + 32
    store = torch.empty(4 * ld + 256, dtype=torch.bfloat16, device="cuda")
    x, base = store.as_strided((5, 64), (ld, 1)), store.as_strided((5, 96), (ld, 1), 128)
    x.copy_(rand((5, 64), torch.bfloat16, 1))
    base.copy_(rand((5, 96), torch.bfloat16, 2))
    a, b = rand((2, 8, 64), torch.bfloat16, 3), rand((2, 8, 96), torch.bfloat16, 4)
    scale = torch.ones(2, device="cuda")
    ids = torch.tensor([1, 0, -1, 1, 0], dtype=torch.int32, device="cuda")
    want = digital.low_rank_add(base.contiguous(), x.contiguous(), a, b, scale, ids)
    assert torch.equal(digital.low_rank_add(base, x, a, b, scale, ids), want)
    digital.low_rank_add(base, x, a, b, scale, ids, out=base)
    assert torch.equal(base, want)
    y, h = digital.add_layer_norm(x, x)
    y2, h2 = digital.add_layer_norm(x.contiguous(), x.contiguous())
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_low_rank_gradient_against_differences():
    """y is linear in each of base, x, a and b: the difference of two forward passes is the gradient up to their roundings."""
    x, base, a, b, scale, ids, starts, _ = adapters_case(90, 4, 2, 64, 96, 8, torch.float32, 5)
    gy = rand((90, 96), torch.float32, 1)
    leaves = [t.requires_grad_() for t in (base, x, a, b)]
    grads = torch.autograd.grad(digital.low_rank_add(*leaves, scale, ids, starts), leaves, gy)
    with torch.no_grad():
        for i, grad in enumerate(grads):
            way = rand(grad.shape, torch.float32, 10 + i)
            plus, minus = ([q + s * way if j == i else q for j, q in enumerate(leaves)] for s in (0.5, -0.5))
            slope = sum(s * float((digital.low_rank_add(*q, scale, ids, starts).double() * gy.double()).sum())
                        for s, q in ((1, plus), (-1, minus)))
            dot = float((grad.double() * way.double()).sum())
            assert abs(slope - dot) <= 1e-4 * float(grad.double().norm() * way.double().norm())


def test_low_rank_gradients_repeat_and_stand_alone():
    """The same bits every time, and for each gradient asked for by itself."""
    x, base, a, b, scale, ids, starts, _ = adapters_case(3000, 6, 2, 256, 320, 16, torch.bfloat16, 5)
    gy = rand((3000, 320), torch.bfloat16, 1)
    full = None
    for want in (("x", "a", "b"), ("x", "a", "b"), ("x",), ("a",), ("b",)):
        t = {"x": x.clone(), "a": a.clone(), "b": b.clone()}
        for name in want:
            t[name].requires_grad_()
        y = digital.low_rank_add(base, t["x"], t["a"], t["b"], scale, ids, starts)
        grads = dict(zip(want, torch.autograd.grad(y, [t[q] for q in want], gy)))
        if full is None:
            full = grads
        if len(want) == 3 or want == ("x",):
            assert all(torch.equal(grads[q], full[q]) for q in want)
        else:  # fewer gradients are cut into other chunks
            u = unit(torch.bfloat16)
            assert all(torch.allclose(grads[q].float(), full[q].float(), rtol=2 * u, atol=1e-3) for q in want)


def test_low_rank_empty_inputs():
    a, b, scale = rand((2, 4, 32), torch.float32, 1), rand((2, 4, 64), torch.float32, 2), torch.ones(2, device="cuda")
    x, base = torch.empty(0, 32, device="cuda"), torch.empty(0, 64, device="cuda")
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    assert digital.low_rank_add(base, x, a, b, scale, ids).shape == (0, 64)
    a.requires_grad_(), b.requires_grad_()
    for starts in (None, torch.zeros(1, dtype=torch.int32, device="cuda")):
        y = digital.low_rank_add(base, x, a, b, scale, ids, starts)
        da, db = torch.autograd.grad(y, [a, b], torch.empty(0, 64, device="cuda"))
        assert (da == 0).all() and (db == 0).all()
    x, base = rand((5, 32), torch.float32, 1), rand((5, 64), torch.float32, 2)
    starts = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = digital.low_rank_add(base, x, a, b, scale, ids, starts)  # rows, but no request
    assert torch.equal(y, base)
    da, db = torch.autograd.grad(y, [a, b], torch.ones(5, 64, device="cuda"))
    assert (da == 0).all() and (db == 0).all()


# ---- streams, graphs, refusals ---------------------------------------------------------------------------------------


def test_another_stream():
    x, res, w, b = norm_case(2000, 768, torch.float32, True, 0.1)
    c = adapters_case(2000, 6, 2, 768, 512, 8, torch.float32, 5)
    want = digital.add_layer_norm(x, res, w, b, p=0.1, seed=1, call=1)
    want_a = digital.low_rank_add(c[1], c[0], *c[2:7])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [torch.empty_like(t) for t in (x, res)]
        for _ in range(20):  # work that the calls have to wait for in stream order
            for t, s in zip(late, (x, res)):
                t.copy_(s * 1.0)
        got = digital.add_layer_norm(late[0], late[1], w, b, p=0.1, seed=1, call=1)
        got_a = digital.low_rank_add(c[1] + 0, c[0] + 0, *c[2:7])
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(got_a, want_a)


def test_captured_step_replays_on_new_inputs():
    """Forward and backward of the three operators in one graph, replayed on other contents."""
    k, n, rows = 128, 128, 320
    x, base, a, b, scale, ids, starts, _ = adapters_case(rows, 5, 2, k, n, 8, torch.float32, 5)
    w, bias = rand((n,), torch.float32, 3, 0.2, 1.0), rand((n,), torch.float32, 4)
    gy = rand((rows, n), torch.float32, 6)
    leaves = [t.requires_grad_() for t in (x, a, b, w, bias)]

    def step():
        d = digital.dropout(leaves[0], 0.1, 1, 2)
        y = digital.low_rank_add(base, d, leaves[1], leaves[2], scale, ids, starts)
        y, h = digital.add_layer_norm(y, leaves[0], leaves[3], leaves[4], p=0.2, seed=1, call=3)
        return (y, h) + torch.autograd.grad([y, h], leaves, [gy, gy])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2):
        with torch.no_grad():
            for i, t in enumerate(leaves[:3] + [gy]):
                t.copy_(rand(t.shape, torch.float32, 100 * seed + i))
            ids.copy_(torch.roll(ids, 1))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_python_refusals():
    x, base = torch.zeros(4, 32, device="cuda"), torch.zeros(4, 64, device="cuda")
    a, b, scale = torch.zeros(2, 3, 32, device="cuda"), torch.zeros(2, 3, 64, device="cuda"), torch.ones(2, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    st = torch.zeros(5, dtype=torch.int32, device="cuda")
    add = digital.low_rank_add
    wide = torch.zeros(4, 128, device="cuda")
    for call in (
            lambda: add(base.half(), x, a, b, scale, ids), lambda: add(base, x, a.half(), b, scale, ids),
            lambda: add(base, x, a, b[:1], scale, ids), lambda: add(base, x, a, b, scale.half(), ids),
            lambda: add(base, x, a, b, scale[:1], ids), lambda: add(base, x, a, b, scale, ids.long()),
            lambda: add(base, x, a, b, scale, ids[:3]), lambda: add(base, x, a, b, scale, ids, st[:4]),
            lambda: add(base, x[:3], a, b, scale, ids), lambda: add(x, x, a, b, scale, ids),
            lambda: add(base, x, a.transpose(1, 2).contiguous().transpose(1, 2), b, scale, ids),
            lambda: add(base, x, a, b, scale, ids, out=x), lambda: add(base, x, a, b, scale, ids, out=base.half()),
            lambda: add(wide[:, :64], x, a, b, scale, ids, out=wide[:, 32:96]),
            lambda: add(base, wide[:, :32], a, b, scale, ids, out=wide[:, 16:80]),
            lambda: add(base, x, a, b, scale, ids, out=base[:1].expand(4, 64)),
            lambda: add(base, x, a.clone().requires_grad_(), b, scale, ids, out=base.clone()),
            lambda: add(base, x, a, b, scale.clone().requires_grad_(), ids),
            lambda: add(base, x, a[:0], b[:0], scale[:0], ids), lambda: add(base, x, a[:, :0], b[:, :0], scale, ids),
            lambda: add(base, x, torch.zeros(1, 257, 32, device="cuda"), torch.zeros(1, 257, 64, device="cuda"), scale[:1], ids),
            lambda: digital.dropout(x, 1.5), lambda: digital.dropout(x, 0.5, -1), lambda: digital.dropout(x, 0.5, 0, 1 << 32),
            lambda: digital.dropout(x, 0.5, residual=base), lambda: digital.dropout(x.int()),
            lambda: digital.dropout(x[0, 0]), lambda: digital.layer_norm(x, scale), lambda: digital.layer_norm(x, x[0].half()),
            lambda: digital.layer_norm(x, x[0], x[0].cpu()), lambda: digital.add_layer_norm(x, base),
            lambda: digital.add_layer_norm(x, None), lambda: digital.add_layer_norm(x, x.half()),
            lambda: digital.layer_norm(torch.zeros(2, 16385, device="cuda")), lambda: digital.layer_norm(x[:, :0]),
            lambda: digital.layer_norm(x.half(), x[0], x[0].half())):
        with pytest.raises(RuntimeError):
            call()
    assert (base == 0).all()


def test_beside_analog_tiles():
    """A layer on tiles, its adapters, and dropout, residual sum and norm behind it, forward and backward, against the same
    run of plain operations in 64 bits around the tiles' own results."""
    from aihwkit_b200.rpu_base import devices as D, tiles as T

    p = D.AnalogTileParameter()
    for io in (p.forward_io, p.backward_io):
        io.is_perfect = True
    p.update.pulse_type = D.PulseType.None_
    k, n, rows = 96, 96, 130
    arr = T.TileArray(p._config(64, 64, D.IdealResistiveDeviceParameter(), seed=1), n, k, 64, 64, cuda_device=0)
    arr.set_weights(torch.randn(n, k, generator=torch.Generator().manual_seed(0)) * 0.1)
    pool = digital.LowRankAdapters(2, k, n, 4, scale=0.5, generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        pool.b.copy_(rand(pool.b.shape, torch.float32, 4, 0.2))
    _, _, _, _, _, ids, starts, per_row = adapters_case(rows, 4, 2, k, n, 4, torch.float32, 7)
    x, res = rand((rows, k), torch.float32, 1).requires_grad_(), rand((rows, n), torch.float32, 2)
    w, b = (rand((n,), torch.float32, 5, 0.2, 1.0).requires_grad_(), rand((n,), torch.float32, 6).requires_grad_())
    base = arr.forward(x.detach())
    y, h = digital.add_layer_norm(pool(base, x, ids, starts), res, w, b, p=0.1, seed=1, call=2)
    gy = rand((rows, n), torch.float32, 8)
    leaves = [x, pool.a, pool.b, w, b]
    grads = torch.autograd.grad(y, leaves, gy)

    x64, a64, b64, w64, bias64 = (t.detach().double().requires_grad_() for t in leaves)
    keep = kept(rows, n, 0.1, 1, 2)
    delta = sum(torch.where((per_row == i)[:, None], 0.5 * (x64 @ a64[i].t()) @ b64[i], 0.0) for i in range(2))
    h64 = torch.where(keep, (base.double() + delta) / 0.9, 0.0) + res.double()
    y64 = torch.nn.functional.layer_norm(h64, (n,), w64, bias64)
    g64 = torch.autograd.grad(y64, [x64, a64, b64, w64, bias64], gy.double())
    # fp32 throughout: relative 2-norm errors of a few hundred roundings at most
    for got, want in [(y, y64), (h, h64)] + list(zip(grads, g64)):
        assert float((got.double() - want).norm()) <= 512 * F * float(want.norm())


# ---- further calls that the documentation allows ---------------------------------------------------------------------


def test_gradients_are_not_differentiable_again():
    x = rand((6, 64), torch.float32, 1).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    for y in (digital.layer_norm(x, w), digital.add_layer_norm(x, x * 2.0, w, p=0.1)[0], digital.dropout(x, 0.3)):
        g, = torch.autograd.grad((y * y).sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable again"):
            torch.autograd.grad(g.sum(), [x])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_low_rank_many_single_rows(dtype):
    """Single rows of few adapters share tiles within a neighbourhood of 1024 requests; longer requests between them, empty
    ones and rows without an adapter keep tiles of their own.  Each row's result is that of a call of its own."""
    rng = np.random.default_rng(5)
    lengths = rng.choice([0, 1, 1, 1, 1, 1, 1, 1, 2, 17], size=2300)
    starts = np.concatenate([[3], 3 + np.cumsum(lengths)])
    rows = int(starts[-1]) + 5
    ids = rng.integers(-1, 3, size=2300)
    per_row = np.full(rows, -1)
    for j in range(2300):
        per_row[starts[j]:starts[j + 1]] = ids[j]
    per_row = torch.tensor(per_row, device="cuda")
    x, base = rand((rows, 64), dtype, 1), rand((rows, 96), dtype, 2)
    a, b = rand((3, 8, 64), dtype, 3, 0.125), rand((3, 8, 96), dtype, 4, 0.35)
    scale = torch.tensor([0.5, 1.0, 2.0], device="cuda")
    ids_t, starts_t = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (ids, starts))
    y64, off, _, _ = adapters_exact(x, base, a, b, scale, per_row)
    y = digital.low_rank_add(base, x, a, b, scale, ids_t, starts_t)
    within(y, y64, unit(dtype) * y64.abs() + off, "y")
    assert torch.equal(y[per_row < 0], base[per_row < 0])
    one = digital.low_rank_add(base, x, a, b, scale, per_row.int())  # each row a request
    within(one, y64, unit(dtype) * y64.abs() + off, "one row each")
    leaves = [t.requires_grad_() for t in (a, b)]
    gy = rand((rows, 96), dtype, 9)
    da, db = torch.autograd.grad(digital.low_rank_add(base, x, a, b, scale, ids_t, starts_t), leaves, gy)
    for i in range(3):
        m = per_row == i
        u = float(scale[i]) * gy[m].double() @ b[i].detach().double().t()
        v = float(scale[i]) * x[m].double() @ a[i].detach().double().t()
        for got, l, r in ((da[i], u, x[m].double()), (db[i], v, gy[m].double())):
            want = l.t() @ r
            # two products and about 2300 sums in a row, 2^-17 of u or v at most beside them
            bound = unit(dtype) * want.abs() + (l.abs().t() @ r.abs()) * (2400 * 2.0 ** -22)
            within(got, want, bound, "gradient")


def test_layer_norm_backward_of_the_c_interface_on_long_fp32_rows():
    """fp32 callers of the C interface may hand over x and the residual as well as their sum."""
    import ctypes as C

    from aihwkit_b200 import _cabi

    lib = _cabi.lib()
    rows, p, seed, call = 5, 0.25, 3, 4
    for cols in (768, 4096, 8192, 16384):
        x, res, w, b = norm_case(rows, cols, torch.float32, True, p)
        gy, gh = rand((rows, cols), torch.float32, 8), rand((rows, cols), torch.float32, 9)
        leaves = [t.clone().requires_grad_() for t in (x, res, w, b)]
        want = torch.autograd.grad(digital.add_layer_norm(*leaves, p=p, seed=seed, call=call), leaves, [gy, gh])
        stats = torch.empty(2, rows, device="cuda")
        y, h = torch.empty_like(x), torch.empty_like(x)
        stream = torch.cuda.current_stream().cuda_stream
        ptr = lambda t: t.data_ptr()
        _cabi.check(lib.ab200_layer_norm_forward(ptr(x), cols, ptr(res), cols, ptr(w), ptr(b), ptr(y), cols, ptr(h), cols, ptr(stats),
                                                 ptr(stats) + 4 * rows, rows, cols, 0, 0, 1e-5, p, seed, call, stream))
        floats = C.c_longlong()
        _cabi.check(lib.ab200_layer_norm_workspace(rows, cols, C.byref(floats)))
        work = torch.empty(floats.value, device="cuda")
        dh, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        _cabi.check(lib.ab200_layer_norm_backward(ptr(gy), cols, ptr(gh), cols, ptr(x), cols, ptr(res), cols, ptr(w), ptr(stats),
                                                  ptr(stats) + 4 * rows, ptr(dh), cols, ptr(dx), cols, ptr(dw), ptr(db), ptr(work),
                                                  rows, cols, 0, 0, p, seed, call, stream))
        for got, ref in zip((dx, dh, dw, db), want):
            assert torch.equal(got, ref)


def test_two_calls_at_once_on_two_streams():
    x, res, w, b = norm_case(3000, 1024, torch.bfloat16, True, 0.1)
    c = adapters_case(3000, 6, 2, 768, 512, 8, torch.bfloat16, 5)
    gy, ga = rand((3000, 1024), torch.bfloat16, 1), rand((3000, 512), torch.bfloat16, 2)

    def norm():
        leaves = [t.detach().requires_grad_() for t in (x, res, w, b)]
        return torch.autograd.grad(digital.add_layer_norm(*leaves, p=0.1, seed=1, call=1)[0], leaves, gy)

    def low_rank():
        leaves = [c[0].detach().requires_grad_(), c[2].detach().requires_grad_(), c[3].detach().requires_grad_()]
        return torch.autograd.grad(digital.low_rank_add(c[1], *leaves, *c[4:7]), leaves, ga)

    want = norm() + low_rank()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            n = norm()
        with torch.cuda.stream(s2):
            l = low_rank()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(n + l, want))


def test_two_captured_graphs_replayed_in_turn():
    """Workspaces belong to a call: two graphs of the same backward pass do not share them."""
    c = adapters_case(600, 5, 2, 256, 320, 8, torch.float32, 5)
    leaves = [t.requires_grad_() for t in (c[0], c[2], c[3])]
    gys = [rand((600, 320), torch.float32, s) for s in (1, 2)]

    def step(gy):
        return torch.autograd.grad(digital.low_rank_add(c[1], *leaves, *c[4:7]), leaves, gy)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(gys[0])
    side.synchronize()
    graphs, outs = [], []
    for gy in gys:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(gy))
        graphs.append(g)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for gy, out in zip(gys, outs):
        assert all(torch.equal(p, q) for p, q in zip(out, step(gy)))


def test_in_place_results_are_seen_by_autograd():
    """A result written over a tensor that autograd has saved is found out, as with torch's own in-place operations."""
    x, base, a, b, scale, ids, starts, _ = adapters_case(40, 4, 2, 64, 96, 8, torch.float32, 3)
    w = torch.ones(96, device="cuda", requires_grad=True)
    y = base * w  # keeps base for the gradient of w
    with torch.no_grad():
        digital.low_rank_add(base, x, a, b, scale, ids, starts, out=base)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_non_finite_rows_stay_to_themselves():
    """Infinities and NaN in rows with an adapter make those rows not finite, and no row beside them in a tile."""
    for dtype in TYPES:
        for requests, ragged in ((40, False), (2, True)):
            x, base, a, b, scale, ids, starts, per_row = adapters_case(40, requests, 2, 64, 96, 8, dtype, 3, ragged)
            want = digital.low_rank_add(base, x, a, b, scale, ids, starts)
            used = (per_row >= 0).nonzero().flatten()
            bad = used[::3]
            x2 = x.clone()
            x2[bad[::2], 5], x2[bad[1::2], 7] = float("nan"), float("inf")
            got = digital.low_rank_add(base, x2, a, b, scale, ids, starts)
            good = torch.ones(40, dtype=torch.bool, device="cuda")
            good[bad] = False
            assert torch.equal(got[good], want[good]) and not torch.isfinite(got[bad]).any()
    x, res, w, b = norm_case(9, 300, torch.bfloat16, True, 0.0)
    y, h = digital.add_layer_norm(x, res, w, b)
    res[4, 17] = float("inf")
    y2, h2 = digital.add_layer_norm(x, res, w, b)
    keep = torch.arange(9, device="cuda") != 4
    assert torch.equal(y2[keep], y[keep]) and torch.isnan(y2[4]).all()
