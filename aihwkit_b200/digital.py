"""Digital operators around the analog tiles of a transformer block: layer norm (with the residual sum and the dropout in
front of it), dropout from a counter-based generator, and low-rank adapters of many requests beside a shared projection.

The conductances of an analog tile are written once, so a model on tiles is adapted digitally.  In the reference these parts
are torch calls around ``AnalogLinear``; here they are kernels of the library (``csrc/layer_norm.cu``, ``csrc/dropout.cu``,
``csrc/low_rank.cu``) behind the C ABI, differentiable where autograd asks.

All of them take CUDA tensors of float32, float16 or bfloat16 whose last dimension lies together in memory (others are
copied first), run on the current stream of the tensors' device, wait for nothing and raise ``RuntimeError`` for what they
do not take.  Sums and means are held in fp32 and results are rounded once.  In the products of the adapters 16-bit factors are
exact; fp32 ones (all of an fp32 call, and ``x a^T`` or ``gy b^T`` on the way into the second product) have at least 22 of their
24 bits there, beside bfloat16 all.  Gradients are those of reverse mode, once: second derivatives, forward mode, tracing and
``torch.func`` are refused.  The calls can be captured into a CUDA graph; a captured dropout repeats the ``call`` it was
captured with.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .build import DIGITAL_OUT

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _load():
    import importlib.util
    import os

    if not os.path.exists(DIGITAL_OUT):
        raise RuntimeError(f"{DIGITAL_OUT} is missing: run `python -m aihwkit_b200.build` (nvcc, sm_100a)")
    spec = importlib.util.spec_from_file_location("ab200_digital", DIGITAL_OUT)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


#: the binding over the C ABI, ``csrc/digital_module.cpp``
_ext = _load()


def dropout(x: torch.Tensor, p: float = 0.5, seed: int = 0, call: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` with every element set to zero with probability ``p`` and divided by ``1 - p`` otherwise, plus ``residual``.

    Which elements stay is a function of ``seed``, ``call``, the element's row (all dimensions but the last, in order), its
    column and the number of columns (``ab200_dropout`` in the header spells it out): vary ``call`` from one dropout to the
    next.  No mask is stored; the backward pass draws it again.  A dropped element is 0 whatever it held, and with
    ``p = 1`` all are."""
    return _ext.dropout(x, p, seed, call, residual)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension (at most 16384 elements).  ``weight``
    and ``bias`` may be missing; they are of the type of ``x`` or float32, and so are their gradients."""
    return _ext.layer_norm(x, weight, bias, eps)


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, p: float = 0.0, seed: int = 0,
                   call: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = residual + dropout(x)`` and ``y = layer_norm(h)`` in one pass; returns ``(y, h)``: what the next layer reads and
    the residual stream behind it.  ``p``, ``seed`` and ``call`` are those of :func:`dropout` (``p = 0``: none); both results
    are rounded from the same fp32 sum."""
    return _ext.add_layer_norm(x, residual, weight, bias, eps, p, seed, call)


def low_rank_add(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor,
                 adapter_ids: torch.Tensor, row_starts: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``base + scale[i] (x a[i]^T) b[i]`` with the adapter ``i`` of each row's request.

    ``x`` is ``[..., k]`` and ``base`` ``[..., n]`` with the same rows; ``a`` is ``[adapters, rank, k]``, ``b``
    ``[adapters, rank, n]`` (both rank first), all of one type; ``scale`` is float32 ``[adapters]``.  Request ``j`` has the
    adapter ``adapter_ids[j]`` (int32 on the device; outside ``[0, adapters)``: none) and the rows from ``row_starts[j]`` up to
    ``row_starts[j + 1]`` (int32 on the device, one more value than requests, not decreasing); without ``row_starts`` request
    ``j`` is row ``j``.  Rows without an adapter, or in no request, are ``base``.  ``out`` takes the result - ``base`` itself
    among others, whose rows without an adapter are then not touched - in calls without gradients.  Differentiable in
    ``base``, ``x``, ``a`` and ``b``.  Neighbouring rows of one adapter cost least as one request: in the backward pass above
    all, where every request takes ``rank * (k + n)`` floats of workspace."""
    return _ext.low_rank_add(base, x, a, b, scale, adapter_ids, row_starts, out)


class LowRankAdapters(torch.nn.Module):
    """A pool of low-rank adapters beside one projection of ``in_features`` to ``out_features``, such as a
    :class:`~aihwkit_b200.rpu_base.tiles.TileArray`: ``y = tiles(x)``, then ``adapters(y, x, adapter_ids, row_starts)``.

    ``a`` is drawn from N(0, 1 / in_features) and ``b`` is zero, so a fresh adapter changes nothing."""

    def __init__(self, n_adapters: int, in_features: int, out_features: int, rank: int, scale: float = 1.0,
                 device="cuda", dtype: torch.dtype = torch.float32, generator: Optional[torch.Generator] = None):
        super().__init__()
        if min(n_adapters, in_features, out_features, rank) < 1 or rank > 256 or n_adapters > 65535:
            raise RuntimeError("LowRankAdapters: 1 to 65535 adapters of rank 1 to 256, at least one feature each way")
        if dtype not in _DTYPES:
            raise RuntimeError(f"LowRankAdapters: float32, float16 or bfloat16, got {dtype}")
        a = torch.randn(n_adapters, rank, in_features, generator=generator) * in_features ** -0.5
        self.a = torch.nn.Parameter(a.to(device=device, dtype=dtype))
        self.b = torch.nn.Parameter(torch.zeros(n_adapters, rank, out_features, device=device, dtype=dtype))
        self.register_buffer("scale", torch.full((n_adapters,), float(scale), device=device, dtype=torch.float32))

    def _apply(self, fn, recurse=True):
        """Conversions of the pool to another type leave ``scale`` in float32, as the calls take it."""
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = self.scale.float() if scale.is_meta else scale.to(self.scale.device)
        return self

    @torch.no_grad()
    def set_adapter(self, index: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Adapter ``index`` becomes ``scale * b @ a`` with ``a [r, in_features]`` and ``b [out_features, r]``, ``r`` at most
        the pool's rank (the rest is zero)."""
        n, rank, k = self.a.shape
        r = a.size(0) if a.dim() == 2 else -1
        if not 0 <= index < n:
            raise RuntimeError(f"adapter index must be between 0 and {n - 1}, got {index}")
        if not 0 <= r <= rank or a.shape != (r, k) or b.shape != (self.b.size(2), r):
            raise RuntimeError(f"expected a [r, {k}] and b [{self.b.size(2)}, r] with r <= {rank}, got {tuple(a.shape)} and "
                               f"{tuple(b.shape)}")
        self.a[index].zero_()
        self.b[index].zero_()
        self.a[index, :r].copy_(a)
        self.b[index, :r].copy_(b.t())
        self.scale[index] = float(scale)

    def forward(self, base: torch.Tensor, x: torch.Tensor, adapter_ids: torch.Tensor,
                row_starts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        return low_rank_add(base, x, self.a, self.b, self.scale, adapter_ids, row_starts, out)
