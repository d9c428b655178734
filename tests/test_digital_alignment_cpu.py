"""Addresses off the alignment that the kernels' accesses need are refused by the C entry points, before anything is launched."""

import pytest

from tests.test_digital_cpu import P, dropout_args, grad_args, low_rank_args, norm_args, norm_grad_args, refused

ARGS = {"ab200_dropout": dropout_args, "ab200_layer_norm_forward": norm_args, "ab200_layer_norm_backward": norm_grad_args,
        "ab200_low_rank_apply": low_rank_args, "ab200_low_rank_grad": grad_args}


@pytest.mark.parametrize("name, pointers", [
    ("ab200_dropout", dict(x="x", r="residual", y="y")),
    ("ab200_layer_norm_forward", dict(x="x", r="residual", y="y", h="h")),
    ("ab200_layer_norm_backward", dict(gy="gy", gh="gh", x="x", r="residual", dh="dh", dx="dx")),
    ("ab200_low_rank_apply", dict(x="x", base="base", y="y", a="a", b="b")),
    ("ab200_low_rank_grad", dict(x="x", gy="gy", da="da", db="db"))])
def test_elements(name, pointers):
    for key, word in pointers.items():
        strides = dict(hs=8, dxs=8)
        for dtype, off in ((0, 2), (0, 1), (1, 1), (2, 1)):
            kw = {key: P + off, "dtype": dtype}
            for other, stride in (("h", "hs"), ("dx", "dxs")):
                if key == other:
                    kw[stride] = strides[stride]
            refused(name, ARGS[name](**kw), f"{word} must lie on a multiple of")


@pytest.mark.parametrize("name, pointers", [
    ("ab200_layer_norm_forward", dict(w="weight", b="bias")),
    ("ab200_layer_norm_backward", dict(w="weight", dw="dweight", db="dbias"))])
def test_parameters(name, pointers):
    for key, word in pointers.items():
        for pdtype, off in ((0, 2), (1, 1), (2, 1)):
            kw = {key: P + off, "pdtype": pdtype}
            if name.endswith("backward"):
                kw["work"] = P
            refused(name, ARGS[name](**kw), f"{word} must lie on a multiple of")


@pytest.mark.parametrize("name, pointers", [
    ("ab200_layer_norm_backward", dict(mean="mean", rstd="rstd", work="workspace")),
    ("ab200_low_rank_apply", dict(scale="scale", ids="adapter_ids", v="v")),
    ("ab200_low_rank_grad", dict(u="u", v="v", ids="adapter_ids"))])
def test_fp32_values_and_tables(name, pointers):
    for key, word in pointers.items():
        refused(name, ARGS[name](**{key: P + 2, "dtype": 1}), f"{word} must lie on a multiple of 4 bytes")
    refused("ab200_layer_norm_forward", norm_args(mean=P, rstd=P + 2), "rstd must lie on a multiple of 4 bytes")
    for name in ("ab200_low_rank_apply", "ab200_low_rank_grad"):
        refused(name, ARGS[name](starts=P + 2), "row_starts must lie on a multiple of 4 bytes")


@pytest.mark.parametrize("off", [4, 8, 12])
def test_workspace_of_the_low_rank_gradients(off):
    """Its partial sums are stored 16 bytes at a time."""
    refused("ab200_low_rank_grad", grad_args(work=P + off), "workspace must lie on a multiple of 16 bytes")
