"""Ends of the ranges of the layer's operators."""

from __future__ import annotations

import pytest
import torch

import moe_close
import moe_ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def moe():
    from gpu_util import lib
    lib()
    from vllm_expert_cache import moe
    return moe


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("T,at", [(1, 0), (33, 20)])
def test_experts_rows_next_to_the_largest_floats(moe, kind, T, at):
    """x whose product with the type's largest value is beyond fp32, an element of it on a
    border between two values of the type."""
    S, H, I, k = 2, 512, 64, 2
    a = moe_close.inputs(kind, T, k, S, H, I, device=DEV)
    top = 21 * 2.0 ** 115                           # 8.7e35
    x = torch.zeros(H, dtype=torch.float64, device=DEV)
    step = top / moe_ref.QMAX[moe_close.DTYPES[kind]]
    # 448: whole steps 448, 416, the tie 272 and -400; 127: the largest and others of its size
    values = [448, 416, 272, -400] if kind == "fp8" else [127, 120, 63.5, -118]
    x[8:12] = torch.tensor(values, dtype=torch.float64, device=DEV) * step
    a["x"][at] = x.to(torch.bfloat16)
    if kind == "fp8":
        assert torch.equal(a["x"][at].double(), x)  # they are values of bf16
    a["s13"][:] *= 1e-33
    want, bound = moe_close.layer(**a)
    got = moe.experts(a["x"], a["weights"], a["ids"], a["w13"], a["w2"], w13_scale=a["s13"],
                      w2_scale=a["s2"])
    assert torch.isfinite(want).all() and (want[at].abs() > 1e-6).any()
    off = ((got.double() - want).abs() / bound)[at].max().item()
    assert off <= 1.0, f"{off:.3f} of the bound"
