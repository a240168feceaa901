"""The experts' kernels against 64 bits within a bound that a lost tail, a lost pair or a
dropped low part exceeds, at served sizes too (``test_moe_close_cpu`` shows that it does)."""

from __future__ import annotations

import pytest
import torch

import moe_close

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def moe():
    from gpu_util import lib
    lib()
    from vllm_expert_cache import moe
    return moe


@pytest.mark.parametrize("kind", moe_close.DTYPES)
@pytest.mark.parametrize("T,k,S,H,I", moe_close.SHAPES)
def test_experts_close(moe, kind, T, k, S, H, I):
    a = moe_close.inputs(kind, T, k, S, H, I, device=DEV)
    got = moe.experts(a["x"], a["weights"], a["ids"], a["w13"], a["w2"], w13_scale=a["s13"],
                      w2_scale=a["s2"])
    off = moe_close.worst(got, *moe_close.layer(**a))
    assert off <= 1.0, f"{off:.3f} of the bound"


@pytest.mark.parametrize("kind", moe_close.DTYPES)
@pytest.mark.parametrize("T,k,S,H,I,L,r", moe_close.LORA_SHAPES)
def test_experts_lora_close(moe, kind, T, k, S, H, I, L, r):
    a = moe_close.inputs(kind, T, k, S, H, I, L, r, device=DEV)
    got = moe.experts_lora(a["x"], a["weights"], a["ids"], a["w13"], a["w2"], *a["lora"],
                           a["adapter"], w13_scale=a["s13"], w2_scale=a["s2"])
    off = moe_close.worst(got, *moe_close.layer(**a))
    assert off <= 1.0, f"{off:.3f} of the bound"
