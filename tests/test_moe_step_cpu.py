"""Which cached steps the plugin gives to the library's own experts kernel
(EXPERT_CACHE_MOE=1), on the stand-ins of ``test_moe_layer_cpu``."""

from __future__ import annotations

import pytest
import torch

from vllm_expert_cache import moe
import test_moe_layer_cpu as stand_ins


@pytest.fixture(autouse=True)
def _env(monkeypatch):
    monkeypatch.setenv("EXPERT_CACHE_SLOTS", "15")
    monkeypatch.setenv("EXPERT_CACHE_MOE", "1")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("T", [1, 8, 9, 15])
def test_steps_that_the_stock_kernel_does_faster_keep_it(monkeypatch, dtype, T):
    layer = stand_ins.Layer(dtype)
    method = stand_ins.Method(
        layer, None if dtype == torch.bfloat16 else stand_ins.per_token(dtype))
    _, calls, _ = stand_ins.armed(layer, method, monkeypatch)
    stand_ins.step(layer, method, T=T, k=1)
    own = T <= 8
    assert moe.STEP_TOKENS == 8 and len(calls) == own and method.stock == (not own)
