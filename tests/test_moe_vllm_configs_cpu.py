"""Which of vLLM's own quantisation configs the plugin gives to the library's experts kernel
(EXPERT_CACHE_MOE=1): the configs come from vLLM's factories, the layer around them from
``test_moe_layer_cpu``."""

from __future__ import annotations

import pytest
import torch

import test_moe_layer_cpu as stand_ins

vllm_config = pytest.importorskip("vllm.model_executor.layers.fused_moe.config")
vllm_int8 = pytest.importorskip("vllm.model_executor.layers.fused_moe.oracle.int8")


@pytest.fixture(autouse=True)
def _env(monkeypatch):
    monkeypatch.setenv("EXPERT_CACHE_SLOTS", str(stand_ins.S))
    monkeypatch.setenv("EXPERT_CACHE_MOE", "1")


def unquantised(layer):
    return vllm_config.FUSED_MOE_UNQUANTIZED_CONFIG


def fp8_per_token(layer):
    return vllm_config.fp8_w8a8_moe_quant_config(
        layer.w13_weight_scale, layer.w2_weight_scale, per_act_token_quant=True,
        per_out_ch_quant=True)


def fp8_per_tensor(layer):
    return vllm_config.fp8_w8a8_moe_quant_config(layer.w13_weight_scale, layer.w2_weight_scale)


def int8_dynamic(layer):
    return vllm_int8.make_int8_moe_quant_config(layer.w13_weight_scale, layer.w2_weight_scale,
                                                per_act_token_quant=True)


def int8_static(layer):
    one = torch.ones(1)
    return vllm_int8.make_int8_moe_quant_config(layer.w13_weight_scale, layer.w2_weight_scale,
                                                one, one, per_act_token_quant=True)


@pytest.mark.parametrize("dtype,config,why", [
    (torch.bfloat16, unquantised, None),
    (torch.float8_e4m3fn, fp8_per_token, None),
    (torch.float8_e4m3fn, fp8_per_tensor, "not quantised dynamically per token"),
    # vLLM runs dynamic int8 layers with bf16 activations
    (torch.int8, int8_dynamic, "unquantised activations"),
    (torch.int8, int8_static, "not quantised dynamically per token"),
])
def test_configs_of_vllm(monkeypatch, dtype, config, why):
    layer = stand_ins.Layer(dtype)
    method = stand_ins.Method(layer)
    method.get_fused_moe_quant_config = config
    _, calls, log = stand_ins.armed(layer, method, monkeypatch)
    stand_ins.step(layer, method)
    assert len(calls) == (why is None) and method.stock == (why is not None)
    assert log.said("keeps its own kernel") == (why is not None)
    if why is not None:
        assert log.said(why), log.msgs
