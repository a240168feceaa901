"""The plugin's use of the library's own experts kernel (EXPERT_CACHE_MOE=1) on stand-ins for
vLLM's classes: which layers qualify, what a cached step then calls, and that everything
else keeps the stock kernel.  ``refresh`` is replaced, so no kernel runs."""

from __future__ import annotations

from dataclasses import dataclass, field

import pytest
import torch

from vllm_expert_cache import moe
from vllm_expert_cache.backends import generic

E, S, H, I = 16, 4, 32, 48


class Log:
    def __init__(self):
        self.msgs = []

    def _rec(self, fmt, *a):
        self.msgs.append(fmt % a if a else fmt)

    warning = info = debug = _rec

    def said(self, needle):
        return any(needle in m for m in self.msgs)


@dataclass
class Shape:
    row: int
    col: int


@dataclass
class Desc:
    dtype: torch.dtype | None = None
    shape: Shape | None = None
    scale: torch.Tensor | None = None
    alpha_or_gscale: torch.Tensor | None = None
    zp: torch.Tensor | None = None
    bias: torch.Tensor | None = None


@dataclass
class Config:
    _a1: Desc = field(default_factory=Desc)
    _a2: Desc = field(default_factory=Desc)
    _w1: Desc = field(default_factory=Desc)
    _w2: Desc = field(default_factory=Desc)
    gemm1_clamp_limit: float | None = None


class TritonExperts:
    def __init__(self, cfg):
        self.quant_config = cfg


class OtherExperts(TritonExperts):
    pass


class MoEPrepareAndFinalizeNoDPEPModular:
    activation_format = type("F", (), {"name": "Standard"})()


class AllToAll(MoEPrepareAndFinalizeNoDPEPModular):
    pass


class Kernel:
    def __init__(self, cfg, experts=TritonExperts, around=MoEPrepareAndFinalizeNoDPEPModular):
        self.fused_experts = experts(cfg)
        self.prepare_finalize = around()

    def supports_expert_map(self):
        return True


class Layer(torch.nn.Module):
    def __init__(self, dtype=torch.bfloat16, hidden=H, inter=I):
        super().__init__()

        def p(*shape, dt=dtype):
            return torch.nn.Parameter(torch.zeros(shape, dtype=dt), requires_grad=False)
        self.w13_weight, self.w2_weight = p(E, 2 * inter, hidden), p(E, hidden, inter)
        if dtype != torch.bfloat16:
            self.w13_weight_scale = p(E, 2 * inter, 1, dt=torch.float32)
            self.w2_weight_scale = p(E, hidden, 1, dt=torch.float32)
        self.global_num_experts = E
        self.activation = type("A", (), {"value": "silu"})()
        self.apply_router_weight_on_input = False
        self.expert_map = None


class Method:
    is_monolithic = False
    disable_expert_map = False

    def __init__(self, layer, cfg=None, **kernel):
        self.act = cfg
        self.moe_quant_config = self.get_fused_moe_quant_config(layer)
        self.moe_kernel = Kernel(self.moe_quant_config, **kernel)
        self.stock = 0

    def get_fused_moe_quant_config(self, layer):
        cfg = Config()
        if self.act is not None:
            cfg._a1, cfg._a2 = self.act(), self.act()
        if hasattr(layer, "w13_weight_scale"):
            cfg._w1 = Desc(layer.w13_weight.dtype, scale=layer.w13_weight_scale)
            cfg._w2 = Desc(layer.w2_weight.dtype, scale=layer.w2_weight_scale)
        return cfg

    def apply(self, layer, x, topk_weights, topk_ids, shared_experts=None,
              shared_experts_input=None):
        self.stock += 1
        return x.clone()


def per_token(dtype):
    return lambda: Desc(dtype, Shape(1, -1))


@pytest.fixture(autouse=True)
def _env(monkeypatch):
    monkeypatch.setenv("EXPERT_CACHE_SLOTS", str(S))
    monkeypatch.setenv("EXPERT_CACHE_MOE", "1")


def armed(layer, method, monkeypatch):
    log = Log()
    assert generic.arm(layer, method, log)
    cache = layer._expert_cache
    calls = []
    cache.refresh = lambda ids: ids
    cache.refresh_ep = lambda ids, emap: emap + 100
    monkeypatch.setattr(moe, "experts", lambda *a, **k: calls.append((a, k)) or a[0] * 2)
    return cache, calls, log


def step(layer, method, T=2, k=2, dtype=torch.bfloat16, **kw):
    return method.apply(layer=layer, x=torch.ones(T, layer.w2_weight.size(1), dtype=dtype),
                        topk_weights=torch.ones(T, k),
                        topk_ids=torch.zeros(T, k, dtype=torch.int32), **kw)


@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, None),
                                       (torch.int8, per_token(torch.int8)),
                                       (torch.float8_e4m3fn, per_token(torch.float8_e4m3fn))])
def test_cached_step_runs_the_own_kernel_on_the_slots(monkeypatch, dtype, act):
    layer = Layer(dtype)
    method = Method(layer, act)
    cache, calls, _ = armed(layer, method, monkeypatch)
    before = layer.w13_weight
    out = step(layer, method)
    assert (out == 2).all() and method.stock == 0 and len(calls) == 1
    (_, _, _, w13, w2), kw = calls[0]
    assert w13 is cache.slots["w13_weight"] and w2 is cache.slots["w2_weight"]
    assert kw["expert_map"] is cache.table
    if act is None:
        assert kw["w13_scale"] is None and kw["w2_scale"] is None
    else:
        assert kw["w13_scale"] is cache.slots["w13_weight_scale"]
        assert kw["w2_scale"] is cache.slots["w2_weight_scale"]
    # the layer is as it was
    assert layer.w13_weight is before and layer.global_num_experts == E
    assert method.moe_kernel.fused_experts.quant_config is method.moe_quant_config


def test_expert_parallel_step_uses_the_composed_map(monkeypatch):
    monkeypatch.setenv("EXPERT_CACHE_EP", "1")
    layer = Layer()
    layer.expert_map = torch.arange(2 * E, dtype=torch.int32)
    method = Method(layer)
    _, calls, _ = armed(layer, method, monkeypatch)
    step(layer, method)
    assert method.stock == 0
    assert torch.equal(calls[0][1]["expert_map"], torch.arange(2 * E, dtype=torch.int32) + 100)
    assert torch.equal(layer.expert_map, torch.arange(2 * E, dtype=torch.int32))


def test_off_by_default(monkeypatch):
    monkeypatch.delenv("EXPERT_CACHE_MOE")
    layer = Layer()
    method = Method(layer)
    _, calls, log = armed(layer, method, monkeypatch)
    step(layer, method)
    assert method.stock == 1 and not calls and not log.said("keeps its own kernel")


@pytest.mark.parametrize("kw", [dict(shared_experts=object()), dict(dtype=torch.float16),
                                dict(T=1, k=33), dict(T=3, k=2)])
def test_other_steps_keep_the_stock_kernel(monkeypatch, kw):
    """Shared experts, another activation type, too many experts a token, wide steps."""
    if kw.get("k") == 33:
        monkeypatch.setenv("EXPERT_CACHE_SLOTS", "15")
    layer = Layer()
    method = Method(layer)
    _, calls, _ = armed(layer, method, monkeypatch)
    step(layer, method, **kw)
    assert method.stock == 1 and not calls


def _gelu(layer, method):
    layer.activation = "gelu"


def _on_input(layer, method):
    layer.apply_router_weight_on_input = True


def _clamp(layer, method):
    orig = method.get_fused_moe_quant_config

    def cfg(l):
        c = orig(l)
        c.gemm1_clamp_limit = 7.0
        return c
    method.get_fused_moe_quant_config = cfg


@pytest.mark.parametrize("make,why", [
    (lambda: (Layer(), dict(experts=OtherExperts)), "another layout"),
    (lambda: (Layer(), dict(around=AllToAll)), "moves tokens"),
    (lambda: (Layer(torch.float32), {}), "weights are"),
    (lambda: (Layer(inter=44), {}), "beyond the kernels' limits"),
    (lambda: (Layer(torch.int8), {}), "unquantised activations"),
    (lambda: (Layer(torch.int8), dict(cfg=lambda: Desc(torch.int8, Shape(-1, -1)))),
     "dynamically per token"),
    (lambda: (Layer(torch.int8), dict(cfg=lambda: Desc(torch.int8, Shape(1, -1),
                                                       scale=torch.ones(1)))),
     "dynamically per token"),
    (lambda: (Layer(), dict(cfg=lambda: Desc(bias=torch.ones(1)))), "bias"),
    (lambda: (Layer(), dict(cfg=per_token(torch.float8_e4m3fn))), "activations are"),
])
def test_layers_that_keep_their_kernel(monkeypatch, make, why):
    layer, kw = make()
    method = Method(layer, **kw)
    _, calls, log = armed(layer, method, monkeypatch)
    assert log.said("keeps its own kernel") and log.said(why), log.msgs
    step(layer, method)
    assert method.stock == 1 and not calls


@pytest.mark.parametrize("change,why", [(_gelu, "activation"), (_on_input, "on the input"),
                                        (_clamp, "clamped")])
def test_layer_settings_that_keep_the_kernel(monkeypatch, change, why):
    layer = Layer()
    method = Method(layer)
    change(layer, method)
    _, calls, log = armed(layer, method, monkeypatch)
    assert log.said(why), log.msgs
    step(layer, method)
    assert method.stock == 1 and not calls


def test_forward_refuses_a_step_wider_than_the_slots(monkeypatch):
    layer = Layer()
    cache, calls, _ = armed(layer, Method(layer), monkeypatch)
    x, w = torch.ones(3, H, dtype=torch.bfloat16), torch.ones(3, 2)
    with pytest.raises(ValueError, match="slots"):
        cache.forward(x, w, torch.zeros(3, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="adapter"):
        cache.forward(x[:2], w[:2], torch.zeros(2, 2, dtype=torch.int32), adapters=(1,) * 5)
    cache.forward(x[:2], w[:2], torch.zeros(2, 2, dtype=torch.int32))
    assert len(calls) == 1 and calls[0][1]["expert_map"] is cache.table


@pytest.mark.parametrize("ids,weights", [(torch.uint32, torch.float32), (torch.int16, torch.float32),
                                         (torch.int32, torch.int32)])
def test_routing_of_other_types_keeps_the_stock_kernel(monkeypatch, ids, weights):
    layer = Layer()
    method = Method(layer)
    _, calls, _ = armed(layer, method, monkeypatch)
    method.apply(layer=layer, x=torch.ones(2, H, dtype=torch.bfloat16),
                 topk_weights=torch.ones(2, 2, dtype=weights),
                 topk_ids=torch.zeros(2, 2, dtype=ids))
    assert method.stock == 1 and not calls
