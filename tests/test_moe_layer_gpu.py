"""Whole cached MoE layers on the GPU: router, cache step (experts fetched from pinned host
memory) and the experts' arithmetic as they are used together, against 64 bits on the full
set of experts."""

from __future__ import annotations

import types

import pytest
import torch

import moe_ref
from gpu_util import DEV, lib, uva_view

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)


class Owner:
    """Expert tensors in pinned host memory, seen by the GPU as vLLM's offloader leaves them."""

    def __init__(self, kind, E, H, I, seed=5):
        import synthetic
        if kind == "int8":
            self.host = synthetic.qwen3_30b_a3b_experts(E=E, seed=seed, hidden=H, inter=I)
        else:
            g = torch.Generator().manual_seed(seed)
            self.host = {n: (torch.randn(s, generator=g) * 0.05).to(torch.bfloat16).pin_memory()
                         for n, s in (("w13_weight", (E, 2 * I, H)), ("w2_weight", (E, H, I)))}
        self.full = {n: t.to(DEV) for n, t in self.host.items()}
        for n, t in self.host.items():
            setattr(self, n, types.SimpleNamespace(data=uva_view(t)))

    def want(self, x, w, ids, **kw):
        f = self.full
        return moe_ref.experts(x, w, ids, f["w13_weight"], f["w2_weight"],
                               f.get("w13_weight_scale"), f.get("w2_weight_scale"), **kw)


def make(kind, E, S, H, I):
    lib()
    from vllm_expert_cache.cache import ExpertSlotCache
    owner = Owner(kind, E, H, I)
    return owner, ExpertSlotCache(owner, list(owner.host), E, S, DEV)


def check(out, want, bound):
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("single_launch", ["1", "0"])
def test_route_and_forward_under_churn(kind, single_launch, monkeypatch):
    monkeypatch.setenv("EXPERT_CACHE_SINGLE_LAUNCH", single_launch)
    E, S, H, I, T, k = 32, 8, 256, 64, 2, 4
    owner, cache = make(kind, E, S, H, I)
    from vllm_expert_cache import moe
    g = gen(1)
    gate = normal(g, E, H, std=0.1)
    seen = set()
    for step in range(8):
        x = normal(g, T, H)
        w, ids = moe.route(x, gate, k)
        ref_w, ref_ids = moe_ref.route(x, gate, k)
        assert torch.equal(ids, ref_ids)
        out = cache.forward(x, w, ids)
        check(out, *owner.want(x, w, ids))
        seen |= set(ids.flatten().tolist())
    assert len(seen) > S                            # experts were swapped
    assert cache.step_timeouts() == 0


def test_forward_pads_and_repeats():
    owner, cache = make("int8", 16, 6, 256, 64)
    g = gen(2)
    x = normal(g, 3, 256)
    w = torch.rand(3, 2, generator=g, device=DEV)
    ids = torch.tensor([[3, 15], [-1, -1], [7, 7]], dtype=torch.int32, device=DEV)
    for dtype in (torch.int32, torch.int64):
        out = cache.forward(x, w, ids.to(dtype))
        check(out, *owner.want(x, w, ids))
        assert (out[1] == 0).all()


def test_forward_with_adapters_follows_experts_through_the_slots():
    E, S, H, I, T, k, L, r = 16, 6, 256, 64, 3, 2, 3, 8
    owner, cache = make("bf16", E, S, H, I)
    g = gen(3)
    lora = (normal(g, L, E, 2 * r, H, std=0.05), normal(g, L, E, 2 * I, r, std=0.1),
            normal(g, L, E, r, I, std=0.05), normal(g, L, E, H, r, std=0.1),
            torch.tensor([1.0, 0.5, 2.0], device=DEV))
    for step in range(6):
        x = normal(g, T, H)
        w = torch.rand(T, k, generator=g, device=DEV)
        ids = torch.stack([torch.randperm(E, generator=g, device=DEV)[:k] for _ in range(T)])
        adapter = torch.randint(-1, L, (T,), generator=g, device=DEV, dtype=torch.int32)
        out = cache.forward(x, w, ids, adapters=lora, adapter=adapter)
        check(out, *owner.want(x, w, ids, lora=lora, adapter=adapter))


def test_forward_expert_parallel():
    """Two ranks' caches over their halves of the experts add up to the whole layer."""
    E, S, H, I, T, k = 16, 5, 256, 64, 2, 2
    owner, _ = make("bf16", E, S, H, I)
    from vllm_expert_cache.cache import ExpertSlotCache
    g = gen(4)
    ranks = []
    for rank in range(2):
        half = types.SimpleNamespace()
        emap = torch.full((E,), -1, dtype=torch.int32, device=DEV)
        emap[rank::2] = torch.arange(E // 2, dtype=torch.int32, device=DEV)
        for n, t in owner.host.items():
            setattr(half, n, types.SimpleNamespace(data=t[rank::2].to(DEV)))
        ranks.append((ExpertSlotCache(half, list(owner.host), E // 2, S, DEV), emap))
    for step in range(4):
        x = normal(g, T, H)
        w = torch.rand(T, k, generator=g, device=DEV)
        ids = torch.stack([torch.randperm(E, generator=g, device=DEV)[:k] for _ in range(T)]).int()
        for rank, (cache, emap) in enumerate(ranks):
            mine = torch.where(ids % 2 == rank, ids, -1)
            check(cache.forward(x, w, ids, expert_map=emap), *owner.want(x, w, mine))


def test_layer_captured_and_replayed():
    """Router, step and experts in one graph: each replay routes, fetches and computes anew."""
    E, S, H, I, T, k = 32, 8, 256, 64, 2, 4
    owner, cache = make("int8", E, S, H, I)
    from vllm_expert_cache import moe
    g = gen(5)
    gate = normal(g, E, H, std=0.1)
    x = normal(g, T, H)

    def layer():
        w, ids = moe.route(x, gate, k)
        return cache.forward(x, w, ids), w, ids
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, w, ids = layer()
    for seed in range(6):
        x.copy_(normal(gen(100 + seed), T, H))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, moe_ref.route(x, gate, k)[1])
        check(out, *owner.want(x, w, ids))
    assert cache.step_timeouts() == 0


def test_two_layers_back_to_back_on_one_stream():
    """Layer after layer without a wait in between: the next layer's step and kernels start
    while the last one's finish."""
    E, S, H, I, T, k = 32, 16, 256, 96, 4, 4
    layers = [make("int8", E, S, H, I), make("bf16", E, S, H, I)]
    g = gen(6)
    x0 = normal(g, T, H)
    w = torch.rand(T, k, generator=g, device=DEV) * 0.1
    ids = [torch.stack([torch.randperm(E, generator=g, device=DEV)[:k] for _ in range(T)]).int()
           for _ in range(8)]
    xs, outs = [], []
    x = x0
    torch.cuda.synchronize()
    for step in range(8):
        out = layers[step % 2][1].forward(x, w, ids[step])
        xs.append(x)
        outs.append(out)
        x = (out / (out.abs().amax() + 1)).to(torch.bfloat16)
    torch.cuda.synchronize()
    for step in range(8):
        check(outs[step], *layers[step % 2][0].want(xs[step], w, ids[step]))
