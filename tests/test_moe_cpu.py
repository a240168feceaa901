"""The MoE layer's operators on a machine without a GPU: the C-ABI refuses bad arguments
with -1 before touching CUDA, the Python functions with ValueError."""

from __future__ import annotations

import ctypes

import pytest
import torch

NULL = None
BUF = 1 << 20          # 256-byte aligned; never dereferenced by a refused call


@pytest.fixture(scope="module")
def h():
    import build_lib
    from vllm_expert_cache import _lib
    build_lib.build()
    return _lib.lib()


def experts(h, lora=None, T=2, ldx=32, H=32, I=32, k=2, S=4, wtype=0, x=BUF, ids=BUF, w=BUF,
            emap=NULL, n_map=0, w13=BUF, s13=NULL, w2=BUF, s2=NULL, out=BUF, ldo=32, ws=BUF,
            nbytes=1 << 20):
    head = (x, T, ldx, H, ids, w, k, emap, n_map, w13, s13, w2, s2, wtype, S, I)
    tail = (out, ldo, ws, nbytes, NULL)
    if lora is None:
        return h.expert_cache_experts(*head, *tail)
    a = dict(adapter=BUF, a13=BUF, b13=BUF, a2=BUF, b2=BUF, scaling=BUF, L=2, E=4, r=8)
    a.update(lora)
    return h.expert_cache_experts_lora(*head, *a.values(), *tail)


BAD = [dict(T=-1), dict(k=0), dict(k=33), dict(S=0), dict(S=1025), dict(wtype=3),
       dict(wtype=-1), dict(H=0), dict(H=36), dict(I=0), dict(I=28), dict(H=32776, ldx=32776),
       dict(I=32776), dict(ldx=24), dict(ldx=36), dict(ldo=31), dict(x=BUF + 8),
       dict(w13=BUF + 8), dict(w2=BUF + 4), dict(out=BUF + 1), dict(x=NULL), dict(ids=NULL),
       dict(w=NULL), dict(w13=NULL), dict(w2=NULL), dict(out=NULL), dict(ids=BUF + 2),
       dict(w=BUF + 1), dict(emap=BUF, n_map=0), dict(emap=BUF, n_map=-1), dict(n_map=-1),
       dict(emap=BUF + 2, n_map=4), dict(s13=BUF), dict(s2=BUF), dict(ws=NULL),
       dict(ws=BUF + 128), dict(nbytes=64), dict(wtype=1), dict(wtype=2, s13=BUF),
       dict(wtype=1, s2=BUF), dict(wtype=1, s13=BUF, s2=BUF, I=24),
       dict(wtype=2, s13=BUF, s2=BUF, H=24, ldx=24), dict(wtype=1, s13=BUF + 1, s2=BUF)]


@pytest.mark.parametrize("kw", BAD)
@pytest.mark.parametrize("lora", [None, {}])
def test_experts_refuse_bad_arguments(h, kw, lora):
    assert experts(h, lora, **kw) == -1


@pytest.mark.parametrize("kw", [dict(L=0), dict(L=-1), dict(E=0), dict(r=0), dict(r=12),
                                dict(r=-8), dict(r=264), dict(adapter=NULL), dict(a13=NULL),
                                dict(b13=NULL), dict(a2=NULL), dict(b2=NULL),
                                dict(scaling=NULL), dict(a13=BUF + 8), dict(b13=BUF + 2),
                                dict(a2=BUF + 8), dict(b2=BUF + 8), dict(adapter=BUF + 2),
                                dict(scaling=BUF + 1)])
def test_experts_lora_refuses_bad_adapters(h, kw):
    assert experts(h, kw) == -1


def test_empty_batch_enqueues_nothing(h):
    assert experts(h, T=0) == 0 and experts(h, {}, T=0) == 0


@pytest.mark.parametrize("args", [(-1, 2, 32, 32, 0, 0), (2, 0, 32, 32, 0, 0),
                                  (2, 33, 32, 32, 0, 0), (2, 2, 36, 32, 0, 0),
                                  (2, 2, 32, 0, 0, 0), (2, 2, 32, 32, 3, 0),
                                  (2, 2, 24, 32, 1, 0), (2, 2, 32, 32, 0, 4),
                                  (2, 2, 32, 32, 0, 264), (2, 2, 32, 32, 0, -8)])
def test_workspace_refuses_bad_sizes(h, args):
    n = ctypes.c_long(-7)
    assert h.expert_cache_experts_workspace(*args, ctypes.byref(n)) == -1 and n.value == -7


def test_workspace_does_not_grow_with_a_long_batch(h):
    n = ctypes.c_long()

    def need(T, wtype=0, r=0):
        assert h.expert_cache_experts_workspace(T, 8, 2048, 768, wtype, r, ctypes.byref(n)) == 0
        return n.value
    assert need(0) == 0
    assert 0 < need(1) < need(4) < need(16)
    assert need(64) == need(10 ** 6)               # a launch takes a bounded number of tokens
    assert need(4, r=16) > need(4)
    for wtype in (1, 2):
        assert need(1, wtype) > 0


@pytest.mark.parametrize("kw", [dict(T=-1), dict(H=0), dict(H=12, ldx=16), dict(H=16392, ldx=16392),
                                dict(ldx=8), dict(ldx=20), dict(E=0), dict(E=2049), dict(k=0),
                                dict(k=9), dict(E=64, k=33), dict(scoring=2), dict(scoring=-1),
                                dict(bias=BUF), dict(x=BUF + 8), dict(gate=BUF + 8),
                                dict(x=NULL), dict(gate=NULL), dict(out=NULL), dict(ids=NULL),
                                dict(out=BUF + 2), dict(ids=BUF + 1),
                                dict(scoring=1, bias=BUF + 2)])
def test_route_refuses_bad_arguments(h, kw):
    a = dict(T=2, ldx=16, H=16, E=8, k=4, x=BUF, gate=BUF, scoring=0, bias=NULL, out=BUF, ids=BUF)
    a.update(kw)

    def call(T):
        return h.expert_cache_route(a["x"], T, a["ldx"], a["H"], a["gate"], a["E"], a["k"],
                                    a["scoring"], 1, a["bias"], 1.0, a["out"], a["ids"], NULL)
    assert call(a["T"]) == -1


def test_route_empty_batch_enqueues_nothing(h):
    assert h.expert_cache_route(BUF, 0, 16, 16, BUF, 8, 4, 0, 1, NULL, 1.0, BUF, BUF, NULL) == 0


def test_python_refuses_host_tensors():
    from vllm_expert_cache import moe
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    ids = torch.zeros(2, 2, dtype=torch.int32)
    w = torch.zeros(2, 2)
    w13, w2 = (torch.zeros(s, dtype=torch.bfloat16) for s in ((4, 32, 32), (4, 32, 16)))
    with pytest.raises(ValueError, match="GPU"):
        moe.experts(x, w, ids, w13, w2)
    with pytest.raises(ValueError, match="GPU"):
        moe.route(x, torch.zeros(4, 32, dtype=torch.bfloat16), 2)
    with pytest.raises(ValueError, match="scoring"):
        moe.route(x, torch.zeros(4, 32, dtype=torch.bfloat16), 2, scoring="relu")
