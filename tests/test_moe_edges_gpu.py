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


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_infinite_scores(moe, scoring, renormalize):
    """A score of +inf makes its token's softmax weights NaN; a sigmoid takes it as 1."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(4, 64, generator=g, device=DEV).abs().to(torch.bfloat16)
    gate = torch.randn(9, 64, generator=g, device=DEV).to(torch.bfloat16)
    x[0, 0] = x[2, 0] = 0                           # 0 times the infinity: a NaN, never picked
    gate[5, 0] = float("inf")
    gate[0:5, 0] = gate[6:, 0] = 0
    gate[5, 1:] = 0
    w, ids = moe.route(x, gate, 6, scoring=scoring, renormalize=renormalize)
    rw, rids = moe_ref.route(x, gate, 6, scoring, renormalize=renormalize)
    assert torch.equal(ids, rids)
    torch.testing.assert_close(w.double(), rw, rtol=2.0 ** -23, atol=1e-37, equal_nan=True)
    for t in (1, 3):
        assert ids[t, 0] == 5
        assert w[t].isnan().all() if scoring == "softmax" else torch.isfinite(w[t]).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_of_a_token_is_the_same_in_every_batch(moe, scoring):
    """Bit for bit: a score is summed in one order whatever the batch."""
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(53, 1000, generator=g, device=DEV).to(torch.bfloat16)
    gate = (torch.randn(300, 1000, generator=g, device=DEV) * 0.03).to(torch.bfloat16)
    w, ids = moe.route(x, gate, 8, scoring=scoring)
    for lo, n in ((0, 1), (52, 1), (7, 3), (20, 5), (4, 30)):
        part = moe.route(x[lo:lo + n], gate, 8, scoring=scoring)
        assert torch.equal(part[0], w[lo:lo + n]) and torch.equal(part[1], ids[lo:lo + n])


def test_rows_further_apart_than_32_bits(moe):
    """x whose rows are 2^32 elements and a row apart: a stride cut to 32 bits is the row
    itself, and would read the second token from behind the first."""
    S, H, I, k = 2, 64, 32, 2
    a = moe_close.inputs("bf16", 2, k, S, H, I, device=DEV)
    far = 2 ** 32 + H
    big = torch.empty(far + H, dtype=torch.bfloat16, device=DEV)
    big[H:2 * H] = 7                                # what a cut stride reads
    x = big.as_strided((2, H), (far, 1))
    x.copy_(a["x"])
    got = moe.experts(x, a["weights"], a["ids"], a["w13"], a["w2"])
    assert moe_close.worst(got, *moe_close.layer(**a)) <= 1.0
    gate = a["w13"][0]
    got, want = moe.route(x, gate, 4), moe.route(a["x"], gate, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_map_of_more_than_32_bits_is_refused(moe):
    a = moe_close.inputs("bf16", 2, 2, 2, 64, 32, device=DEV)
    emap = torch.empty(2 ** 32 + 4, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="expert_map"):
        moe.experts(a["x"], a["weights"], a["ids"], a["w13"], a["w2"], expert_map=emap)
