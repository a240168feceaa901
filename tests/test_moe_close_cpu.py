"""What the close bound of ``moe_close`` notices: the layer in 32 bits passes it, a lost tail, a
lost pair or, in bf16, a dropped low part does not, at every shape that the GPU tests use."""

from __future__ import annotations

import pytest
import torch

import moe_close
import moe_ref

CASES = [(kind, *s, 0, 0) for kind in moe_close.DTYPES for s in moe_close.SHAPES] + \
    [(kind, *s) for kind in moe_close.DTYPES for s in moe_close.LORA_SHAPES]


def single(x, weights, ids, w13, w2, s13=None, s2=None, lora=None, adapter=None):
    """The layer in 32 bits, h and the adapters' sums as two bf16 values."""
    dtype, I = w13.dtype, w2.size(2)
    out = torch.zeros(x.shape)

    def two(v):
        hi = v.to(torch.bfloat16).float()
        return hi + (v - hi).to(torch.bfloat16).float()

    def project(w, scale, v):
        if scale is None:
            return w.float() @ v
        top = v.abs().max().clamp_min(1e-10)
        q = v * moe_ref.QMAX[dtype] / top
        q = q.round() if dtype == torch.int8 else q.to(dtype).float()
        # (sums of int8 products are exact, which 32-bit floats are not)
        y = (w.double() @ q.double()).float() if dtype == torch.int8 else w.float() @ q
        return y * (top / moe_ref.QMAX[dtype]) * scale.reshape(-1)

    for t, picks in enumerate(ids.tolist()):
        v = x[t].float()
        n = -1 if lora is None else int(adapter[t])
        for j, s in enumerate(picks):
            gu = project(w13[s], None if s13 is None else s13[s], v)
            if n >= 0:
                a13, b13, a2, b2 = (m[n, s].float() for m in lora[:4])
                c, r = lora[4][n], a2.size(0)
                u = two(c * (a13 @ v))
                gu = gu + torch.cat([b13[:I] @ u[:r], b13[I:] @ u[r:]])
            g = gu[:I]
            h = g / (1 + torch.exp(-g)) * gu[I:]
            wt = weights[t, j]
            y = w2[s].float() @ two(wt * h) if s2 is None else wt * project(w2[s], s2[s], h)
            if n >= 0:
                y = y + b2 @ two(c * wt * (a2 @ h))
            out[t] += y
    return out.to(torch.bfloat16)


@pytest.mark.parametrize("kind,T,k,S,H,I,L,r", CASES)
def test_bound_takes_32_bits_and_refuses_faults(kind, T, k, S, H, I, L, r):
    # (a bound is of rows and of the layer's widths: one token of two experts says as much)
    T, S, k = 1, 2, min(k, 2)
    a = moe_close.inputs(kind, T, k, S, H, I, L, r)
    want, bound = moe_close.layer(**a)
    assert moe_close.worst(single(**a), want, bound) <= 1.0
    for fault in moe_close.FAULTS:
        if fault[0] in "uv" and not L:
            continue
        # a dropped low part shows in columns near zero, of which 16 may have none; with a
        # quantised h the values next to a border take it in
        if fault.endswith("high only") and (kind != "bf16" or H < 32):
            continue
        wrong, _ = moe_close.layer(**a, fault=fault)
        off = moe_close.worst(wrong.to(torch.bfloat16), want, bound)
        assert off > 1.0, f"{fault}: {off:.2f} of the bound"
