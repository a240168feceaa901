"""The MoE layer's operators from their definitions in 64 bits, with a bound on what a right
kernel may be off by: every product and sum in fp32 (a sum of n terms is off by at most
n * 2^-23 of the sum of their magnitudes, whatever its order), h in 16 bits of mantissa, one
rounding of the output to bf16 (half a step: 2^-8 of the value).  For 8-bit weights the
quantised h may land on either side of a border that its own error reaches."""

from __future__ import annotations

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
EPS = 2.0 ** -23
TINY = 1e-30


def to_grid(v, dtype):
    """v (64 bits) on the 8-bit type's values, ties to even."""
    if dtype == torch.int8:
        return torch.round(v).clamp(-127, 127)
    return v.clamp(-448, 448).to(torch.float8_e4m3fn).double()


def quantise(v, dtype):
    """(q, scale, top) of one row in 64 bits."""
    top = v.abs().max().clamp_min(1e-10)
    return to_grid(v * QMAX[dtype] / top, dtype), top / QMAX[dtype], top


def slot_of(i, S, expert_map):
    if expert_map is not None:
        i = int(expert_map[i]) if 0 <= i < expert_map.numel() else -1
    return i if 0 <= i < S else -1


def experts(x, weights, ids, w13, w2, s13=None, s2=None, expert_map=None, lora=None,
            adapter=None):
    """(out, bound), both [T, H] in 64 bits.  lora: (a13, b13, a2, b2, scaling)."""
    S, I, dtype = w2.size(0), w2.size(2), w13.dtype
    T, H = x.shape
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    err, mag = out.clone(), out.clone()
    emap = None if expert_map is None else expert_map.cpu()
    for t in range(T):
        xt = x[t].double()
        for j, i in enumerate(ids[t].tolist()):
            s = slot_of(i, S, emap)
            if s < 0:
                continue
            w13s, w2s = w13[s].double(), w2[s].double()
            if dtype in QMAX:
                q, sc, _ = quantise(xt, dtype)
                w13s = w13s * s13[s].double().reshape(-1, 1)
                gu, m = w13s @ (q * sc), w13s.abs() @ (q * sc).abs()
                d = (H + 8) * EPS * m if dtype != torch.int8 else 8 * EPS * m
            else:
                gu, m = w13s @ xt, w13s.abs() @ xt.abs()
                d = H * EPS * m
            a = int(adapter[t]) if lora is not None else -1
            a = a if lora is not None and 0 <= a < lora[0].size(0) and \
                0 <= i < lora[0].size(1) else -1
            if a >= 0:
                a13, b13, a2, b2 = (m_[a, i].double() for m_ in lora[:4])
                c, r = float(lora[4][a]), a2.size(0)
                u, um = a13 @ xt, a13.abs() @ xt.abs()
                for half in (0, 1):
                    b = b13[half * I:(half + 1) * I]
                    k = slice(half * r, (half + 1) * r)
                    gu[half * I:(half + 1) * I] += c * (b @ u[k])
                    # (A x and A2 h, like h, in 16 bits of mantissa)
                    d[half * I:(half + 1) * I] += abs(c) * (
                        (H + r + 4) * EPS + 2.0 ** -16) * (b.abs() @ um[k])
            g, up = gu[:I], gu[I:]
            act = g * torch.sigmoid(g)
            h = act * up
            # silu's slope is at most 1.1; expf and the division: a few units in the last place
            dh = 1.1 * up.abs() * d[:I] + act.abs() * d[I:] + h.abs() * 2.0 ** -16 + TINY
            wt = float(weights[t, j])
            y_h, dy_h = h, dh
            if dtype in QMAX:
                q, sc, top = quantise(h, dtype)
                wide = dh + h.abs() * (dh.max() / top + 4 * EPS)
                near = [to_grid((h + side * wide) * QMAX[dtype] / top, dtype) for side in (-1, 1)]
                dq = torch.maximum((near[0] - q).abs(), (near[1] - q).abs())
                y_h, dy_h = q * sc, dq * sc + (q * sc).abs() * (dh.max() / top + 4 * EPS)
                w2s = w2s * s2[s].double().reshape(-1, 1)
            y = w2s @ y_h
            dy = w2s.abs() @ dy_h
            ym = w2s.abs() @ y_h.abs()
            if a >= 0:
                v = a2 @ h
                y = y + c * (b2 @ v)
                vm = a2.abs() @ h.abs()
                dv = a2.abs() @ dh + ((I + r + 4) * EPS + 2.0 ** -16) * vm
                dy = dy + abs(c) * (b2.abs() @ dv)
                ym = ym + abs(c) * (b2.abs() @ vm)
            out[t] += wt * y
            err[t] += abs(wt) * dy
            mag[t] += abs(wt) * ym
    n = I * max(1, ids.size(1)) + 16
    return out, err + n * EPS * mag + 2.0 ** -8 * out.abs() + 1e-38


def route(x, gate_w, k, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    """(weights in 64 bits, ids) with ties to the lower id, NaN and -inf never picked."""
    z = x.double() @ gate_w.double().T
    if scoring == "softmax":
        top = torch.where(z.isnan(), -torch.inf, z).amax(1, keepdim=True)
        p = torch.exp(z - top)
        p = p / torch.where(z.isnan(), 0.0, p).sum(1, keepdim=True)
        key = z.clone()
    else:
        p = torch.sigmoid(z)
        key = p + (0 if bias is None else bias.double())
    key = torch.where(key.isnan(), -torch.inf, key)
    best = torch.sort(key, dim=1, descending=True, stable=True)
    ids = best.indices[:, :k].clone()
    gone = best.values[:, :k] == -torch.inf
    w = torch.where(gone, 0.0, p.gather(1, ids))
    ids[gone] = -1
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, w)
    return w * scale, ids.to(torch.int32)
