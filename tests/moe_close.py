"""The experts' layer from its definition in 64 bits with a close bound, for inputs of random
signs.

A sum's error is the sum of its steps' roundings.  A step rounds the running sum, which for
terms of random signs is of the size of sqrt(sum of squares), not of the sum of magnitudes;
the kernels add 16 terms (tensor cores) or 8 of every 256 (a warp's lanes) a step, so n terms
are n / 16 steps, and 16 more for the parts, warps and scales that are added at the end.  Each
rounds (or truncates) by at most 2^-23 of what it holds:

    sum(n) = (n / 16 + 16) 2^-23 sqrt(sum of squares).

What is held as two bf16 values is off by at most 2^-17.  Errors of different columns are
independent and at most this large, so through a matrix they add by squares; of such a sum of
bounded errors four times the root of the squares is passed with a probability below
2 exp(-8) even if every one is of the full size (they are a third of it in the mean).  The
output's rounding to bf16 is half a step, 2^-8 of the value.  A quantised h may land on either
side of a border that its error reaches; these few are added by magnitude.

``fault`` plants a mistake in the 64-bit sums, so that a test can ask whether the bound would
notice it.
"""

from __future__ import annotations

import torch

import moe_ref

EPS = 2.0 ** -23
DTYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
FAULTS = ("x tail", "h tail", "h high only", "a pair", "u high only", "v high only")

SHAPES = [  # T, k, S, H, I: odd ones, and the forms with and without h and x on chip
    (1, 1, 1, 16, 16), (1, 8, 64, 2048, 768), (2, 2, 4, 512, 1024), (5, 3, 21, 1232, 416),
    (8, 4, 9, 48, 16), (9, 2, 5, 272, 2064), (16, 8, 128, 256, 64), (17, 5, 7, 144, 336),
    (32, 8, 40, 512, 96), (33, 1, 3, 96, 128), (70, 6, 30, 160, 48), (3, 32, 40, 64, 32),
    (16, 4, 10, 2064, 4096), (32, 8, 40, 160, 1040), (2, 2, 4, 1024, 14336),
    (1, 3, 3, 64, 32768), (16, 1, 3, 16384, 32),
    (4, 8, 32, 2048, 768), (8, 8, 64, 2048, 768), (16, 8, 48, 2048, 768), (32, 8, 24, 2048, 768)]
LORA_SHAPES = [  # T, k, S, H, I, L, r
    (1, 8, 64, 512, 192, 4, 16), (1, 1, 1, 16, 16, 1, 8), (11, 2, 13, 720, 208, 3, 8),
    (8, 4, 10, 256, 128, 9, 32), (20, 3, 6, 128, 80, 2, 24), (37, 2, 5, 96, 64, 5, 64),
    (3, 2, 4, 64, 48, 2, 256), (21, 4, 36, 480, 3184, 2, 8), (13, 8, 8, 736, 3936, 3, 256),
    (8, 8, 24, 2048, 768, 8, 32)]


def inputs(kind, T, k, S, H, I, L=0, r=0, device="cpu", seed=0):
    """Arguments of ``layer`` by name; every token has k different slots where there are as
    many."""
    g = torch.Generator(device=device).manual_seed(seed + 1000 * T + I)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device=device) * std).to(dtype)

    a = {"x": normal(T, H)}
    w = torch.rand(T, k, generator=g, device=device) + 0.05
    a["weights"] = w / w.sum(1, keepdim=True)
    a["ids"] = (torch.stack([torch.randperm(S, generator=g, device=device)[:k]
                             for _ in range(T)]) if S >= k else
                torch.randint(0, S, (T, k), generator=g, device=device)).to(torch.int32)
    for name, shape in (("13", (S, 2 * I, H)), ("2", (S, H, I))):
        if kind == "bf16":
            a["w" + name] = normal(*shape, std=0.05)
            a["s" + name] = None
            continue
        a["w" + name] = (torch.randint(-127, 128, shape, generator=g, device=device,
                                       dtype=torch.int8) if kind == "int8" else
                         normal(*shape, std=80.0, dtype=torch.float32).clamp(-448, 448).to(
                             torch.float8_e4m3fn))
        a["s" + name] = (torch.rand(S, shape[1], 1, generator=g, device=device) + 0.5) * 0.05 / 80
    if L:
        # (the adapters' part of a sum about as large as the experts')
        a["lora"] = (normal(L, S, 2 * r, H, std=0.05), normal(L, S, 2 * I, r, std=r ** -0.5),
                     normal(L, S, r, I, std=0.05), normal(L, S, H, r, std=2 * r ** -0.5),
                     torch.linspace(1.0, 2.0, L, device=device))
        a["adapter"] = torch.arange(T, dtype=torch.int32, device=device) % (L + 1) - 1
        a["adapter"][0] = 0
    return a


def _sum(n, w, v):
    """What the roundings of a sum of n terms w v amount to."""
    return (n / 16 + 16) * EPS * _root(w, v)


def _root(w, v):
    return ((w * w) @ (v * v)).sqrt()


def _high(v):
    return v.to(torch.bfloat16).double()


def layer(x, weights, ids, w13, w2, s13=None, s2=None, lora=None, adapter=None, fault=None):
    """(out, bound), both [T, H] in 64 bits."""
    (S, H, I), dtype, k = w2.shape, w13.dtype, ids.size(1)
    quantised = dtype in moe_ref.QMAX
    vec = 16 if quantised else 8
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    err, squares, flips = out.clone(), out.clone(), out.clone()
    for t, picks in enumerate(ids.tolist()):
        xt = x[t].double()
        cut = xt.clone()
        if fault == "x tail":
            cut[-vec:] = 0
        for j, s in enumerate(picks):
            if fault == "a pair" and t == len(ids) - 1 and j == k - 1:
                continue
            a, b = w13[s].double(), w2[s].double()
            if quantised:
                q, sc, _ = moe_ref.quantise(xt, dtype)
                q = torch.where(cut == xt, q, 0)
                a = a * s13[s].double().reshape(-1, 1)
                b = b * s2[s].double().reshape(-1, 1)
                gu = a @ (q * sc)
                d = 8 * EPS * gu.abs()
                if dtype != torch.int8:
                    d = d + _sum(H, a, q * sc)
            else:
                gu = a @ cut
                d = _sum(H, a, xt)
            n = -1 if lora is None else int(adapter[t])
            if n >= 0:
                a13, b13, a2, b2 = (m[n, s].double() for m in lora[:4])
                c, r = float(lora[4][n]), a2.size(0)
                u = a13 @ cut
                du = _sum(H, a13, xt) + (2.0 ** -17 + 2 * EPS) * u.abs()
                if fault == "u high only":
                    u = _high(c * u) / c
                for half in range(2):
                    rows, of = slice(half * I, (half + 1) * I), slice(half * r, (half + 1) * r)
                    gu[rows] += c * (b13[rows] @ u[of])
                    d[rows] += abs(c) * (_root(b13[rows], du[of]) + _sum(r, b13[rows], u[of]))
            g, up = gu[:I], gu[I:]
            act = g * torch.sigmoid(g)
            h = act * up
            # silu's slope is at most 1.1; expf, the division and three products: a few units
            dh = 1.1 * up.abs() * d[:I] + act.abs() * d[I:] + 16 * EPS * h.abs() + 1e-30
            wt = float(weights[t, j])
            if quantised:
                q, sc, top = moe_ref.quantise(h, dtype)
                off = 4 * dh.max() / top + 4 * EPS
                wide = 4 * dh + h.abs() * off
                near = [moe_ref.to_grid((h + side * wide) * moe_ref.QMAX[dtype] / top, dtype)
                        for side in (-1, 1)]
                dq = torch.maximum((near[0] - q).abs(), (near[1] - q).abs())
                held = q * sc
                y = b @ _without_tail(held, vec, fault)
                flips[t] += wt * (b.abs() @ (dq * sc) + off * y.abs())
                dy = torch.zeros_like(y)
            else:
                held = h
                dh = dh + 2.0 ** -17 * h.abs()
                y = b @ _without_tail(_high(wt * h) / wt if fault == "h high only" else h, vec, fault)
                dy = _root(b, dh)
            square = (b * b) @ (held * held)
            if n >= 0:
                v = a2 @ _without_tail(h, vec, fault)
                dv = _root(a2, dh) + _sum(I, a2, h) + (2.0 ** -17 + 2 * EPS) * v.abs()
                if fault == "v high only":
                    v = _high(c * wt * v) / (c * wt)
                y = y + c * (b2 @ v)
                dy = dy + abs(c) * (_root(b2, dv) + _sum(r, b2, v))
                square = square + c * c * ((b2 * b2) @ (v * v))
            out[t] += wt * y
            err[t] += (wt * dy) ** 2
            squares[t] += wt * wt * square
    err = 4 * (err.sqrt() + (I * k / 16 + 16) * EPS * squares.sqrt()) + flips
    return out, (1 + 2.0 ** -7) * err + 2.0 ** -8 * out.abs() + 1e-38


def _without_tail(h, vec, fault):
    if fault == "h tail":
        h = h.clone()
        h[-vec:] = 0
    return h


def worst(got, want, bound):
    return ((got.double() - want).abs() / bound).max().item()
