"""Measured cases of the cached MoE layer's operators, with their plain forms.

Three operators of ``vllm_expert_cache.moe``, on the sizes that a cached step meets:

* ``experts``       a whole MoE layer for a few tokens, read from the cache's slots:
                    out[t] = sum_j w[t,j] * W2[s] (silu(G) * U),  [G; U] = W13[s] x[t],
                    s the slot of the token's j-th expert.  Weights in bf16, or in int8 or
                    e4m3 with one scale per output row and the activations quantised per
                    row: q(v) = round(v * Q / max|v|), scale max|v| / Q, Q = 127 or 448.
* ``experts_lora``  the same layer with low-rank adapters of many requests beside the
                    experts' shared projections: token t of adapter a and expert e adds
                    c_a B13[a,e] (A13[a,e] x[t]) to [G; U] and c_a B2[a,e] (A2[a,e] h) to
                    the expert's output (the unquantised x and h).
* ``route``         the router: scores of all experts, the k best per token (ties to the
                    lowest expert id) and their weights.

``run`` computes them in elementary torch operations while ``own`` is false and calls the
framework's kernels while it is true.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
_QMAX = {"int8": 127.0, "fp8": 448.0}


# ---------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # one token of the 30B-A3B shape, W8A8, half of the 128 experts resident: the call
        # that a decode step at batch 1 makes once a layer, where latency counts
        _experts("experts-int8-1", "int8", T=1, k=8, S=64, D=8, H=2048, I=768),
        # the same token in bf16: twice the bytes
        _experts("experts-bf16-1", "bf16", T=1, k=8, S=64, D=8, H=2048, I=768),
        # eight decoding requests of one tensor-parallel rank (half of the 235B shape's
        # expert width), fp8, the smallest cache that a step of this width fits
        _experts("experts-fp8-8", "fp8", T=8, k=8, S=64, D=44, H=4096, I=768),
        # sixteen requests, every slot of a full cache routed; two rows are batch padding
        _experts("experts-int8-16", "int8", T=16, k=8, S=128, D=96, H=2048, I=768, pad=2),
        # two tokens of the 8x7B shape in bf16: few experts, each of 352 MB (the largest)
        _experts("experts-bf16-wide", "bf16", T=2, k=2, S=4, D=4, H=4096, I=14336),
        # odd sizes, expert parallel: some routed experts are another rank's
        _experts("experts-bf16-odd", "bf16", T=5, k=3, S=21, D=7, H=1224, I=408, ep=True),
        # one request with an adapter
        _experts("lora-bf16-1", "bf16", T=1, k=8, S=64, D=8, H=2048, I=768, L=4, r=16),
        # eight requests with adapters of their own beside int8 experts
        _experts("lora-int8-8", "int8", T=8, k=8, S=64, D=44, H=2048, I=768, L=8, r=32),
        # odd sizes, requests without an adapter among them
        _experts("lora-bf16-odd", "bf16", T=11, k=2, S=13, D=9, H=712, I=200, pad=1, L=3,
                 r=8),
        # the router of the 30B-A3B shape at batch 1
        _route("route-softmax-1", T=1, E=128, k=8, H=2048, scoring="softmax"),
        # sixteen requests, sigmoid scores with a selection bias
        _route("route-sigmoid-16", T=16, E=256, k=8, H=4096, scoring="sigmoid"),
        # odd sizes
        _route("route-softmax-odd", T=53, E=61, k=5, H=1000, scoring="softmax"),
    ]


def _experts(name, wtype, T, k, S, D, H, I, pad=0, ep=False, L=0, r=0):
    """T tokens (the last `pad` of them batch padding, ids -1) of k experts over S slots, D
    of them routed to; L adapters of rank r (0: none)."""
    return {"name": name, "kind": "lora" if L else "experts", "wtype": wtype, "T": T, "k": k,
            "S": S, "D": D, "H": H, "I": I, "pad": pad, "ep": ep, "L": L, "r": r}


def _route(name, T, E, k, H, scoring):
    return {"name": name, "kind": "route", "T": T, "E": E, "k": k, "H": H,
            "scoring": scoring}


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi, max(lo, round(v / step) * step))


def draw(rng):
    if rng.random() < 0.25:
        E = _log(rng, 4, 512)
        case = _route(None, T=_log(rng, 1, 64), E=E, k=rng.randint(1, min(10, E)),
                      H=_log(rng, 64, 8192, 8), scoring=rng.choice(["softmax", "sigmoid"]))
    else:
        wtype = rng.choice(["bf16", "int8", "fp8"])
        step = 8 if wtype == "bf16" else 16
        T = _log(rng, 1, 32)
        k = rng.randint(1, 8)
        pad = rng.choice([0, 0, 1]) if T > 1 else 0
        S = max(k, _log(rng, 2, 128))
        D = max(k, min(S, round((T - pad) * k * rng.uniform(0.4, 1.0))))
        lora = rng.random() < 0.4
        H, I = _log(rng, 256, 4096, step), _log(rng, 128, 4096, step)
        # as many bytes as the largest listed case at most, and no more than the adapters
        # and the plain forms' fp32 copies of every routed expert leave room for
        while 12 * T * k * H * I > 6e9 or 3 * S * H * I > 7e8:
            I = max(128, I // 2 // step * step)
        L = rng.randint(1, 8) if lora else 0
        case = _experts(None, wtype, T=T, k=k, S=S, D=D, H=H, I=I, pad=pad,
                        ep=not lora and rng.random() < 0.3, L=L,
                        r=rng.choice([8, 16, 24, 32, 64]) if lora else 0)
        while 4 * case["L"] * S * case["r"] * 3 * (H + I) > 2e9:   # the adapters' bytes
            case["L"], case["r"] = max(1, case["L"] // 2), 8
    del case["name"]
    return case


def work(case):
    T, k, H = case["T"], case["k"], case["H"]
    if case["kind"] == "route":
        E = case["E"]
        bias = 4 * E if case["scoring"] == "sigmoid" else 0
        return {"bytes": 2 * (T + E) * H + bias + 8 * T * k, "flops": 2 * T * E * H}
    I, D, r = case["I"], case["D"], case["r"]
    item = 2 if case["wtype"] == "bf16" else 1
    scales = 0 if case["wtype"] == "bf16" else 4 * (2 * I + H)
    pairs = (T - case["pad"]) * k
    b = D * (3 * H * I * item + scales) + 4 * T * H + 8 * T * k
    f = 2 * pairs * 3 * H * I
    if case["L"]:
        with_adapter = _adapted(case) * k       # (adapter, expert) pairs
        b += with_adapter * 2 * r * (3 * H + 3 * I) + 4 * T
        f += with_adapter * 2 * r * (3 * H + 3 * I)
    return {"bytes": b, "flops": f}


def _adapted(case):
    """Tokens with an adapter: every one, but for each fifth of a batch."""
    n = case["T"] - case["pad"]
    return n - n // 5


# ---------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = torch.Generator().manual_seed(seed + 1)
    T, k, H = case["T"], case["k"], case["H"]

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype).mul_(std)

    s = {"case": case, "x": normal(T, H)}
    if case["kind"] == "route":
        s["gate_w"] = normal(case["E"], H, std=0.02)
        s["bias"] = (normal(case["E"], std=0.1, dtype=torch.float32)
                     if case["scoring"] == "sigmoid" else None)
        return s

    S, I, D, wtype = case["S"], case["I"], case["D"], case["wtype"]
    if wtype == "bf16":
        s["w13"], s["w2"] = normal(S, 2 * I, H, std=0.02), normal(S, H, I, std=0.02)
        s["s13"] = s["s2"] = None
    else:
        spread = 32.0 if wtype == "int8" else 100.0
        for name, shape in (("13", (S, 2 * I, H)), ("2", (S, H, I))):
            q = normal(*shape, std=spread).clamp_(-_QMAX[wtype], _QMAX[wtype])
            s["w" + name] = (q.round_().to(torch.int8) if wtype == "int8"
                             else q.to(torch.float8_e4m3fn))
            s["s" + name] = (torch.rand((S, shape[1], 1), generator=g, device=DEV) + 0.5
                             ).mul_(0.02 / spread)

    # Routing: the first tokens walk through the D routed slots, the others draw from them;
    # ids are experts of a layer with twice as many experts as slots, and a table (or, for
    # an expert-parallel layer, the composed map) takes them to slots.
    E = 2 * S
    experts = torch.randperm(E, generator=c)
    table = torch.full((E,), -1, dtype=torch.int32)
    table[experts[:S]] = torch.randperm(S, generator=c).to(torch.int32)
    n = T - case["pad"]
    ids = torch.full((T, k), -1, dtype=torch.int64)
    for t in range(n):
        if t * k < D:
            pick = (torch.arange(k) + t * k) % D
        else:
            pick = torch.randperm(D, generator=c)[:k]
        ids[t] = experts[pick]
        if case["ep"] and t * k >= D:        # another rank's experts: not in the map
            other = torch.rand(k, generator=c) < 0.5
            ids[t][other] = experts[S + torch.randperm(S, generator=c)[:k]][other]
    w = torch.rand(T, k, generator=c) + 0.05
    s["ids"] = ids.to(torch.int32).to(DEV)
    s["table"] = table.to(DEV)
    s["weights"] = (w / w.sum(1, keepdim=True)).to(DEV)

    if case["L"]:
        L, r = case["L"], case["r"]
        s["a13"], s["b13"] = normal(L, E, 2 * r, H, std=0.02), normal(L, E, 2 * I, r, std=0.02)
        s["a2"], s["b2"] = normal(L, E, r, I, std=0.02), normal(L, E, H, r, std=0.02)
        s["scaling"] = torch.full((L,), 2.0, device=DEV)
        a = torch.arange(T) % L
        a[_adapted(case):] = -1
        s["adapter"] = a[torch.randperm(n, generator=c).tolist() + list(range(n, T))].to(
            torch.int32).to(DEV)
    return s


# ---------------------------------------------------------------------------------------
# one pass

def run(s):
    if own:
        moe = _moe()
        if s["case"]["kind"] == "route":
            return moe.route(s["x"], s["gate_w"], s["case"]["k"], scoring=s["case"]["scoring"],
                             bias=s["bias"])
        args = (s["x"], s["weights"], s["ids"], s["w13"], s["w2"])
        scales = {"w13_scale": s["s13"], "w2_scale": s["s2"], "expert_map": s["table"]}
        if s["case"]["kind"] == "experts":
            return moe.experts(*args, **scales)
        return moe.experts_lora(*args, s["a13"], s["b13"], s["a2"], s["b2"], s["scaling"],
                                s["adapter"], **scales)
    return _plain_route(s) if s["case"]["kind"] == "route" else _plain_experts(s)


def _moe():
    root = str(Path(__file__).resolve().parents[1] / "vllm-expert-cache_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from vllm_expert_cache import moe
    return moe


def _plain_route(s):
    """Scores in 64 bits: which expert is the k-th best hangs on the last bits."""
    logits = s["x"].double() @ s["gate_w"].double().T
    if s["case"]["scoring"] == "softmax":
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
        order = logits
    else:
        score = 1.0 / (1.0 + torch.exp(-logits))
        order = score + s["bias"].double()
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :s["case"]["k"]]
    w = score.gather(1, ids)
    w = w / w.sum(1, keepdim=True)
    return w.float(), ids.to(torch.int32)


def _quantised(v, wtype):
    """(quantised values as fp32, scale per row) of fp32 rows."""
    top = v.abs().amax(-1, keepdim=True).clamp_min(1e-10)
    q = v * _QMAX[wtype] / top
    q = q.round() if wtype == "int8" else q.to(torch.float8_e4m3fn).float()
    return q, top / _QMAX[wtype]


def _plain_experts(s):
    case = s["case"]
    T, k, I, wtype, r = case["T"], case["k"], case["I"], case["wtype"], case["r"]
    ids = s["ids"].long().reshape(-1)
    slots = torch.where(ids >= 0, s["table"].long()[ids.clamp_min(0)], -1)
    here = slots >= 0
    at = slots.clamp_min(0)
    x = s["x"].float().repeat_interleave(k, 0)                     # a row for each pair
    gu = _project(x, s["w13"], s["s13"], at, wtype)
    if r:
        a = s["adapter"].long().repeat_interleave(k)
        add = s["scaling"][a.clamp_min(0)].mul(a >= 0).unsqueeze(1)
        pick = (a.clamp_min(0), ids.clamp_min(0))
        u = _product(s["a13"][pick].float(), x).unflatten(1, (2, r))
        b = s["b13"][pick].float().unflatten(1, (2, I))
        gu = gu + add * (b * u.unsqueeze(2)).sum(-1).flatten(1)
    gate, up = gu[:, :I], gu[:, I:]
    h = gate / (1.0 + torch.exp(-gate)) * up
    y = _project(h, s["w2"], s["s2"], at, wtype)
    if r:
        v = _product(s["a2"][pick].float(), h)
        y = y + add * _product(s["b2"][pick].float(), v)
    y = torch.where(here.unsqueeze(1), y * s["weights"].reshape(-1, 1), 0.0)
    return y.unflatten(0, (T, k)).sum(1).to(s["x"].dtype)


def _product(w, v):
    """w [n, rows, cols] by v [n, cols], row by row of n."""
    return torch.bmm(w, v.unsqueeze(2)).squeeze(2)


def _project(v, w, scale, at, wtype):
    if wtype == "bf16":
        return _product(w[at].float(), v)
    q, top = _quantised(v, wtype)
    return _product(w[at].float(), q) * top * scale[at].squeeze(2)


# ---------------------------------------------------------------------------------------
# in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    k = case["k"]
    if case["kind"] == "route":
        x, g = s["x"].double(), s["gate_w"].double()
        z = (x[:, None, :] * g[None, :, :]).sum(-1) if x.size(0) * g.numel() < 5e8 else \
            torch.einsum("th,eh->te", x, g)
        if case["scoring"] == "softmax":
            p = torch.softmax(z, 1)
            key = p
        else:
            p = torch.sigmoid(z)
            key = p + s["bias"].double()
        ids = torch.argsort(-key, dim=1, stable=True)[:, :k]
        w = torch.take_along_dim(p, ids, 1)
        return (w / w.sum(1, keepdim=True)), ids.to(torch.int32)

    def rows(w, scale, v):
        """w v for one expert's matrix, v quantised where w is."""
        if case["wtype"] == "bf16":
            return w.double() @ v
        m = max(float(v.abs().max()), 1e-10)
        q = v * _QMAX[case["wtype"]] / m
        q = torch.round(q) if case["wtype"] == "int8" else \
            q.to(torch.float8_e4m3fn).double()
        return (w.double() @ q) * (m / _QMAX[case["wtype"]]) * scale.double().reshape(-1)

    I, r = case["I"], case["r"]
    out = torch.zeros_like(s["x"], dtype=torch.float64)
    table = s["table"].tolist()
    for t, picks in enumerate(s["ids"].tolist()):
        x = s["x"][t].double()
        for j, e in enumerate(picks):
            slot = table[e] if e >= 0 else -1
            if slot < 0:
                continue
            scale = lambda n: None if s[n] is None else s[n][slot]  # noqa: E731
            gu = rows(s["w13"][slot], scale("s13"), x)
            a = int(s["adapter"][t]) if r else -1
            if a >= 0:
                c = float(s["scaling"][a])
                u = s["a13"][a, e].double() @ x
                gu[:I] += c * (s["b13"][a, e, :I].double() @ u[:r])
                gu[I:] += c * (s["b13"][a, e, I:].double() @ u[r:])
            h = gu[:I] * torch.sigmoid(gu[:I]) * gu[I:]
            y = rows(s["w2"][slot], scale("s2"), h)
            if a >= 0:
                y += c * (s["b2"][a, e].double() @ (s["a2"][a, e].double() @ h))
            out[t] += float(s["weights"][t, j]) * y
    return out
