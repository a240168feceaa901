"""The cached MoE layer's operators: router, experts, experts with adapters.

The cache decides which experts are in its slots and brings them there; these operators do
the layer's arithmetic on them, for the few tokens of a decode step:

* :func:`route`         hidden states -> the k best experts of each token and their weights
                        (``expert_cache_route``);
* :func:`experts`       the routed experts' SwiGLU layer read straight from the slots
                        (``expert_cache_experts``): bf16 weights, or int8 / fp8 (e4m3)
                        weights with one scale per output row and activations quantised
                        per row;
* :func:`experts_lora`  the same with low-rank adapters of many requests beside the
                        experts' projections (``expert_cache_experts_lora``).

All run on the current stream of the tensors' device, allocate their outputs and workspace
from torch's caching allocator, read nothing back and can be captured into CUDA graphs.
``ExpertSlotCache.forward`` runs them as one cached step.  They have no counterpart in the
reference, which leaves the layer to vLLM's kernels (vllm_expert_cache/cache.py:118-163
ends with the gathered slots).
"""

from __future__ import annotations

import ctypes
import functools

import torch

from ._lib import lib

# Weight types of the C-ABI (EXPERT_CACHE_BF16 / _INT8 / _FP8).
WEIGHT_TYPES = {torch.bfloat16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}
SCORING = {"softmax": 0, "sigmoid": 1}
MAX_TOPK = 32           # EXPERT_CACHE_EXPERTS_MAX_TOPK
MAX_DIM = 32768         # EXPERT_CACHE_EXPERTS_MAX_DIM
MAX_SLOTS = 1024        # EXPERT_CACHE_MAX_SLOTS
MAX_RANK = 256          # EXPERT_CACHE_LORA_MAX_RANK


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, x on {device}")


def _rows(x: torch.Tensor, name: str = "x") -> torch.Tensor:
    """x as the kernels read it: bf16 rows of unit inner stride, 16-byte aligned."""
    _need(x.dim() == 2 and x.dtype == torch.bfloat16,
          f"{name} must be a 2-D bf16 tensor, not {tuple(x.shape)} {x.dtype}")
    if x.stride(1) != 1 or x.stride(0) % 8 or x.stride(0) < x.size(1) or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _call(device, fn, *args) -> None:
    """`fn(*args, stream)` on the current stream of `device`."""
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise RuntimeError(f"{fn.__name__} failed rc={rc}")


def route(x: torch.Tensor, gate_w: torch.Tensor, k: int, *, scoring: str = "softmax",
          renormalize: bool = True, bias: torch.Tensor | None = None,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The k best of E experts for each row of ``x`` [T, H] under the router's weight
    ``gate_w`` [E, H] (both bf16): ``(weights, ids)``, fp32 and int32 [T, k], best first.

    ``scoring`` "softmax" takes the softmax over all experts; "sigmoid" takes each score's
    sigmoid and picks by sigmoid + ``bias`` (fp32 [E], optional).  ``renormalize`` divides a
    row's weights by their sum; ``scale`` multiplies them.  Scores are summed in 64 bits and
    ties go to the lower id, so the choice is the same whatever the order of a sum.  NaN
    scores are never picked; a row with fewer than k others ends in id -1, weight 0.
    """
    _need(scoring in SCORING, f"scoring must be one of {sorted(SCORING)}, not {scoring!r}")
    _need(x.is_cuda, "x must be on a GPU")
    _need(gate_w.dim() == 2 and gate_w.dtype == torch.bfloat16 and gate_w.is_contiguous(),
          "gate_w must be a contiguous 2-D bf16 tensor")
    _on(x.device, gate_w=gate_w, bias=bias)
    x = _rows(x)
    (T, H), E = x.shape, gate_w.size(0)
    _need(gate_w.size(1) == H, f"gate_w has {gate_w.size(1)} columns, x {H}")
    _need(H % 8 == 0 and 0 < H <= 16384, f"hidden size {H} is not a multiple of 8 in [8, 16384]")
    _need(0 < E <= 2048, f"{E} experts: 1 to 2048 are supported")
    _need(1 <= k <= min(E, MAX_TOPK), f"k={k} of {E} experts: 1 to {min(E, MAX_TOPK)}")
    _need(gate_w.data_ptr() % 16 == 0, "gate_w is not 16-byte aligned")
    if bias is not None:
        _need(scoring == "sigmoid", "a selection bias needs scoring='sigmoid'")
        _need(bias.shape == (E,) and bias.dtype == torch.float32 and bias.is_contiguous(),
              f"bias must be a contiguous fp32 [{E}] tensor")
    weights = torch.empty((T, k), dtype=torch.float32, device=x.device)
    ids = torch.empty((T, k), dtype=torch.int32, device=x.device)
    _call(x.device, lib().expert_cache_route, x.data_ptr(), T, x.stride(0), H,
          gate_w.data_ptr(), E, k, SCORING[scoring], int(renormalize),
          None if bias is None else bias.data_ptr(), float(scale), weights.data_ptr(),
          ids.data_ptr())
    return weights, ids


@functools.lru_cache(maxsize=256)
def workspace_bytes(T: int, k: int, H: int, I: int, wtype: int, r: int = 0) -> int:
    """Device workspace of one call (``expert_cache_experts_workspace``)."""
    n = ctypes.c_long()
    rc = lib().expert_cache_experts_workspace(T, k, H, I, wtype, r, ctypes.byref(n))
    _need(rc == 0, f"unsupported sizes: T={T} k={k} H={H} I={I} wtype={wtype} r={r}")
    return n.value


def _scale(scale: torch.Tensor | None, S: int, n: int, name: str):
    if scale is None:
        raise ValueError(f"8-bit weights need {name}")
    _need(scale.dtype == torch.float32 and scale.is_contiguous()
          and scale.shape in ((S, n), (S, n, 1)),
          f"{name} must be contiguous fp32 [{S}, {n}] or [{S}, {n}, 1], not "
          f"{tuple(scale.shape)} {scale.dtype}")
    return scale.data_ptr()


def _layer_args(x, topk_weights, topk_ids, w13, w2, w13_scale, w2_scale, expert_map):
    """Checked arguments of both experts entry points up to I; and the tensors that they
    point into (a converted copy has to live until the launch is enqueued)."""
    _need(x.is_cuda, "x must be on a GPU")
    device = x.device
    _on(device, topk_weights=topk_weights, topk_ids=topk_ids, w13=w13, w2=w2,
        w13_scale=w13_scale, w2_scale=w2_scale, expert_map=expert_map)
    x = _rows(x)
    T, H = x.shape
    wtype = WEIGHT_TYPES.get(w13.dtype)
    _need(wtype is not None and w2.dtype == w13.dtype,
          f"weights must both be bf16, int8 or float8_e4m3fn, not {w13.dtype} and {w2.dtype}")
    _need(w13.dim() == 3 and w2.dim() == 3, "w13 and w2 must be 3-D")
    S, I = w2.size(0), w2.size(2)
    _need(w13.shape == (S, 2 * I, H) and w2.shape == (S, H, I),
          f"w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} are not [S, 2I, H] and [S, H, I] "
          f"for H={H}")
    _need(w13.is_contiguous() and w2.is_contiguous(), "w13 and w2 must be contiguous")
    _need(not (w13.data_ptr() | w2.data_ptr()) & 15, "w13 and w2 must be 16-byte aligned")
    vec = 16 if wtype else 8
    _need(H % vec == 0 and I % vec == 0 and 0 < H <= MAX_DIM and 0 < I <= MAX_DIM,
          f"H={H} and I={I} must be multiples of {vec} up to {MAX_DIM}")
    _need(0 < S <= MAX_SLOTS, f"{S} slots: 1 to {MAX_SLOTS} are supported")
    if wtype:
        s13 = _scale(w13_scale, S, 2 * I, "w13_scale")
        s2 = _scale(w2_scale, S, H, "w2_scale")
    else:
        _need(w13_scale is None and w2_scale is None, "bf16 weights take no scales")
        s13 = s2 = None
    _need(topk_ids.dim() == 2 and topk_ids.size(0) == T
          and topk_ids.dtype in (torch.int32, torch.int64),
          f"topk_ids must be int32 or int64 [{T}, k], not {tuple(topk_ids.shape)} "
          f"{topk_ids.dtype}")
    k = topk_ids.size(1)
    _need(1 <= k <= MAX_TOPK, f"k={k}: 1 to {MAX_TOPK} are supported")
    _need(topk_weights.shape == topk_ids.shape and topk_weights.is_floating_point(),
          f"topk_weights must be floating point [{T}, {k}], not {tuple(topk_weights.shape)} "
          f"{topk_weights.dtype}")
    if topk_ids.dtype != torch.int32:
        # ids outside int32 must stay out of range, not wrap into it
        topk_ids = topk_ids.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    if not topk_ids.is_contiguous():
        topk_ids = topk_ids.contiguous()
    if topk_weights.dtype != torch.float32 or not topk_weights.is_contiguous():
        topk_weights = topk_weights.to(torch.float32).contiguous()
    if expert_map is not None:
        _need(expert_map.dim() == 1 and expert_map.dtype == torch.int32
              and expert_map.is_contiguous() and expert_map.numel() > 0,
              "expert_map must be a contiguous, non-empty int32 vector")
    args = (x.data_ptr(), T, x.stride(0), H, topk_ids.data_ptr(), topk_weights.data_ptr(), k,
            None if expert_map is None else expert_map.data_ptr(),
            0 if expert_map is None else expert_map.numel(), w13.data_ptr(), s13,
            w2.data_ptr(), s2, wtype, S, I)
    return args, (x, topk_ids, topk_weights)


def _finish(fn, x, args, more, r):
    T, H, k, wtype, I = x.size(0), x.size(1), args[6], args[13], args[15]
    out = torch.empty((T, H), dtype=torch.bfloat16, device=x.device)
    nbytes = workspace_bytes(T, k, H, I, wtype, r)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=x.device)
    _call(x.device, fn, *args, *more, out.data_ptr(), H, ws.data_ptr(), nbytes)
    return out


def experts(x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
            w13: torch.Tensor, w2: torch.Tensor, *, w13_scale: torch.Tensor | None = None,
            w2_scale: torch.Tensor | None = None,
            expert_map: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = sum_j topk_weights[t, j] * W2[s] (silu(G) * U)`` with
    ``[G; U] = W13[s] x[t]``, bf16 [T, H].

    ``x`` bf16 [T, H]; ``topk_ids`` and ``topk_weights`` [T, k]; ``w13`` [S, 2I, H] (gate
    rows, then up rows) and ``w2`` [S, H, I] are slot buffers (bf16, or int8 / float8_e4m3fn
    with fp32 scales per output row).  ``s`` is the id itself, or ``expert_map[id]`` (a
    cache's ``table`` with expert ids, the composed map of ``refresh_ep`` with global ids).
    An id or slot out of range adds nothing, so padded rows carry -1 and give zeros.
    """
    args, keep = _layer_args(x, topk_weights, topk_ids, w13, w2, w13_scale, w2_scale,
                             expert_map)
    return _finish(lib().expert_cache_experts, keep[0], args, (), 0)


def experts_lora(x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                 w13: torch.Tensor, w2: torch.Tensor, a13: torch.Tensor, b13: torch.Tensor,
                 a2: torch.Tensor, b2: torch.Tensor, scaling: torch.Tensor,
                 adapter: torch.Tensor, *, w13_scale: torch.Tensor | None = None,
                 w2_scale: torch.Tensor | None = None,
                 expert_map: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`experts` with low-rank adapters of many requests.

    ``adapter`` [T] (int32) names each token's adapter, -1 for none.  The L adapters' bf16
    matrices are held per expert, ``a13`` [L, E, 2r, H] (the gate's r rows, then the up
    projection's), ``b13`` [L, E, 2I, r], ``a2`` [L, E, r, I], ``b2`` [L, E, H, r], and are
    indexed by ``topk_ids`` as given, before ``expert_map``: with a cache's ``table`` as the
    map an adapter follows its expert through the slots without being moved.  ``scaling``
    is fp32 [L].
    """
    args, keep = _layer_args(x, topk_weights, topk_ids, w13, w2, w13_scale, w2_scale,
                             expert_map)
    x = keep[0]
    T, H, I = x.size(0), x.size(1), args[15]
    _on(x.device, a13=a13, b13=b13, a2=a2, b2=b2, scaling=scaling, adapter=adapter)
    _need(a13.dim() == 4 and a2.dim() == 4, "adapter matrices must be 4-D")
    L, E, r = a13.size(0), a13.size(1), a2.size(2)
    _need(L > 0 and E > 0 and r % 8 == 0 and 0 < r <= MAX_RANK,
          f"L={L} adapters, E={E} experts, rank {r}: the rank must be a multiple of 8 up to "
          f"{MAX_RANK}")
    for name, t, shape in (("a13", a13, (L, E, 2 * r, H)), ("b13", b13, (L, E, 2 * I, r)),
                           ("a2", a2, (L, E, r, I)), ("b2", b2, (L, E, H, r))):
        _need(t.shape == shape and t.dtype == torch.bfloat16 and t.is_contiguous()
              and t.data_ptr() % 16 == 0,
              f"{name} must be contiguous, 16-byte aligned bf16 {shape}, not "
              f"{tuple(t.shape)} {t.dtype}")
    _need(scaling.shape == (L,) and scaling.dtype == torch.float32 and scaling.is_contiguous(),
          f"scaling must be contiguous fp32 [{L}]")
    _need(adapter.shape == (T,) and adapter.dtype == torch.int32 and adapter.is_contiguous(),
          f"adapter must be contiguous int32 [{T}]")
    more = (adapter.data_ptr(), a13.data_ptr(), b13.data_ptr(), a2.data_ptr(), b2.data_ptr(),
            scaling.data_ptr(), L, E, r)
    return _finish(lib().expert_cache_experts_lora, x, args, more, r)
