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
They serve only: none has a backward pass, and their results carry no gradient.
``ExpertSlotCache.forward`` runs them as one cached step.  They have no counterpart in the
reference, which leaves the layer to vLLM's kernels (vllm_expert_cache/cache.py:118-163
ends with the gathered slots).

A layer's kernels take some 15 us for one token, so a call's checks are written to be cheap:
plain comparisons, with the message put together only where one fails.
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
MAX_HIDDEN = 16384      # EXPERT_CACHE_PREGATE_MAX_HIDDEN
MAX_EXPERTS = 2048      # EXPERT_CACHE_PREGATE_MAX_EXPERTS
# Steps up to this many tokens (one column tile of the experts' kernels) are as fast on them as on
# vLLM's Triton kernel or faster, 1.0 to 1.9 times (bf16 and e4m3, ten shapes of 1 to 10 experts a
# token, experts of 3 to 352 MB, vLLM's configuration for the number of slots, which is its
# default one).  With 9 to 16 tokens it was 0.6 to 1.2 times, with 17 to 32 0.3 to 0.97 times, with
# 33 to 96 0.4 to 0.8 times.
STEP_TOKENS = 8
MAX_INT = 2 ** 31 - 1   # the C-ABI's int: ctypes cuts what is larger to 32 bits

_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
# The current stream's handle without building a Stream object (2 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _is(t: torch.Tensor) -> str:
    return f"{tuple(t.shape)} {t.dtype} on {t.device}"


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as the kernels read it: bf16 rows of unit inner stride, 16-byte aligned."""
    if x.dtype is not _BF16 or x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"x must be a 2-D bf16 tensor on a GPU, not {_is(x)}")
    if x.size(0) > MAX_INT:
        raise ValueError(f"{x.size(0)} rows of x: up to {MAX_INT} are supported")
    row = x.stride(0)
    if x.stride(1) != 1 or row % 8 or not x.size(1) <= row <= MAX_INT or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _call(index: int, fn, *args) -> None:
    """`fn(*args, stream)` on the current stream of GPU `index`."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise RuntimeError(f"{fn.__name__} failed rc={rc}")


def _row_stride(x: torch.Tensor) -> int:
    # (a tensor of one row or none may carry any stride)
    return x.stride(0) if x.size(0) > 1 else (x.size(1) + 7) // 8 * 8


def route(x: torch.Tensor, gate_w: torch.Tensor, k: int, *, scoring: str = "softmax",
          renormalize: bool = True, bias: torch.Tensor | None = None,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The k best of E experts for each row of ``x`` [T, H] under the router's weight
    ``gate_w`` [E, H] (both bf16): ``(weights, ids)``, fp32 and int32 [T, k], best first.

    ``scoring`` "softmax" takes the softmax over all experts; "sigmoid" takes each score's
    sigmoid and picks by sigmoid + ``bias`` (fp32 [E], optional).  ``renormalize`` divides a
    row's weights by their sum; ``scale`` multiplies them.  Scores are summed in 64 bits, in
    one order whatever the batch, and ties go to the lower id.  NaN scores are never picked; a
    row with fewer than k others ends in id -1, weight 0.
    """
    mode = SCORING.get(scoring)
    if mode is None:
        raise ValueError(f"scoring must be one of {sorted(SCORING)}, not {scoring!r}")
    x = _rows(x)
    T, H = x.shape
    index = x.get_device()
    if gate_w.dim() != 2 or gate_w.dtype is not _BF16 or not gate_w.is_contiguous() \
            or gate_w.get_device() != index or gate_w.size(1) != H or gate_w.data_ptr() % 16:
        raise ValueError(f"gate_w must be a contiguous, 16-byte aligned bf16 [E, {H}] tensor "
                         f"beside x, not {_is(gate_w)}")
    E = gate_w.size(0)
    if H % 8 or not 0 < H <= MAX_HIDDEN:
        raise ValueError(f"hidden size {H} is not a multiple of 8 up to {MAX_HIDDEN}")
    if not 0 < E <= MAX_EXPERTS:
        raise ValueError(f"{E} experts: 1 to {MAX_EXPERTS} are supported")
    if not 1 <= k <= min(E, MAX_TOPK):
        raise ValueError(f"k={k} of {E} experts: 1 to {min(E, MAX_TOPK)} are supported")
    at_bias = None
    if bias is not None:
        if mode != 1:
            raise ValueError("a selection bias needs scoring='sigmoid'")
        if bias.dim() != 1 or bias.size(0) != E or bias.dtype is not _F32 \
                or not bias.is_contiguous() or bias.get_device() != index:
            raise ValueError(f"bias must be a contiguous fp32 [{E}] tensor beside x, not "
                             f"{_is(bias)}")
        at_bias = bias.data_ptr()
    weights = x.new_empty((T, k), dtype=_F32)
    ids = x.new_empty((T, k), dtype=_I32)
    _call(index, lib().expert_cache_route, x.data_ptr(), T, _row_stride(x), H,
          gate_w.data_ptr(), E, k, mode, int(renormalize), at_bias, scale,
          weights.data_ptr(), ids.data_ptr())
    return weights, ids


@functools.lru_cache(maxsize=256)
def workspace_bytes(T: int, k: int, H: int, I: int, wtype: int, r: int = 0) -> int:
    """Device workspace of one call (``expert_cache_experts_workspace``)."""
    n = ctypes.c_long()
    rc = lib().expert_cache_experts_workspace(T, k, H, I, wtype, r, ctypes.byref(n))
    if rc != 0:
        raise ValueError(f"unsupported sizes: T={T} k={k} H={H} I={I} wtype={wtype} r={r}")
    return n.value


def _scale(scale: torch.Tensor | None, S: int, n: int, name: str, index: int) -> int:
    if scale is None:
        raise ValueError(f"8-bit weights need {name}")
    if scale.dtype is not _F32 or scale.shape not in ((S, n, 1), (S, n)) \
            or not scale.is_contiguous() or scale.get_device() != index:
        raise ValueError(f"{name} must be contiguous fp32 [{S}, {n}] or [{S}, {n}, 1] beside "
                         f"x, not {_is(scale)}")
    return scale.data_ptr()


def _layer(fn, x, topk_weights, topk_ids, w13, w2, w13_scale, w2_scale, expert_map,
           adapters=None):
    """Checks and the call of both experts entry points."""
    x = _rows(x)
    T, H = x.shape
    index = x.get_device()
    dtype = w13.dtype
    wtype = WEIGHT_TYPES.get(dtype)
    if wtype is None or w2.dtype is not dtype:
        raise ValueError("w13 and w2 must both be bf16, int8 or float8_e4m3fn, not "
                         f"{dtype} and {w2.dtype}")
    if w2.dim() != 3:
        raise ValueError(f"w13 and w2 must be 3-D, not {_is(w13)} and {_is(w2)}")
    S, rows, I = w2.shape
    if rows != H or w13.shape != (S, 2 * I, H):
        raise ValueError(f"w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} are not [S, 2I, H] "
                         f"and [S, H, I] for H={H}")
    at13, at2 = w13.data_ptr(), w2.data_ptr()
    if (at13 | at2) & 15 or not w13.is_contiguous() or not w2.is_contiguous() \
            or w13.get_device() != index or w2.get_device() != index:
        raise ValueError("w13 and w2 must be contiguous, 16-byte aligned and beside x on "
                         f"GPU {index}")
    vec = 16 if wtype else 8
    if H % vec or I % vec or not 0 < H <= MAX_DIM or not 0 < I <= MAX_DIM:
        raise ValueError(f"H={H} and I={I} must be multiples of {vec} up to {MAX_DIM}")
    if not 0 < S <= MAX_SLOTS:
        raise ValueError(f"{S} slots: 1 to {MAX_SLOTS} are supported")
    if wtype:
        s13 = _scale(w13_scale, S, 2 * I, "w13_scale", index)
        s2 = _scale(w2_scale, S, H, "w2_scale", index)
    else:
        if w13_scale is not None or w2_scale is not None:
            raise ValueError("bf16 weights take no scales")
        s13 = s2 = None
    ids, weights = topk_ids, topk_weights
    shape = ids.shape
    if len(shape) != 2 or shape[0] != T or ids.get_device() != index \
            or ids.dtype not in (_I32, _I64):
        raise ValueError(f"topk_ids must be int32 or int64 [{T}, k] beside x, not {_is(ids)}")
    k = shape[1]
    if not 1 <= k <= MAX_TOPK:
        raise ValueError(f"k={k}: 1 to {MAX_TOPK} are supported")
    if weights.shape != shape or weights.get_device() != index \
            or not weights.is_floating_point():
        raise ValueError(f"topk_weights must be floating point [{T}, {k}] beside x, not "
                         f"{_is(weights)}")
    if ids.dtype is not _I32:
        # ids outside int32 must stay out of range, not wrap into it
        ids = ids.clamp(-1, 2 ** 31 - 1).to(_I32)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if weights.dtype is not _F32 or not weights.is_contiguous():
        weights = weights.to(_F32).contiguous()
    at_map = n_map = 0
    if expert_map is not None:
        n_map = expert_map.numel()
        if expert_map.dtype is not _I32 or not 0 < n_map <= MAX_INT or expert_map.dim() != 1 \
                or not expert_map.is_contiguous() or expert_map.get_device() != index:
            raise ValueError("expert_map must be a contiguous, non-empty int32 vector of up to "
                             f"{MAX_INT} entries beside x, not {_is(expert_map)}")
        at_map = expert_map.data_ptr()
    r, more = 0, ()
    if adapters is not None:
        r, more = _adapters(T, H, I, index, *adapters)
    nbytes = workspace_bytes(T, k, H, I, wtype, r)
    out = torch.empty_like(x)              # x's rows are dense or strided: out's are dense
    workspace = x.new_empty(nbytes // 2)
    _call(index, fn, x.data_ptr(), T, _row_stride(x), H, ids.data_ptr(), weights.data_ptr(), k,
          at_map, n_map, at13, s13, at2, s2, wtype, S, I, *more, out.data_ptr(),
          _row_stride(out), workspace.data_ptr(), nbytes)
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
    return _layer(lib().expert_cache_experts, x, topk_weights, topk_ids, w13, w2, w13_scale,
                  w2_scale, expert_map)


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
    return _layer(lib().expert_cache_experts_lora, x, topk_weights, topk_ids, w13, w2,
                  w13_scale, w2_scale, expert_map, (a13, b13, a2, b2, scaling, adapter))


def _adapters(T, H, I, index, a13, b13, a2, b2, scaling, adapter):
    """Rank and arguments of the adapters, checked."""
    if a13.dim() != 4 or a2.dim() != 4:
        raise ValueError(f"adapter matrices must be 4-D, not {_is(a13)} and {_is(a2)}")
    L, E, r = a13.size(0), a13.size(1), a2.size(2)
    if L < 1 or E < 1 or r % 8 or not 0 < r <= MAX_RANK:
        raise ValueError(f"{L} adapters of {E} experts, rank {r}: the rank must be a multiple "
                         f"of 8 up to {MAX_RANK}")
    args = []
    for name, t, rows, cols in (("a13", a13, 2 * r, H), ("b13", b13, 2 * I, r),
                                ("a2", a2, r, I), ("b2", b2, H, r)):
        at = t.data_ptr()
        if t.shape != (L, E, rows, cols) or t.dtype is not _BF16 or at % 16 \
                or not t.is_contiguous() or t.get_device() != index:
            raise ValueError(f"{name} must be contiguous, 16-byte aligned bf16 "
                             f"{(L, E, rows, cols)} beside x, not {_is(t)}")
        args.append(at)
    if scaling.shape != (L,) or scaling.dtype is not _F32 or not scaling.is_contiguous() \
            or scaling.get_device() != index:
        raise ValueError(f"scaling must be contiguous fp32 [{L}] beside x, not {_is(scaling)}")
    if adapter.shape != (T,) or adapter.dtype is not _I32 or not adapter.is_contiguous() \
            or adapter.get_device() != index:
        raise ValueError(f"adapter must be contiguous int32 [{T}] beside x, not {_is(adapter)}")
    return r, (adapter.data_ptr(), *args, scaling.data_ptr(), L, E, r)
