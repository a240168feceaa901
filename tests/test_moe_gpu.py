"""The MoE layer's operators on the GPU against their definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

import moe_ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def moe():
    from gpu_util import lib
    lib()
    from vllm_expert_cache import moe
    return moe


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def weights_of(g, kind, S, I, H):
    """w13, w2, w13_scale, w2_scale with entries of about N(0, 0.02 .. 0.05)."""
    if kind == "bf16":
        return normal(g, S, 2 * I, H, std=0.05), normal(g, S, H, I, std=0.05), None, None
    out = []
    for shape in ((S, 2 * I, H), (S, H, I)):
        if kind == "int8":
            w = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
        else:
            w = normal(g, *shape, std=80.0, dtype=torch.float32).clamp(-448, 448).to(
                torch.float8_e4m3fn)
        scale = (torch.rand(S, shape[1], 1, generator=g, device=DEV) + 0.5) * 0.05 / 80
        out += [w, scale]
    return out[0], out[2], out[1], out[3]


def routing(g, T, k, n):
    ids = torch.stack([torch.randperm(n, generator=g, device=DEV)[:k] for _ in range(T)]) \
        if n >= k else torch.randint(0, n, (T, k), generator=g, device=DEV)
    w = torch.rand(T, k, generator=g, device=DEV) + 0.05
    return w / w.sum(1, keepdim=True), ids.to(torch.int32)


def check(out, want, bound, tag=""):
    assert out.dtype == torch.bfloat16 and out.shape == want.shape
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all(), tag
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{tag}: {worst:.3f} of the bound"


SHAPES = [  # T, k, S, H, I
    (1, 1, 1, 16, 16),
    (1, 8, 64, 2048, 768),
    (2, 2, 4, 512, 1024),
    (5, 3, 21, 1232, 416),
    (8, 4, 9, 48, 16),
    (9, 2, 5, 272, 2064),
    (16, 8, 128, 256, 64),
    (17, 5, 7, 144, 336),
    (32, 8, 40, 512, 96),
    (33, 1, 3, 96, 128),
    (70, 6, 30, 160, 48),
    (3, 32, 40, 64, 32),
]


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("T,k,S,H,I", SHAPES)
def test_experts(moe, kind, T, k, S, H, I):
    g = gen(T * 1000 + k)
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    got = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
    again = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
    check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2), f"{kind} T={T}")
    assert torch.equal(got, again)          # the same inputs give the same bits


def test_experts_bf16_smallest_width(moe):
    """The narrowest bf16 rows: one 16-byte vector each."""
    g = gen(3)
    w13, w2, _, _ = weights_of(g, "bf16", 2, 8, 8)
    x = normal(g, 3, 8)
    w, ids = routing(g, 3, 2, 2)
    check(moe.experts(x, w, ids, w13, w2), *moe_ref.experts(x, w, ids, w13, w2))


@pytest.mark.parametrize("kind", DTYPES)
def test_experts_ids_out_of_range_padding_repeats_and_map(moe, kind):
    g = gen(11)
    T, k, S, H, I = 12, 4, 6, 96, 80
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    ids[0] = -1                                     # batch padding
    ids[1, 2] = S                                   # not a slot
    ids[2] = torch.tensor([3, 3, 3, 3])             # one slot four times
    ids[3] = torch.tensor([5, 1, 5, 1])
    ids[4, 0] = -2 ** 31
    ids[5, 3] = 2 ** 31 - 1
    w[0] = float("nan")                             # weights of pairs that add nothing
    w[1, 2] = float("inf")
    args = dict(w13_scale=s13, w2_scale=s2)
    got = moe.experts(x, w, ids, w13, w2, **args)
    check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2), kind)
    assert (got[0] == 0).all()
    # global ids through a map: two of three ids are another rank's
    emap = torch.full((18,), -1, dtype=torch.int32, device=DEV)
    emap[2::3] = torch.randperm(S, generator=g, device=DEV).to(torch.int32)
    emap[0] = S + 3                                 # not a slot either
    w, ids = routing(g, T, k, 18)
    ids[7, 1], ids[8, 0] = 18, -5
    got = moe.experts(x, w, ids, w13, w2, expert_map=emap, **args)
    check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2, expert_map=emap), kind)
    # no token has an expert here
    none = torch.full((T, k), -1, dtype=torch.int32, device=DEV)
    assert (moe.experts(x, w, none, w13, w2, **args) == 0).all()


def test_experts_every_token_on_one_slot(moe):
    g = gen(12)
    T, k, S, H, I = 32, 3, 4, 64, 48
    w13, w2, _, _ = weights_of(g, "bf16", S, I, H)
    x = normal(g, T, H)
    w, _ = routing(g, T, k, S)
    ids = torch.full((T, k), 2, dtype=torch.int32, device=DEV)
    check(moe.experts(x, w, ids, w13, w2), *moe_ref.experts(x, w, ids, w13, w2))


@pytest.mark.parametrize("kind", DTYPES)
def test_experts_strided_rows_and_converted_routing(moe, kind):
    g = gen(13)
    T, k, S, H, I = 7, 2, 5, 128, 64
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    big = normal(g, T, 3 * H)
    w, ids = routing(g, T, k, S)
    want, bound = moe_ref.experts(big[:, H:2 * H], w, ids, w13, w2, s13, s2)
    args = dict(w13_scale=s13, w2_scale=s2)
    check(moe.experts(big[:, H:2 * H], w, ids, w13, w2, **args), want, bound)
    odd = torch.empty(T * (H + 1) + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, H + 1)
    odd[:, :H] = big[:, H:2 * H]                    # rows that no 16-byte load can take
    check(moe.experts(odd[:, :H], w, ids, w13, w2, **args), want, bound)
    turned = big[:, H:2 * H].t().contiguous().t()   # inner stride T
    ids64 = ids.long().t().contiguous().t()
    check(moe.experts(turned, w.double(), ids64, w13, w2, **args), want, bound)
    far = ids64.clone()
    far[0, 0] += 2 ** 32                            # must not wrap into a slot
    got = moe.experts(turned, w, far, w13, w2, **args)
    ids[0, 0] = -1
    check(got, *moe_ref.experts(big[:, H:2 * H], w, ids, w13, w2, s13, s2))


@pytest.mark.parametrize("kind", DTYPES)
def test_experts_nan_inf_and_zero_rows_stay_in_their_token(moe, kind):
    g = gen(14)
    T, k, S, H, I = 6, 2, 5, 128, 64
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, 4)                    # slot 4 is never routed
    clean = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
    if kind == "int8":
        s13[4], s2[4] = float("nan"), float("nan")
    else:
        w13[4], w2[4] = float("nan"), float("nan")  # what an empty slot may hold
    x[1, 5], x[3, 7] = float("nan"), float("inf")
    x[4] = 0
    got = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
    for t in (0, 2, 5):
        assert torch.equal(got[t], clean[t])
    assert got[1].isnan().all() and not torch.isfinite(got[3]).any()
    assert (got[4] == 0).all()
    ids[1] = -1                                     # a padded row's content is never seen
    assert (moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)[1] == 0).all()


def test_experts_large_h_saturates_to_inf_not_nan(moe):
    """h beyond bf16: inf, as the definition rounds, without a NaN remainder."""
    x = torch.full((1, 8), 1e19, dtype=torch.bfloat16, device=DEV)
    w13 = torch.full((1, 16, 8), 1e2, dtype=torch.bfloat16, device=DEV)
    w2 = torch.ones((1, 8, 8), dtype=torch.bfloat16, device=DEV)
    out = moe.experts(x, torch.ones(1, 1, device=DEV),
                      torch.zeros(1, 1, dtype=torch.int32, device=DEV), w13, w2)
    assert (out == float("inf")).all()


def test_experts_slots_past_32_bits(moe):
    """The last of 1024 slots starts 6 GB into w13."""
    g = gen(15)
    S, H, I, k = 1024, 2048, 768, 2
    w13 = torch.empty(S, 2 * I, H, dtype=torch.bfloat16, device=DEV)
    w2 = torch.empty(S, H, I, dtype=torch.bfloat16, device=DEV)
    use = [0, S - 1, S - 2]
    for s in use:
        w13[s], w2[s] = normal(g, 2 * I, H, std=0.05), normal(g, H, I, std=0.05)
    x = normal(g, 2, H)
    w, _ = routing(g, 2, k, S)
    ids = torch.tensor([[S - 1, 0], [S - 2, S - 1]], dtype=torch.int32, device=DEV)
    check(moe.experts(x, w, ids, w13, w2), *moe_ref.experts(x, w, ids, w13, w2))


def test_experts_empty_batch(moe):
    g = gen(16)
    w13, w2, _, _ = weights_of(g, "bf16", 2, 16, 32)
    out = moe.experts(normal(g, 0, 32), torch.empty(0, 2, device=DEV),
                      torch.empty(0, 2, dtype=torch.int32, device=DEV), w13, w2)
    assert out.shape == (0, 32)


@pytest.mark.parametrize("kind", DTYPES)
def test_experts_wide_rows(moe, kind):
    """Rows too wide for the on-chip copy of x of this many tokens."""
    g = gen(17)
    T, k, S, H, I = 16, 1, 3, 16384, 32
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H, std=0.3)
    w, ids = routing(g, T, k, S)
    got = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
    check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2))


def test_experts_on_a_side_stream_and_captured(moe):
    g = gen(18)
    T, k, S, H, I = 4, 2, 8, 256, 128
    w13, w2, s13, s2 = weights_of(g, "int8", S, I, H)
    args = dict(w13_scale=s13, w2_scale=s2)
    cases = [(normal(g, T, H), *routing(g, T, k, S)) for _ in range(3)]
    eager = [moe.experts(x, w, i, w13, w2, **args) for x, w, i in cases]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        on_side = [moe.experts(x, w, i, w13, w2, **args) for x, w, i in cases]
    side.synchronize()
    for a, b in zip(eager, on_side):
        assert torch.equal(a, b)
    sx, sw, si = (t.clone() for t in cases[0])
    graphs = []
    for _ in range(2):                              # two graphs over the same inputs
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = moe.experts(sx, sw, si, w13, w2, **args)
            out2 = moe.experts(out, sw, si, w13, w2, **args)
        graphs.append((gr, out, out2))
    for x, w, i in cases:
        sx.copy_(x); sw.copy_(w); si.copy_(i)
        for gr, _, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        want = moe.experts(x, w, i, w13, w2, **args)
        want2 = moe.experts(want, w, i, w13, w2, **args)
        for _, o, o2 in graphs:
            assert torch.equal(o, want) and torch.equal(o2, want2)


# ---------------------------------------------------------------------------------------
# adapters

def adapters_of(g, L, E, r, H, I):
    return (normal(g, L, E, 2 * r, H, std=0.05), normal(g, L, E, 2 * I, r, std=0.1),
            normal(g, L, E, r, I, std=0.05), normal(g, L, E, H, r, std=0.1),
            torch.linspace(0.5, 2.0, L, device=DEV))


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("T,k,S,H,I,L,r", [
    (1, 8, 64, 512, 192, 4, 16), (1, 1, 1, 16, 16, 1, 8), (11, 2, 13, 720, 208, 3, 8),
    (8, 4, 10, 256, 128, 9, 32), (20, 3, 6, 128, 80, 2, 24), (37, 2, 5, 96, 64, 5, 64),
    (3, 2, 4, 64, 48, 2, 256)])
def test_experts_lora(moe, kind, T, k, S, H, I, L, r):
    g = gen(T * 100 + r)
    E = 2 * S
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, E)
    table = torch.full((E,), -1, dtype=torch.int32, device=DEV)
    at = torch.randperm(E, generator=g, device=DEV)[:S]
    table[at] = torch.randperm(S, generator=g, device=DEV).to(torch.int32)
    lora = adapters_of(g, L, E, r, H, I)
    adapter = torch.randint(-1, L, (T,), generator=g, device=DEV, dtype=torch.int32)
    adapter[0] = 0
    ids[0, 0] = at[0]
    got = moe.experts_lora(x, w, ids, w13, w2, *lora, adapter, w13_scale=s13, w2_scale=s2,
                           expert_map=table)
    want, bound = moe_ref.experts(x, w, ids, w13, w2, s13, s2, table, lora, adapter)
    check(got, want, bound, f"{kind} T={T} r={r}")
    # adapters matter at all here
    plain = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2, expert_map=table)
    assert ((plain.double() - want).abs() > bound).any()


@pytest.mark.parametrize("kind", DTYPES)
def test_experts_lora_without_adapters_is_experts(moe, kind):
    g = gen(30)
    T, k, S, H, I, L, r = 9, 3, 7, 128, 96, 2, 16
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    ids[4] = -1
    lora = adapters_of(g, L, S, r, H, I)
    args = dict(w13_scale=s13, w2_scale=s2)
    want = moe.experts(x, w, ids, w13, w2, **args)
    for none in (-1, L, 2 ** 31 - 1, -2 ** 31):     # outside [0, L): no adapter
        adapter = torch.full((T,), none, dtype=torch.int32, device=DEV)
        assert torch.equal(moe.experts_lora(x, w, ids, w13, w2, *lora, adapter, **args), want)


def test_experts_lora_id_past_the_adapters_experts(moe):
    """A routed id that the adapter matrices do not cover has no adapter."""
    g = gen(31)
    T, k, S, H, I, L, r = 5, 3, 8, 64, 48, 2, 8
    w13, w2, _, _ = weights_of(g, "bf16", S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    lora = adapters_of(g, L, 4, r, H, I)            # experts 4..7: none
    adapter = torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32, device=DEV)
    got = moe.experts_lora(x, w, ids, w13, w2, *lora, adapter)
    check(got, *moe_ref.experts(x, w, ids, w13, w2, lora=lora, adapter=adapter))


# ---------------------------------------------------------------------------------------
# router

def check_route(got, want):
    weights, ids = got
    assert weights.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids, want[1])
    # scores in 64 bits, one rounding to fp32 (half a step: 2^-24) and room for exp's
    torch.testing.assert_close(weights.double(), want[0], rtol=2.0 ** -23, atol=1e-37)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,H", [(1, 128, 8, 2048), (1, 1, 1, 8), (3, 8, 8, 64),
                                     (16, 256, 8, 4096), (53, 61, 5, 1000), (2, 2048, 32, 136),
                                     (130, 33, 32, 16), (5, 512, 10, 7168), (1, 7, 2, 16384)])
def test_route(moe, scoring, T, E, k, H):
    g = gen(T + E)
    x, gate = normal(g, T, H), normal(g, E, H, std=1.0 / H ** 0.5)
    bias = normal(g, E, std=0.1, dtype=torch.float32) if scoring == "sigmoid" else None
    check_route(moe.route(x, gate, k, scoring=scoring, bias=bias),
                moe_ref.route(x, gate, k, scoring, bias))
    check_route(moe.route(x, gate, k, scoring=scoring, renormalize=False, scale=2.5),
                moe_ref.route(x, gate, k, scoring, renormalize=False, scale=2.5))


def test_route_ties_go_to_the_lower_id(moe):
    g = gen(40)
    x, gate = normal(g, 4, 256), normal(g, 12, 256)
    gate[3] = gate[9]
    gate[5] = gate[9]
    x[2] = 0                                        # every score equal
    for scoring in ("softmax", "sigmoid"):
        got = moe.route(x, gate, 12, scoring=scoring)
        check_route(got, moe_ref.route(x, gate, 12, scoring))
        assert got[1][2].tolist() == list(range(12))


def test_route_scores_closer_than_fp32_sums(moe):
    """Experts whose scores differ by less than an fp32 sum of these terms resolves."""
    g = gen(41)
    H, E = 4096, 16
    x = normal(g, 8, H)
    gate = normal(g, 1, H).repeat(E, 1)
    for e in range(E):                              # one weight, off by one bf16 step
        gate[e, e] = gate[0, e] * (1 + 2.0 ** -7)
    x[:, :E] *= 2.0 ** -12
    check_route(moe.route(x, gate, 8), moe_ref.route(x, gate, 8))


def test_route_nan_and_inf_scores(moe):
    g = gen(42)
    x, gate = normal(g, 3, 64).abs(), normal(g, 6, 64)
    gate[1, 3] = float("nan")
    gate[4, 0] = float("-inf")
    x[1] = float("nan")
    for scoring in ("softmax", "sigmoid"):
        w, ids = moe.route(x, gate, 6, scoring=scoring)
        rw, rids = moe_ref.route(x, gate, 6, scoring)
        assert torch.equal(ids, rids)
        torch.testing.assert_close(w.double(), rw, rtol=2.0 ** -23, atol=1e-37)
        assert (ids[1] == -1).all() and (w[1] == 0).all()


def test_route_strided_rows_and_empty(moe):
    g = gen(43)
    big, gate = normal(g, 6, 256), normal(g, 9, 64)
    check_route(moe.route(big[:, 64:128], gate, 3), moe_ref.route(big[:, 64:128], gate, 3))
    w, ids = moe.route(big[:0, :64], gate, 3)
    assert w.shape == (0, 3) and ids.shape == (0, 3)


def test_route_then_experts_captured(moe):
    """Router and experts as one captured step, replayed on new hidden states."""
    g = gen(44)
    T, k, S, H, I = 6, 4, 16, 256, 96
    w13, w2, s13, s2 = weights_of(g, "fp8", S, I, H)
    gate = normal(g, S, H, std=0.1)
    x = normal(g, T, H)

    def step():
        w, ids = moe.route(x, gate, k)
        return moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2), w, ids
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, w, ids = step()
    for seed in range(3):
        x.copy_(normal(gen(seed), T, H))
        graph.replay()
        torch.cuda.synchronize()
        check_route((w, ids), moe_ref.route(x, gate, k))
        check(out, *moe_ref.experts(x, w, ids, w13, w2, s13, s2))


def test_route_subnormal_and_tiny_operands(moe):
    """Operands at the bottom of the type's range still order the experts."""
    g = gen(45)
    gate = normal(g, 24, 512)
    x = normal(g, 5, 512)
    x[0] *= 2.0 ** -130                             # subnormal
    x[1] *= 2.0 ** -120
    x[2, ::2] = 2.0 ** -133                         # the smallest subnormal among ordinary ones
    x[3] = 0
    x[3, 7] = 2.0 ** -133
    check_route(moe.route(x, gate, 24), moe_ref.route(x, gate, 24))
    gate[5] *= 2.0 ** -128                          # and in the router's weight
    gate[9] = 0
    gate[9, 3] = 2.0 ** -133
    check_route(moe.route(x, gate, 24), moe_ref.route(x, gate, 24))


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("T,k,S,H,I,L,r", [
    (16, 4, 10, 2064, 4096, 0, 0), (21, 4, 36, 488, 3184, 2, 8), (32, 8, 40, 160, 1040, 0, 0),
    (2, 2, 4, 1024, 14336, 0, 0), (13, 8, 8, 736, 3936, 3, 256), (1, 3, 3, 64, 32768, 0, 0)])
def test_experts_h_in_segments(moe, kind, T, k, S, H, I, L, r):
    """More of h than the second kernel can hold at once."""
    g = gen(T + I)
    vec = 8 if kind == "bf16" else 16
    H = H // vec * vec
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    ids[T // 2, 0] = -1
    args = dict(w13_scale=s13, w2_scale=s2)
    if L:
        lora = adapters_of(g, L, S, r, H, I)
        adapter = torch.randint(-1, L, (T,), generator=g, device=DEV, dtype=torch.int32)
        got = moe.experts_lora(x, w, ids, w13, w2, *lora, adapter, **args)
        check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2, None, lora, adapter))
    else:
        got = moe.experts(x, w, ids, w13, w2, **args)
        check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2))
        assert torch.equal(got, moe.experts(x, w, ids, w13, w2, **args))


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("T,H,I", [(2, 128, 64), (12, 256, 96), (20, 96, 4096), (32, 128, 64)])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_experts_bad_weights_stay_with_the_tokens_routed_there(moe, kind, T, H, I, bad):
    """An infinity or a NaN in an expert's weights reaches the tokens that are routed to it
    and leaves the others' bits alone."""
    g = gen(T + I)
    S, k, v = 12, 3, float(bad)
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S - 1)
    ids[T // 2, 1] = ids[0, 2] = S - 1              # the bad one, of two tokens
    hit = [0, T // 2]
    others = [t for t in range(T) if t not in hit]
    clean = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
    where = [lambda: w2[S - 1].view(-1)[::7].fill_(v), lambda: w13[S - 1].view(-1)[::5].fill_(v)]
    if kind != "bf16":
        where = [lambda: s2[S - 1].fill_(v), lambda: s13[S - 1, 3].fill_(v)]
    if kind == "fp8":                               # (e4m3 has a NaN of its own)
        where.append(lambda: w2[S - 1].view(torch.uint8).view(-1)[::7].fill_(0x7f))
    for plant in where:
        plant()
        got = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2)
        assert torch.equal(got[others], clean[others])
        assert not torch.isfinite(got[hit]).all(1).any()


@pytest.mark.parametrize("kind", DTYPES)
@pytest.mark.parametrize("T,H,I,r", [(2, 128, 64, 8), (12, 256, 96, 16), (20, 96, 4096, 136)])
@pytest.mark.parametrize("matrix", range(4))
def test_experts_lora_bad_adapter_stays_with_its_tokens(moe, kind, T, H, I, r, matrix):
    g = gen(T + r)
    S, k, L = 6, 3, 3
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    lora = adapters_of(g, L, S, r, H, I)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    adapter = torch.arange(T, dtype=torch.int32, device=DEV) % (L + 1) - 1
    hit = [t for t in range(T) if t % (L + 1) == 2]                # adapter 1
    others = [t for t in range(T) if t not in hit]

    def run():
        return moe.experts_lora(x, w, ids, w13, w2, *lora, adapter, w13_scale=s13, w2_scale=s2)

    clean = run()
    lora[matrix][1].view(-1)[::11].fill_(float("nan"))
    got = run()
    assert torch.equal(got[others], clean[others])
    assert not hit or not torch.isfinite(got[hit]).all(1).any()


@pytest.mark.parametrize("kind", DTYPES)
def test_experts_lora_repeated_slots(moe, kind):
    """A token that names an expert twice, or two experts in one slot: each pair adds its
    own, and with its own expert's adapter."""
    g = gen(77)
    T, k, S, H, I, L, r = 6, 4, 5, 128, 64, 2, 8
    w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
    x = normal(g, T, H)
    w, ids = routing(g, T, k, S)
    lora = adapters_of(g, L, 2 * S, r, H, I)
    table = (torch.arange(2 * S, dtype=torch.int32, device=DEV) % S).contiguous()
    ids[1] = ids[1, 0]
    ids[2, 1], ids[4, 3] = ids[2, 0] + S, ids[4, 0] + S        # another expert, the same slot
    adapter = torch.tensor([0, 1, 0, -1, 1, 0], dtype=torch.int32, device=DEV)
    got = moe.experts_lora(x, w, ids, w13, w2, *lora, adapter, w13_scale=s13, w2_scale=s2,
                           expert_map=table)
    check(got, *moe_ref.experts(x, w, ids, w13, w2, s13, s2, table, lora, adapter), kind)


def test_layers_on_two_streams_at_once(moe):
    """Calls in flight on two streams, of kernels that start early and share SMs: each has
    the bits of a call alone."""
    g = gen(78)
    T, k, S, H, I, E = 6, 4, 24, 512, 256, 64
    work = []
    for kind in DTYPES:
        w13, w2, s13, s2 = weights_of(g, kind, S, I, H)
        lora = adapters_of(g, 2, S, 16, H, I)
        gate = normal(g, E, H, std=0.1)
        adapter = torch.arange(T, dtype=torch.int32, device=DEV) % 3 - 1
        table = (torch.arange(E, dtype=torch.int32, device=DEV) % S).contiguous()

        def layer(x, w13=w13, w2=w2, s13=s13, s2=s2, lora=lora, gate=gate):
            w, ids = moe.route(x, gate, k)
            x = moe.experts(x, w, ids, w13, w2, w13_scale=s13, w2_scale=s2, expert_map=table)
            return moe.experts_lora(x, w, ids, w13, w2, *lora, adapter, w13_scale=s13,
                                    w2_scale=s2, expert_map=table)

        work.append(layer)
    xs = [normal(g, T, H) for _ in range(8)]
    want = [[f(x) for f in work] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for x in xs * 4:
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append([f(x) for f in work])
    torch.cuda.synchronize()
    for mine in got:
        for i, outs in enumerate(mine):
            for o, v in zip(outs, want[i % len(xs)]):
                assert torch.equal(o, v)


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing needs a call outside of a capture first."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from vllm_expert_cache import moe
g = torch.Generator(device="cuda").manual_seed(1)
def n(*s):
    return (torch.randn(s, generator=g, device="cuda") * 0.1).bfloat16()
x, gate, w13, w2 = n(3, 256), n(128, 256), n(128, 128, 256), n(128, 256, 64)
lora = n(2, 128, 16, 256), n(2, 128, 128, 8), n(2, 128, 8, 64), n(2, 128, 256, 8)
c, ad = torch.ones(2, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda") % 2
def layer():
    w, ids = moe.route(x, gate, 4)
    return moe.experts(x, w, ids, w13, w2), moe.experts_lora(x, w, ids, w13, w2, *lora, c, ad)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = layer()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(out, layer()):
    assert torch.equal(a, b) and a.abs().max() > 0
"""
    root = Path(__file__).resolve().parent.parent / "vllm-expert-cache_b200"
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
