"""Mixture-of-experts operators on the GPU at the edges of what callers may pass: activations with a mean, values that are not
finite, offsets that are a slice of longer ones, single rows of odd strides, tall tiles filled to the end.

Plain 64-bit computations and tolerances are those of ``test_gpu_experts`` (derived at its top)."""
import pytest
import torch

import gemlite_amd
from gemlite_amd import ExpertPlan, GemLiteExperts, GemLiteLinear, GemLiteMoE
from gemlite_amd.helper import A16W4_HQQ_INT
from test_gpu_experts import DT, FORMATS, _gen, check, make_layers, make_x, ref_plan, ref_route, ref_rows, run_case, silu

pytestmark = pytest.mark.gpu

# a tile configuration of every product kernel: streaming kernel (4- and 16-row tiles, with K splits), tiled GEMM
KERNELS = [4, 16, 2016, 64, 2064, 128, 256]


# ---------------------------------------------------------------------------
# 4-bit weights with a zero point in codes
# ---------------------------------------------------------------------------
def shifted_layers(kind, dtype, E, K, N, gs, seed=0):
    """E layers whose weights are (q - zero) * scale, and these weights [E, K, N] in float64."""
    g = _gen(seed)
    dt, gdt = DT[dtype]
    layers, weights = [], []
    for _ in range(E):
        q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.int32).to(torch.uint8)
        if kind == "channelwise":     # fractional zeros, one scale per output channel
            s = ((0.5 + torch.rand((N, 1), generator=g)) / (4.6 * K ** 0.5)).to(dt)
            z = (torch.rand((N, 1), generator=g) * 3 + 6).to(dt)
            layer = A16W4_HQQ_INT(device="cuda", dtype=dt).from_weights(q.cuda(), s.cuda(), z.cuda())
            w = (q.double() - z.double()) * s.double()
        else:                         # one integer zero for all groups
            s = ((0.5 + torch.rand((N * K // gs, 1), generator=g)) / (4.6 * K ** 0.5)).to(dt)
            layer = GemLiteLinear(4, gs, K, N, gdt, gdt).pack(q.cuda(), s.cuda(), 7)
            w = ((q.double() - 7).view(N, K // gs, gs) * s.double().view(N, K // gs, 1)).view(N, K)
        layers.append(layer)
        weights.append(w.t())
    return layers, torch.stack(weights)


@pytest.mark.parametrize("kind", ["channelwise", "integer"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("tile_config", [16, 64, 128])
def test_shifted_codes_and_activations_with_a_mean(kind, dtype, tile_config):
    """Every weight is rounded to the activation type at most once: an error of zero * scale, the same for all codes of a
    group, would add up with the sum of the activations.  The roundings of the weights and the result are independent and
    uniform, 0.58 u each: 0.82 u in the 2-norm, below u as in ``test_gpu_experts``."""
    E, R, K, N = 2, 150, 2048, 96
    layers, W = shifted_layers(kind, dtype, E, K, N, 128)
    e = GemLiteExperts.from_layers(layers)
    assert e.meta_args[10] == 3
    u = torch.finfo(DT[dtype][0]).eps / 2
    x = (make_x(R, K, "bf16").float() + 1).to(DT[dtype][0])
    offsets = torch.tensor([0, 70, R], dtype=torch.int32)
    y, mag = ref_rows("w4", x, W, offsets)
    s = max(float(layer.scales.data.abs().max()) for layer in layers)
    off = 128 if dtype == "bf16" else 1024
    slack = u * mag + K * 2.0 ** -24 * x.double().abs().sum(1, keepdim=True) * ((off + 15) * s + 16 * s)
    out = gemlite_amd.experts_functional(x.cuda(), None, e.get_tensor_args(), e.get_meta_args(), offsets.cuda(), tile_config=tile_config)
    check(out, y, slack, u, u)


def test_route_of_one_row_of_any_stride():
    """A [1, E] row is contiguous whatever its row stride says (a transposed [E, 1] product has 1)."""
    values = torch.randn(64, generator=_gen(0)).cuda()
    want = gemlite_amd.route_experts(values[:16].view(1, 16), 4)
    for row in (values[:16].view(16, 1).t(), values.as_strided((1, 16), (0, 1)), values.as_strided((1, 16), (64, 1))):
        assert row.stride(0) != 16 and all(torch.equal(a, b) for a, b in zip(gemlite_amd.route_experts(row, 4), want))


@pytest.mark.parametrize("T,E,k", [(39, 128, 8), (40, 8, 2), (41, 8, 2), (63, 60, 6), (40, 1024, 16), (41, 512, 8)])
def test_routes_around_the_single_workgroup(T, E, k):
    logits = torch.randn((T, E), generator=_gen(T)).half().float()   # ties
    plan = gemlite_amd.route_experts(logits.cuda(), k)
    w, ids = ref_route(logits, k, "softmax", True, 1.0)
    offsets, order, places = ref_plan(ids, E)
    for got, want in zip(plan[1:], (ids, offsets, order, places)):
        assert torch.equal(got.cpu().long(), want)
    # (as in test_gpu_experts: exp of a difference below 32, a sum of up to E of them, one division)
    assert bool(((plan.weights.cpu().double() - w).abs() <= (2.0 ** -18 + E * 2.0 ** -24) * w).all())
    again = gemlite_amd.plan_experts(plan.expert_ids, plan.weights, E)
    assert all(torch.equal(a, b) for a, b in zip(plan, again))


# ---------------------------------------------------------------------------
# values that are not finite
# ---------------------------------------------------------------------------
def same_kind(y, ref):
    """NaN, +inf and -inf in the same places (``ref`` in 64 bits, sums of moderate size otherwise)."""
    y = y.cpu().double()
    return torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isposinf(y), torch.isposinf(ref)) and torch.equal(
        torch.isneginf(y), torch.isneginf(ref))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tile_config", KERNELS)
def test_infinite_activations_of_fp8_experts(dtype, tile_config):
    """s = inf / 448 = inf, 1 / s = 0, code = e4m3(inf * 0) = NaN: a block with an infinity is NaN by the definition."""
    E, R, K, N = 2, 40, 512, 64
    layers, W = make_layers("fp8", dtype, E, K, N)
    e = GemLiteExperts.from_layers(layers)
    off = torch.tensor([0, 13, R], dtype=torch.int32, device="cuda")
    x = make_x(R, K, dtype).cuda()
    args = (None, e.get_tensor_args(), e.get_meta_args(), off)
    clean = gemlite_amd.experts_functional(x, *args, tile_config=tile_config)
    x[3, 200], x[20, 7], x[30, 511], x[30, 0] = float("inf"), float("-inf"), float("inf"), float("-inf")
    out = gemlite_amd.experts_functional(x, *args, tile_config=tile_config)
    odd = torch.zeros(R, dtype=torch.bool, device="cuda")
    odd[[3, 20, 30]] = True
    assert torch.equal(out[~odd], clean[~odd])
    assert bool(torch.isnan(out[odd]).all())


@pytest.mark.parametrize("fmt", ["w4", "h16"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tile_config", KERNELS)
def test_infinite_activations_of_unquantised_rows(fmt, dtype, tile_config):
    """An infinity times a weight is an infinity of its sign in every kernel, two of opposite sign make NaN."""
    E, R, K, N = 2, 40, 512, 64
    layers, W = make_layers(fmt, dtype, E, K, N, 64)
    e = GemLiteExperts.from_layers(layers)
    offsets = torch.tensor([0, 13, R], dtype=torch.int32)
    x = make_x(R, K, dtype)
    args = (None, e.get_tensor_args(), e.get_meta_args(), offsets.cuda())
    clean = gemlite_amd.experts_functional(x.cuda(), *args, tile_config=tile_config)
    x[3, 200], x[20, 7], x[30, 511], x[30, 0], x[39, 100] = float("inf"), float("-inf"), float("inf"), float("-inf"), float("nan")
    out = gemlite_amd.experts_functional(x.cuda(), *args, tile_config=tile_config)
    odd = torch.zeros(R, dtype=torch.bool)
    odd[[3, 20, 30, 39]] = True
    assert torch.equal(out.cpu()[~odd], clean.cpu()[~odd])
    assert same_kind(out, ref_rows(fmt, x, W, offsets)[0])


@pytest.mark.parametrize("tile_config", KERNELS)
def test_large_activations_of_4_bit_experts(tile_config):
    """Values whose product with a code of 128 + q would overflow fp32 while that with the weight does not."""
    E, R, K, N = 2, 24, 256, 64
    layers, W = make_layers("w4", "bf16", E, K, N, 64)
    e = GemLiteExperts.from_layers(layers)
    offsets = torch.tensor([0, 13, R], dtype=torch.int32)
    x = make_x(R, K, "bf16")
    x[5] = 0
    x[5, 17] = 2.0 ** 124          # 128 of it: 2^131
    x[20, 3], x[20, 4] = 2.0 ** 122, -(2.0 ** 123)
    y, mag = ref_rows("w4", x, W, offsets)
    u = 2.0 ** -8
    assert float(y.abs().max()) < 2.0 ** 127
    out = gemlite_amd.experts_functional(x.cuda(), None, e.get_tensor_args(), e.get_meta_args(), offsets.cuda(), tile_config=tile_config).cpu().double()
    # (one rounding of each weight and one of the result; fp32 sums of these few terms of one size)
    for r in (5, 20):
        assert bool(((out[r] - y[r]).abs() <= (2 * u + K * 2.0 ** -24) * mag[r]).all())


# ---------------------------------------------------------------------------
# offsets that do not start at the first row
# ---------------------------------------------------------------------------
def poison(*shapes):
    """Leave memory full of NaN to the allocator, so that rows nobody writes show."""
    held = [torch.full(s, float("nan"), device="cuda") for s in shapes for _ in range(2)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile_config", KERNELS + [-1])
def test_offsets_of_a_slice_of_the_experts(fmt, tile_config):
    """Rows before offsets[0], such as those of another rank's experts, have no expert: zeros, and nothing in a combination."""
    E, R, K, N = 4, 300, 512, 64
    layers, _ = make_layers(fmt, "bf16", E, K, N)
    e = GemLiteExperts.from_layers(layers)
    x = make_x(R, K, "bf16").cuda()
    targs, meta = e.get_tensor_args(), e.get_meta_args()
    for first in (1, 7, 64, 70, 290):
        off = torch.tensor([first, first, first + 5, first + 5, first + 8], dtype=torch.int32, device="cuda")
        inner = x[first:first + 8].contiguous()
        want = gemlite_amd.experts_functional(inner, None, targs, meta, off - first, tile_config=tile_config)
        poison((R, N), (4, R, N), (R, N // 2), (R, K))
        out = gemlite_amd.experts_functional(x, None, targs, meta, off, tile_config=tile_config)
        assert not out[:first].any() and not out[first + 8:].any()
        if tile_config != -1:     # (-1: the number of rows chooses the kernel)
            assert torch.equal(out[first:first + 8], want)
        order = torch.arange(R, dtype=torch.int32, device="cuda")
        plan = ExpertPlan(torch.ones((R, 1), device="cuda"), order.view(R, 1), off, order, order.view(R, 1))
        poison((R, N), (4, R, N), (R, N // 2), (R, K))
        gated = gemlite_amd.experts_gated_functional(x, None, targs, meta, plan, tile_config=tile_config)
        assert gated[first:first + 8].any() and not gated[:first].any() and not gated[first + 8:].any()
        poison((R, N), (4, R, N), (R, N // 2), (R, K))
        combined = gemlite_amd.experts_combined_functional(x, None, targs, meta, plan, tile_config=tile_config)
        assert not combined[:first].any() and not combined[first + 8:].any()
        if tile_config != -1:
            assert torch.equal(combined[first:first + 8], want)
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_row_in_front_of_the_first_expert(fmt):
    E, R, K, N = 4, 200, 128, 64
    layers, _ = make_layers(fmt, "bf16", E, K, N)
    e = GemLiteExperts.from_layers(layers)
    off = torch.full((E + 1,), R, dtype=torch.int32, device="cuda")
    poison((R, N), (4, R, N))
    assert not e(make_x(R, K, "bf16").cuda(), off).any()


# ---------------------------------------------------------------------------
# 4-bit codes are multiplied as they are: no weight is rounded
# ---------------------------------------------------------------------------
def raw_w4(dtype, E, K, N, gs, mode, scales, zeros, seed=0):
    """Random codes with these group scales / zeros [E, K / gs, N] (float64 values of the type): tensors, meta, weights."""
    dt, gdt = DT[dtype]
    W = torch.randint(-2 ** 31, 2 ** 31, (E, K // 8, N), generator=_gen(seed), dtype=torch.int64).to(torch.int32)
    q = torch.stack([(W >> (4 * i)) & 15 for i in range(8)], 2).reshape(E, K, N).double()
    s, z = scales.to(dt), zeros.to(dt)
    full = lambda t: t.double().repeat_interleave(gs, 1)   # noqa: E731
    w = {2: q * full(s), 3: (q - full(z)) * full(s), 4: q * full(s) + full(z)}[mode]
    zt = torch.empty(0, dtype=torch.int32) if mode == 2 else z
    return [W.cuda(), s.cuda(), zt.cuda()], [0, 4, gs, 15, 8, gdt.value, gdt.value, 0, gdt.value, 0, mode, 1], w


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mode", [2, 3, 4])
@pytest.mark.parametrize("gs", [32, 64, 96, 128, 192, 1152])
@pytest.mark.parametrize("tile_config", [16, 2016, 64, 2064, 3064, 128])
def test_4_bit_products_are_rounded_once(dtype, mode, gs, tile_config):
    """The one rounding of the result: uniform over a step, so an rms of u / sqrt(3) of each value or less (rounding every
    weight as well would come to more than that)."""
    E, R, K, N = 2, 150, 1152, 96
    g = _gen(3)
    s = (0.5 + torch.rand((E, K // gs, N), generator=g, dtype=torch.float64)) / (4.6 * K ** 0.5)
    s *= torch.where(torch.rand(s.shape, generator=g) < 0.3, -1.0, 1.0)
    z = 6 + 3 * torch.rand(s.shape, generator=g, dtype=torch.float64)
    targs, meta, W = raw_w4(dtype, E, K, N, gs, mode, s, z if mode == 3 else -s * z)
    x = (make_x(R, K, "bf16").float() + 0.25).to(DT[dtype][0])
    offsets = torch.tensor([0, 70, R], dtype=torch.int32)
    u = torch.finfo(DT[dtype][0]).eps / 2
    y, mag = ref_rows("w4", x, W, offsets)
    out = gemlite_amd.experts_functional(x.cuda(), None, targs, meta, offsets.cuda(), tile_config=tile_config)
    off = 128 if dtype == "bf16" else 1024
    slack = K * 2.0 ** -24 * (mag + x.double().abs().sum(1, keepdim=True) * (off + 15) * float(s.abs().max()))
    check(out, y, slack, u, u / 3 ** 0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("tile_config", [16, 64, 2064, 128])
def test_4_bit_groups_of_any_scale(dtype, gs, tile_config):
    """Scales of 0 (a group of constants, or of nothing) and scales of one column that lie far apart."""
    E, R, K, N = 1, 40, 512, 64
    G, g = K // gs, _gen(5)
    s = (0.5 + torch.rand((E, G, N), generator=g, dtype=torch.float64)) / 64
    z = torch.randn((E, G, N), generator=g, dtype=torch.float64) / 16
    s[:, torch.rand(G, generator=g) < 0.5, 8:16] = 0
    s[:, 0, 16:24] = 0
    s[:, :, 24:32] = 0
    s[:, :, 32:40], z[:, :, 32:40] = 0, 0
    s[:, ::2, 40:48] *= 2.0 ** -9
    if dtype == "bf16":   # as far apart as only this type can
        s[:, ::2, 48:56] *= 2.0 ** -90
        z[:, ::2, 48:56] *= 2.0 ** -90
    targs, meta, W = raw_w4(dtype, E, K, N, gs, 4, s, z)
    x = make_x(R, K, dtype)
    offsets = torch.tensor([0, R], dtype=torch.int32)
    u = torch.finfo(DT[dtype][0]).eps / 2
    y, mag = ref_rows("w4", x, W, offsets)
    out = gemlite_amd.experts_functional(x.cuda(), None, targs, meta, offsets.cuda(), tile_config=tile_config)
    off = 128 if dtype == "bf16" else 1024
    scale = targs[1].cpu().double().abs().amax(1)
    slack = K * 2.0 ** -24 * (mag + x.double().abs().sum(1, keepdim=True) * (off + 15) * scale)
    slack[:, 48:56] += u * mag[:, 48:56]    # (scales 2^60 apart: from weights rounded to 16 bits)
    check(out, y, slack, u, u)
    assert not out[:, 32:40].any()


@pytest.mark.parametrize("mode", ["gated", "combined"])
@pytest.mark.parametrize("K,gs", [(4608, 32), (4352, 128), (2144, 32)])
def test_many_groups_of_4_bit_experts(mode, K, gs):
    """More groups than are joined at a time, an odd number of them, K that ends inside a stage."""
    run_case("w4", "bf16", 3, 90, 2, K, 80, gs, drop=0.1, modes=(mode,))
    run_case("w4", "fp16", 3, 90, 2, K, 80, gs, tile_config=5064, modes=(mode,))


@pytest.mark.parametrize("gs", [96, 128, 192, 1152])
@pytest.mark.parametrize("tile_config", [2016, 2064, 3064, 5064])
def test_one_group_of_another_scale_and_k_splits(gs, tile_config):
    """A column that one split takes from rounded weights (scales far apart) and the others do not; groups at the splits' ends."""
    E, R, K, N = 1, 40, 1152, 64
    G, g = K // gs, _gen(6)
    s = (0.5 + torch.rand((E, G, N), generator=g, dtype=torch.float64)) / 64
    z = torch.randn((E, G, N), generator=g, dtype=torch.float64) / 16
    s[:, min(1, G - 1), ::2] *= 2.0 ** -90
    targs, meta, W = raw_w4("bf16", E, K, N, gs, 4, s, z)
    x = (make_x(R, K, "bf16").float() + 1).bfloat16()
    offsets = torch.tensor([0, R], dtype=torch.int32)
    y, mag = ref_rows("w4", x, W, offsets)
    out = gemlite_amd.experts_functional(x.cuda(), None, targs, meta, offsets.cuda(), tile_config=tile_config)
    u = 2.0 ** -8
    slack = u * mag + K * 2.0 ** -24 * (mag + x.double().abs().sum(1, keepdim=True) * (128 + 15) * float(s.max()))
    check(out, y, slack, u, 1.5 * u)


@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("tile_config", [16, 64, 128])
def test_scales_that_climb_far(order, tile_config):
    """Steps that are each in range and leave the range together; only the group of the least scale has activations."""
    E, R, K, N = 1, 24, 512, 64
    steps = torch.tensor([-100, -40, 20, 80], dtype=torch.float64)
    s = (2.0 ** steps.flip(0) if order < 0 else 2.0 ** steps).view(1, 4, 1).expand(1, 4, N).clone()
    targs, meta, W = raw_w4("bf16", E, K, N, 128, 2, s, s)
    x = make_x(R, K, "bf16")
    x[:, 128:] = 0
    if order < 0:
        x = x.flip(1).contiguous()
    offsets = torch.tensor([0, R], dtype=torch.int32)
    y, mag = ref_rows("w4", x, W, offsets)
    out = gemlite_amd.experts_functional(x.cuda(), None, targs, meta, offsets.cuda(), tile_config=tile_config)
    u = 2.0 ** -8
    check(out, y, u * mag + K * 2.0 ** -24 * (mag + x.double().abs().sum(1, keepdim=True) * (128 + 15) * 2.0 ** -100), u, 1.5 * u)


# ---------------------------------------------------------------------------
# tall tiles, filled
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tile_config", [128, 256])
def test_tiles_filled_to_the_last_row(fmt, dtype, tile_config):
    """Experts of 256 rows and more, some of whose last tile ends one row past a shorter tile."""
    E, K, N = 5, 320, 272
    if fmt == "fp8":
        K = 384
    layers, W = make_layers(fmt, dtype, E, K, N, 64)
    e = GemLiteExperts.from_layers(layers)
    counts = [256, 0, 512 + 129, 256 + 65, 255]
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    R = int(offsets[-1])
    x = make_x(R, K, dtype)
    u = torch.finfo(DT[dtype][0]).eps / 2
    y, mag = ref_rows(fmt, x, W, offsets)
    slack = K * 2.0 ** -24 * mag + (u * mag if fmt == "w4" else 0)
    out = gemlite_amd.experts_functional(x.cuda(), None, e.get_tensor_args(), e.get_meta_args(), offsets.cuda(), tile_config=tile_config)
    check(out, y, slack, u, u)


@pytest.mark.parametrize("fmt,E,T,K,N", [("h16", 2, 2400, 64, 4096), ("fp8", 2, 700, 256, 272), ("fp8", 4, 9, 4096, 64), ("fp8", 4, 8, 2560, 64), ("fp8", 4, 24, 4096, 64),
                                          ("fp8", 4, 60, 4096, 64), ("fp8", 2, 400, 128, 256), ("w4", 2, 300, 256, 144)])
def test_heights_the_library_chooses(fmt, E, T, K, N):
    """256-row tiles of 16-bit and fp8 weights, streamed fp8 weights, 128-row tiles of 4-bit weights."""
    run_case(fmt, "bf16", E, T, 1, K, N)


@pytest.mark.parametrize("fmt", FORMATS)
def test_replayed_blocks_of_many_tokens(fmt):
    """Launches in front of the tiled kernels (quantiser, sums of groups) in a captured graph, against eager calls."""
    E, k, hidden, inter, T = 4, 2, 256, 128, 300
    gate_up = GemLiteExperts.from_layers(make_layers(fmt, "bf16", E, hidden, 2 * inter, 64, 0)[0])
    down = GemLiteExperts.from_layers(make_layers(fmt, "bf16", E, inter, hidden, 64, 50)[0])
    moe = GemLiteMoE(gate_up, down, k)
    x, logits = make_x(T, hidden, "bf16").cuda(), torch.randn((T, E), generator=_gen(1)).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe(x, logits)
    for i in range(4):
        x.copy_(make_x(T, hidden, "bf16", 20 + i).cuda())
        logits.copy_(torch.randn((T, E), generator=_gen(30 + i)).cuda())
        want = moe(x, logits)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_many_slots_for_a_token():
    """(token, slot) indices whose product with the number of slots passes 2^32: the token of a row is still exact."""
    E, T, k, K, N = 2, 512, 4097, 32, 16
    layers, W = make_layers("h16", "bf16", E, K, N)
    e = GemLiteExperts.from_layers(layers)
    x = make_x(T, K, "bf16")
    R = T * k
    slot = torch.arange(R, dtype=torch.int64, device="cuda")
    expert = (slot % k) % E
    order = torch.sort(expert, stable=True).indices
    places = torch.empty_like(order)
    places[order] = slot
    offsets = torch.tensor([0, int((expert == 0).sum()), R], dtype=torch.int32, device="cuda")
    plan = ExpertPlan(torch.zeros((T, k), device="cuda"), expert.view(T, k).int(), offsets, order.int(), places.view(T, k).int())
    h = e.forward_gated(x.cuda(), plan)
    z = torch.stack([x.double() @ W[i] for i in range(E)], 1)      # [T, E, N]
    want = (silu(z[..., : N // 2]) * z[..., N // 2:]).cuda()
    got = h[plan.places.view(-1).long()].view(T, k, N // 2)
    for i in range(E):
        mine = got[:, i::E]
        assert bool((mine == mine[:, :1]).all())                   # every slot of a token with this expert has one result
        err = (mine[:, 0].double() - want[:, i]).norm() / want[:, i].norm()
        assert float(err) <= 2.0 ** -8
