"""Mixture-of-experts operators on the GPU against plain 64-bit computations of the same definitions.

Tolerances.  u = eps / 2 of the output type is the largest relative error of the one final rounding.  Around it an
element may be off by what the sum itself loses:
  * fp32 accumulation of K products: at most K 2^-24 of the sum of their magnitudes.  4-bit codes may enter the matrix
    unit with an offset of 128 (bf16) or 1024 (fp16) that is taken off again, so the magnitudes count with
    (offset + 15) * scale + |zero|;
  * 4-bit weights that are rounded to the activation type in front of the matrix unit: u of the sum of |x w|.
The gated output multiplies two such sums: |d(silu(g) u)| <= 1.1 |u| dg + |silu(g)| du + 1.1 dg du (the slope of silu is below 1.1).
Independent errors hardly ever add up to these bounds, so the whole output's 2-norm error has to stay below u as well:
the roundings (one of the result and, in the worst case, one of every weight) are uniform, with a root mean square of
u / sqrt(3) or less each, so 2-norm errors of 0.58 u for the result, 0.82 u with the weights' and 1.05 u for the gated product of
two such sums: bounds of u, and 1.5 u for gated 4-bit experts."""
import numpy as np
import pytest
import torch

import gemlite_amd
from gemlite_amd import DType, ExpertPlan, GemLiteExperts, GemLiteLinear, GemLiteMoE
from gemlite_amd.helper import A16W4_HQQ_INT, A8W8_fp8_dynamic

pytestmark = pytest.mark.gpu

DT = {"bf16": (torch.bfloat16, DType.BF16), "fp16": (torch.float16, DType.FP16)}


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def make_layers(fmt, dtype, E, K, N, gs=64, seed=0, bias=False, device="cuda"):
    """E packed layers of one kind and their dequantised weights [E, K, N] in float64 (on the CPU)."""
    g = _gen(seed)
    dt, gdt = DT[dtype]
    layers, weights = [], []
    for _ in range(E):
        b = (torch.randn(N, generator=g)).to(dt) if bias else None
        if fmt == "w4":
            q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.int32).to(torch.uint8)
            s = ((0.5 + torch.rand((N * K // gs, 1), generator=g)) / (4.6 * K ** 0.5)).to(dt)
            z = (torch.rand((N * K // gs, 1), generator=g) * 3 + 6).to(dt)
            layer = A16W4_HQQ_INT(device=device, dtype=dt).from_weights(q.to(device), s.to(device), z.to(device), bias=b)
            sc, zp = layer.scales.data.cpu().double(), layer.zeros.data.cpu().double()    # [K / gs, N], fma form
            q = q.t().double().view(K // gs, gs, N)
            if layer.channel_scale_mode == 1:   # one group for the whole of K: (q - z) s
                w = (q - zp[:, None, :]) * sc[:, None, :]
            else:
                w = q * sc[:, None, :] + zp[:, None, :]
            weights.append(w.reshape(K, N))
        elif fmt == "fp8":
            w = torch.randn((N, K), generator=g) / K ** 0.5
            layer = A8W8_fp8_dynamic(device=device, dtype=dt, block_quant=True)
            layer.fp8 = torch.float8_e4m3fn
            layer = layer.from_weights(w.to(device), bias=b)
            sc = layer.scales.data.cpu().double()
            full = sc.repeat_interleave(128, 0)[:K].repeat_interleave(128, 1)[:, :N]
            weights.append(layer.W_q.data.cpu().float().double() * full)
        else:
            w = (torch.randn((N, K), generator=g) / K ** 0.5).to(dt)
            layer = GemLiteLinear(16, None, K, N, gdt, gdt).pack(w.to(device), None, None, b.to(device) if bias else None)
            weights.append(w.t().double())
        layers.append(layer)
    return layers, torch.stack(weights)


def make_x(rows, K, dtype, seed=1):
    return torch.randn((rows, K), generator=_gen(seed)).to(DT[dtype][0])


def make_ids(T, E, k, seed=2, drop=0.0, only=None):
    g = _gen(seed)
    score = torch.rand((T, E), generator=g)
    if only is not None:
        score[:, only] += 10.0
    ids = torch.argsort(score, dim=1, descending=True)[:, :k].to(torch.int32)
    if drop:
        ids[torch.rand((T, k), generator=g) < drop] = -1
    return ids, torch.rand((T, k), generator=g) + 0.1


def ref_plan(ids, E):
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= E), torch.full_like(flat, E), flat)
    order = torch.sort(key, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel())
    offsets = torch.tensor([0] + [int((key == e).sum()) for e in range(E)]).cumsum(0)
    return offsets, order, places.view(ids.shape)


def quantised(x):
    """Rows as fp8 codes with a scale per 128 values, by the definition's fp32 steps; as float64."""
    b = x.float().view(x.shape[0], -1, 128)
    s = (b.abs().amax(2, keepdim=True) * torch.tensor(1 / 448, dtype=torch.float32)).clamp_min(1e-6)
    q = (b * (1.0 / s)).clamp(-448, 448).to(torch.float8_e4m3fn)
    return (q.float().double() * s.double()).view(x.shape)


def ref_rows(fmt, x, W, offsets, bias=None):
    """[R, N] products of rows sorted by expert and the sums of their magnitudes, in float64 (zeros without an expert)."""
    R, (E, K, N) = x.shape[0], W.shape
    xd = quantised(x) if fmt == "fp8" and R else x.double()
    y, mag = torch.zeros(R, N, dtype=torch.float64), torch.zeros(R, N, dtype=torch.float64)
    for e in range(E):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        y[lo:hi] = xd[lo:hi] @ W[e]
        mag[lo:hi] = xd[lo:hi].abs() @ W[e].abs()
        if bias is not None:
            y[lo:hi] += bias[e]
    return y, mag


def sum_slack(fmt, dtype, x, layers, mag, u):
    """How far an fp32 sum may be from the exact one (see the module's comment); per element or broadcast."""
    K = x.shape[1]
    slack = K * 2.0 ** -24 * mag
    if fmt == "w4":
        s = max(float(layer.scales.data.abs().max()) for layer in layers)
        z = max(float(layer.zeros.data.abs().max()) for layer in layers) * (s if layers[0].channel_scale_mode == 1 else 1.0)
        off = 128 if dtype == "bf16" else 1024
        slack = u * mag + K * 2.0 ** -24 * x.double().abs().sum(1, keepdim=True) * ((off + 15) * s + z)
    return slack


def silu(v):
    return v / (1 + torch.exp(-v))


def check(y, ref, slack, u, norm):
    y = y.cpu().double()
    assert y.shape == ref.shape
    err = (y - ref).abs()
    bound = u * ref.abs() + (1 + u) * slack + 1e-30
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"element off by {worst} of its bound"
    total = float(ref.norm())
    if total > 0:
        assert float(err.norm()) / total <= norm, f"norm error {float(err.norm()) / total} of {norm}"


def run_case(fmt, dtype, E, T, k, K, N, gs=64, drop=0.0, only=None, bias=False, tile_config=-1, seed=0, modes=("rows", "gated", "combined")):
    layers, W = make_layers(fmt, dtype, E, K, N, gs, seed, bias)
    experts = GemLiteExperts.from_layers(layers)
    B = None if not bias else torch.stack([layer.bias.data.cpu().double() for layer in layers])
    u = torch.finfo(DT[dtype][0]).eps / 2
    ids, w = make_ids(T, E, k, seed + 2, drop, only)
    offsets, order, places = ref_plan(ids, E)
    plan = gemlite_amd.plan_experts(ids.cuda(), w.cuda(), E)
    assert torch.equal(plan.offsets.cpu().long(), offsets) and torch.equal(plan.order.cpu().long(), order)
    assert torch.equal(plan.places.cpu().long(), places)
    x = make_x(T, K, dtype, seed + 1)
    targs, meta = experts.get_tensor_args(), experts.get_meta_args()
    xs = x[order // k]
    y, mag = ref_rows(fmt, xs, W, offsets, B)
    slack = sum_slack(fmt, dtype, xs, layers, mag, u)
    if "rows" in modes:
        out = gemlite_amd.experts_functional(xs.cuda(), experts.bias, targs, meta, plan.offsets, tile_config=tile_config)
        check(out, y, slack, u, u)
        assert not out[int(offsets[E]):].any()
    if "gated" in modes:
        out = gemlite_amd.experts_gated_functional(x.cuda(), experts.bias, targs, meta, plan, tile_config=tile_config)
        g, up, half = y[:, : N // 2], y[:, N // 2:], slack.expand(y.shape)
        dg, du = half[:, : N // 2], half[:, N // 2:]
        # (and the fp32 arithmetic of silu: a handful of roundings of 2^-24, the exponential's argument up to 2^-18)
        s = 1.1 * up.abs() * dg + silu(g).abs() * du + 1.1 * dg * du + 2.0 ** -16 * (silu(g) * up).abs()
        check(out, silu(g) * up, s, u, 1.5 * u if fmt == "w4" else u)
        assert not out[int(offsets[E]):].any()
    if "combined" in modes:
        out = gemlite_amd.experts_combined_functional(xs.cuda(), experts.bias, targs, meta, plan, tile_config=tile_config)
        live = (ids >= 0).double() * w.double()
        take = lambda t: (t.expand(y.shape)[places.reshape(-1)].view(T, k, -1) * live[:, :, None])   # noqa: E731
        ref = take(y).sum(1)
        check(out, ref, take(slack).sum(1) + (k + 1) * 2.0 ** -24 * take(y.abs()).sum(1), u, u)
    return experts


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------
def ref_route(logits, k, scoring, renormalize, scale):
    x = logits.double().clone()
    T, E = x.shape
    x[torch.isnan(x)] = float("-inf")
    order = torch.sort(x, dim=1, descending=True, stable=True)
    best, ids = order.values[:, :k], order.indices[:, :k].clone()
    none = best == float("-inf")
    if scoring == "sigmoid":
        p = 1 / (1 + torch.exp(-best))
        total = p.masked_fill(none, 0).sum(1, keepdim=True)
    else:
        top = best[:, :1]
        e = torch.where(best == top, torch.ones_like(best), torch.exp(best - top)).masked_fill(none, 0)
        every = torch.where(x == top, torch.ones_like(x), torch.exp(x - top)).masked_fill(x == float("-inf"), 0)
        p, total = e, (e if renormalize else every).sum(1, keepdim=True)
    p = p.masked_fill(none, 0)
    if renormalize or scoring == "softmax":
        p = torch.where(total > 0, p / total, torch.zeros_like(p))
    return p * scale, ids.masked_fill(none, -1)


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (1, 1, 1), (3, 60, 6), (64, 64, 8), (128, 128, 8), (129, 128, 8), (1024, 1, 1), (1025, 2, 1),
                                    (17, 1024, 64), (500, 256, 8), (2000, 160, 6), (4097, 100, 3), (9001, 128, 8), (40000, 8, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_route(T, E, k, dtype):
    g = _gen(T + E)
    logits = (2 * torch.randn((T, E), generator=g)).to(dtype)   # 16-bit logits: many ties
    logits[torch.rand((T, E), generator=g) < 0.1] = float("-inf")
    for scoring, renormalize, scale in (("softmax", True, 1.0), ("softmax", False, 2.5), ("sigmoid", True, 1.0), ("sigmoid", False, 1.0)):
        plan = gemlite_amd.route_experts(logits.cuda(), k, scoring, renormalize, scale)
        w, ids = ref_route(logits, k, scoring, renormalize, scale)
        assert torch.equal(plan.expert_ids.cpu().long(), ids)
        # exp of a difference below 32 (2^-19 off), a sum of up to E of them, one division
        np.testing.assert_allclose(plan.weights.cpu().double().numpy(), w.numpy(), rtol=2.0 ** -18 + E * 2.0 ** -24, atol=1e-37)
        offsets, order, places = ref_plan(ids, E)
        assert torch.equal(plan.offsets.cpu().long(), offsets)
        assert torch.equal(plan.order.cpu().long(), order)
        assert torch.equal(plan.places.cpu().long(), places)


def test_route_special_values():
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[nan, 1.0, -inf, 1.0], [-inf] * 4, [nan] * 4, [inf, 0.0, inf, 5.0], [0.0, -0.0, 0.0, -0.0],
                           [-3e38, 3e38, -3e38, 1.0], [-inf, -inf, 2.0, -inf]])
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            plan = gemlite_amd.route_experts(logits.cuda(), 3, scoring, renormalize)
            w, ids = ref_route(logits, 3, scoring, renormalize, 1.0)
            assert torch.equal(plan.expert_ids.cpu().long(), ids)
            np.testing.assert_allclose(plan.weights.cpu().double().numpy(), w.numpy(), rtol=1e-6, atol=1e-37)


def test_route_strided_logits_and_no_tokens():
    wide = torch.randn((50, 40), generator=_gen(3))
    for view in (wide[:, 3:19], wide[::2, :16], wide.t()[:16].t(), wide[:, :16].t().contiguous().t()):
        plan = gemlite_amd.route_experts(view.cuda() if view.is_contiguous() else view.cuda(), 2)
        assert torch.equal(plan.expert_ids.cpu().long(), ref_route(view, 2, "softmax", True, 1.0)[1])
    on_gpu = wide.cuda()
    for view, cpu in ((on_gpu[:, 3:19], wide[:, 3:19]), (on_gpu[::2, :16], wide[::2, :16]), (on_gpu.t()[:16].t(), wide[:, :16])):
        assert torch.equal(gemlite_amd.route_experts(view, 2).expert_ids.cpu().long(), ref_route(cpu, 2, "softmax", True, 1.0)[1])
    plan = gemlite_amd.route_experts(torch.empty((0, 16), device="cuda"), 2)
    assert plan.weights.shape == (0, 2) and plan.order.shape == (0,) and not plan.offsets.any() and plan.offsets.shape == (17,)


@pytest.mark.parametrize("T,k", [(5, 2), (700, 4)])
def test_plan_of_foreign_ids(T, k):
    """Ids of another rank's experts, repeated ids and ids that 32 bits cannot hold."""
    g = _gen(T)
    ids = torch.randint(-3, 12, (T, k), generator=g)
    ids[0, 0], ids[T - 1, k - 1], ids[T // 2, 0] = 2 ** 40, -2 ** 40, 2 ** 32 + 1
    plan = gemlite_amd.plan_experts(ids.cuda(), torch.ones((T, k), device="cuda"), 8)
    offsets, order, places = ref_plan(ids, 8)
    assert torch.equal(plan.offsets.cpu().long(), offsets) and torch.equal(plan.order.cpu().long(), order)
    assert torch.equal(plan.places.cpu().long(), places)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
FORMATS = ["w4", "fp8", "h16"]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("E,T,k,K,N,gs", [(4, 1, 2, 256, 64, 64), (8, 5, 3, 384, 208, 128), (3, 70, 2, 640, 144, 32), (130, 40, 4, 128, 32, 64),
                                          (16, 300, 4, 256, 272, 128), (2, 600, 1, 512, 96, 64), (1, 33, 1, 1152, 112, 64)])
def test_products(fmt, dtype, E, T, k, K, N, gs):
    run_case(fmt, dtype, E, T, k, K, N, gs, drop=0.1 if T > 4 else 0.0)


@pytest.mark.parametrize("fmt", ["w4", "h16"])
@pytest.mark.parametrize("K,gs", [(32, 32), (96, 32), (160, 32), (192, 192), (320, 64), (480, 96), (416, 416)])
def test_ragged_k(fmt, K, gs):
    """K that ends inside a pipeline stage, groups that are no power of two, one group for the whole of K."""
    for T, k in ((2, 1), (90, 2)):
        run_case(fmt, "bf16", 3, T, k, K, 80, gs)
        run_case(fmt, "fp16", 3, T, k, K, 80, gs)


@pytest.mark.parametrize("fmt", FORMATS)
def test_one_expert_gets_everything(fmt):
    run_case(fmt, "bf16", 6, 150, 1, 256, 96, only=4)


@pytest.mark.parametrize("fmt", FORMATS)
def test_no_slot_has_an_expert(fmt):
    run_case(fmt, "bf16", 6, 20, 2, 256, 96, drop=2.0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_bias(fmt, dtype):
    for T in (3, 200):
        run_case(fmt, dtype, 4, T, 2, 256, 160, drop=0.2, bias=True)


TILES = [4, 16, 2016, 3004, 64, 128, 256]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tile_config", TILES)
def test_every_kernel_variant(fmt, dtype, tile_config):
    for T, K, N, gs in ((1, 512, 144, 128), (77, 1024, 272, 64), (330, 384, 528, 32)):
        run_case(fmt, dtype, 5, T, 2, K, N, gs, drop=0.05, tile_config=tile_config, bias=T == 77)


@pytest.mark.parametrize("gs", [32, 64, 128])
def test_many_column_tiles_of_4_bit_weights(gs):
    """Enough workgroups for two-wave ones (K of 16 units and more), a K range that does not divide evenly."""
    run_case("w4", "bf16", 8, 40, 2, 2176, 6240, gs, drop=0.1)


# ---------------------------------------------------------------------------
# operands as callers have them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
def test_strided_and_misaligned_activations(fmt):
    E, T, k, K, N = 4, 37, 2, 256, 96
    layers, _ = make_layers(fmt, "bf16", E, K, N)
    experts = GemLiteExperts.from_layers(layers)
    ids, w = make_ids(T, E, k)
    plan = gemlite_amd.plan_experts(ids.cuda(), w.cuda(), E)
    x = make_x(T, K, "bf16").cuda()
    want = experts.forward_gated(x, plan)
    wide = torch.zeros((T, K + 24), dtype=x.dtype, device="cuda")
    for lo in (0, 8, 3, 16):            # rows 16-byte aligned, then rows that are not
        view = wide[:, lo:lo + K]
        view.copy_(x)
        assert torch.equal(experts.forward_gated(view, plan), want)
    odd = torch.zeros((T, K + 5), dtype=x.dtype, device="cuda")[:, :K]
    odd.copy_(x)
    assert torch.equal(experts.forward_gated(odd, plan), want)
    assert torch.equal(experts.forward_gated(x.t().contiguous().t(), plan), want)
    flat = torch.zeros(T * K + 1, dtype=x.dtype, device="cuda")[1:].view(T, K)
    flat.copy_(x)
    assert torch.equal(experts.forward_gated(flat, plan), want)
    every_second = torch.zeros((2 * T, K), dtype=x.dtype, device="cuda")[::2]
    every_second.copy_(x)
    assert torch.equal(experts.forward_gated(every_second, plan), want)


def _moe(fmt, dtype, E, hidden, inter, seed=0):
    up, Wu = make_layers(fmt, dtype, E, hidden, 2 * inter, 64, seed)
    down, Wd = make_layers(fmt, dtype, E, inter, hidden, 64, seed + 50)
    return GemLiteExperts.from_layers(up), GemLiteExperts.from_layers(down), Wu, Wd


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 9, 250])
def test_block_of_experts(fmt, T):
    """Routing and both products as a module runs them, against 64 bits."""
    E, k, hidden, inter = 8, 2, 256, 128
    gate_up, down, Wu, Wd = _moe(fmt, "bf16", E, hidden, inter)
    moe = GemLiteMoE(gate_up, down, k)
    x = make_x(T, hidden, "bf16")
    logits = torch.randn((T, E), generator=_gen(5))
    y = moe(x.cuda().view(1, T, hidden), logits.cuda().view(1, T, E)).cpu().double()
    w, ids = ref_route(logits, k, "softmax", True, 1.0)
    ref = torch.zeros((T, hidden), dtype=torch.float64)
    xd = quantised(x) if fmt == "fp8" else x.double()
    for t in range(T):
        for j in range(k):
            z = xd[t] @ Wu[ids[t, j]]
            h = (silu(z[:inter]) * z[inter:]).to(torch.bfloat16)
            hd = quantised(h[None])[0] if fmt == "fp8" else h.double()
            ref[t] += w[t, j] * (hd @ Wd[ids[t, j]])
    assert y.shape == (1, T, hidden)
    # h is rounded to bf16 on both sides but from sums that differ by fp32 or, for rounded 4-bit weights, bf16 noise: up to
    # one more rounding of h (and, fp8, of its codes: 2^-4 of the few that cross a border) and one of the result
    u = 2.0 ** -9
    assert float((y[0] - ref).norm() / ref.norm()) <= (2 * u if fmt != "fp8" else 4 * u) * 2


def test_graph_replays_equal_eager_calls():
    E, k, hidden, inter, T = 8, 2, 256, 128, 24
    for fmt in FORMATS:
        gate_up, down, _, _ = _moe(fmt, "fp16", E, hidden, inter)
        moe = GemLiteMoE(gate_up, down, k)
        x, logits = make_x(T, hidden, "fp16").cuda(), torch.randn((T, E), generator=_gen(1)).cuda()
        moe(x, logits)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = moe(x, logits)
        other = torch.cuda.CUDAGraph()
        x2, logits2 = make_x(T, hidden, "fp16", 9).cuda(), torch.randn((T, E), generator=_gen(9)).cuda()
        with torch.cuda.graph(other):
            y2 = moe(x2, logits2)
        for i in range(4):
            x.copy_(make_x(T, hidden, "fp16", 20 + i).cuda())
            logits.copy_(torch.randn((T, E), generator=_gen(30 + i)).cuda())
            want, want2 = moe(x, logits), moe(x2, logits2)
            torch.cuda.synchronize()
            graph.replay()
            other.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(y2, want2)


def test_streams_and_threads_do_not_share_scratch():
    import threading

    E, k, hidden, inter, T = 8, 4, 256, 128, 100
    gate_up, down, _, _ = _moe("w4", "bf16", E, hidden, inter)
    moe = GemLiteMoE(gate_up, down, k)
    inputs = [(make_x(T, hidden, "bf16", s).cuda(), torch.randn((T, E), generator=_gen(s)).cuda()) for s in range(4)]
    want = [moe(*i) for i in inputs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[n] = moe(*inputs[n])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_that_are_not_a_plan(fmt):
    """Whatever offsets, order and places hold, rows outside the call are neither read nor written."""
    E, R, K, N = 4, 40, 128, 64
    layers, _ = make_layers(fmt, "bf16", E, K, N)
    e = GemLiteExperts.from_layers(layers)
    x = make_x(R, K, "bf16").cuda()
    good = torch.tensor([0, 10, 20, 30, 40], dtype=torch.int32, device="cuda")
    full = e(x, good)
    for off in ([0, 10, 20, 30, 10 ** 6], [-5, 10, 20, 30, 40]):
        assert torch.equal(e(x, torch.tensor(off, dtype=torch.int32, device="cuda")), full)
    y = e(x, torch.tensor([0, 10, 20, 30, 33], dtype=torch.int32, device="cuda"))
    assert torch.equal(y[:33], full[:33]) and not y[33:].any()
    for off in ([40, 0, 40, 0, 40], [7, 7, 7, 7, 7]):
        assert e(x, torch.tensor(off, dtype=torch.int32, device="cuda")).shape == (R, N)
    big = torch.full((R,), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    plan = ExpertPlan(torch.ones((R // 2, 2), device="cuda"), big.view(-1, 2), good, big, big.view(-1, 2))
    assert e.forward_gated(x[: R // 2], plan).shape == (R, N // 2)
    assert not e.forward_combined(x, plan).any()      # no place is one of the rows
    plan = plan._replace(order=-big, places=-big.view(-1, 2))
    e.forward_gated(x[: R // 2], plan)
    assert not e.forward_combined(x, plan).any()
    torch.cuda.synchronize()


def test_values_that_are_not_finite_stay_in_their_rows():
    """A row with an infinity or a NaN changes no other row, and slots without an expert are not looked at."""
    for fmt in FORMATS:
        E, T, k, K, N = 4, 20, 2, 256, 64
        layers, _ = make_layers(fmt, "bf16", E, K, N)
        e = GemLiteExperts.from_layers(layers)
        ids, w = make_ids(T, E, k)
        plan = gemlite_amd.plan_experts(ids.cuda(), w.cuda(), E)
        x = make_x(T, K, "bf16")
        clean = e.forward_gated(x.cuda(), plan).cpu()
        x[3, 7], x[11, 100] = float("inf"), float("nan")
        dirty = e.forward_gated(x.cuda(), plan).cpu()
        rows = plan.order.cpu() // k
        ok = (rows != 3) & (rows != 11)
        assert torch.equal(clean[ok], dirty[ok]) and not torch.isfinite(dirty[rows == 11].float()).any()
        ids[5, 1] = -1
        plan = gemlite_amd.plan_experts(ids.cuda(), w.cuda(), E)
        h = make_x(T * k, K, "bf16").cuda()
        y = e.forward_combined(h, plan)
        h[int(plan.places[5, 1])] = float("nan")
        weights = plan.weights.clone()
        weights[5, 1] = float("nan")
        assert torch.equal(e.forward_combined(h, plan._replace(weights=weights)), y)


def test_empty_calls():
    for fmt in FORMATS:
        layers, _ = make_layers(fmt, "bf16", 4, 128, 64)
        e = GemLiteExperts.from_layers(layers)
        x = torch.empty((0, 128), dtype=torch.bfloat16, device="cuda")
        assert e(x, torch.zeros(5, dtype=torch.int32, device="cuda")).shape == (0, 64)
        plan = gemlite_amd.route_experts(torch.empty((0, 4), device="cuda"), 2)
        assert e.forward_gated(x, plan).shape == (0, 32) and e.forward_combined(x, plan).shape == (0, 64)


def test_refusals_on_the_gpu():
    layers, _ = make_layers("w4", "bf16", 4, 128, 64)
    e = GemLiteExperts.from_layers(layers)
    x = make_x(8, 128, "bf16").cuda()
    off = torch.tensor([0, 2, 4, 6, 8], dtype=torch.int32, device="cuda")
    plan = gemlite_amd.route_experts(torch.zeros((4, 4), device="cuda"), 2)
    for bad, exc in ((lambda: e(x[:, :64], off), ValueError), (lambda: e(x.float(), off), NotImplementedError), (lambda: e(x.half(), off), NotImplementedError),
                     (lambda: e(x, off.long()), ValueError), (lambda: e(x, off[:4]), ValueError), (lambda: e(x, off.cpu()), RuntimeError),
                     (lambda: e.forward_gated(x, plan), ValueError), (lambda: e.forward_combined(x[:4], plan), ValueError),
                     (lambda: e.forward_combined(x, plan._replace(weights=plan.weights.half())), ValueError),
                     (lambda: e.forward_combined(x, plan._replace(places=plan.places.t())), ValueError),
                     (lambda: e.forward_gated(x[:4], plan._replace(order=plan.order[::2])), ValueError),
                     (lambda: gemlite_amd.route_experts(torch.zeros((4, 4), device="cuda"), 5), ValueError),
                     (lambda: gemlite_amd.route_experts(torch.zeros((4, 4), device="cuda", dtype=torch.float64), 2), NotImplementedError),
                     (lambda: gemlite_amd.route_experts(torch.zeros((4, 2000), device="cuda"), 2), ValueError)):
        for _ in range(2):   # the second time as the first: nothing refused is remembered as accepted
            with pytest.raises(exc):
                bad()
    assert e(x, off).shape == (8, 64)


def test_compiled_module_equals_the_eager_one():
    E, k, hidden, inter, T = 8, 2, 256, 128, 12
    for fmt in FORMATS:
        gate_up, down, _, _ = _moe(fmt, "bf16", E, hidden, inter)
        moe = GemLiteMoE(gate_up, down, k)
        x, logits = make_x(T, hidden, "bf16").cuda(), torch.randn((T, E), generator=_gen(1)).cuda()
        graphs = []

        def backend(graph, _):
            graphs.append(graph)
            return graph.forward

        compiled = torch.compile(moe, backend=backend, fullgraph=True)
        assert torch.equal(compiled(x, logits), moe(x, logits))
        names = [str(n.target) for g in graphs for n in g.graph.nodes if n.op == "call_function"]
        assert sum("route_experts" in n for n in names) == 1 and sum("gemlite.experts" in n for n in names) == 2


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile_config", [4, 16, 64, 128, 256])
def test_a_nan_reaches_its_row_in_every_kernel(fmt, tile_config):
    E, T, k, K, N = 2, 30, 1, 256, 64
    layers, _ = make_layers(fmt, "bf16", E, K, N)
    e = GemLiteExperts.from_layers(layers)
    off = torch.tensor([0, 13, 30], dtype=torch.int32, device="cuda")
    x = make_x(T, K, "bf16").cuda()
    args = (None, e.get_tensor_args(), e.get_meta_args(), off)
    clean = gemlite_amd.experts_functional(x, *args, tile_config=tile_config)
    x[20, 200] = float("nan")
    dirty = gemlite_amd.experts_functional(x, *args, tile_config=tile_config)
    rest = torch.arange(T, device="cuda") != 20
    assert torch.equal(clean[rest], dirty[rest]) and bool(torch.isnan(dirty[20].float()).all())
