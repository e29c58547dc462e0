"""Mixture-of-experts operators without a GPU: ABI, refusals, stacking of layers, checkpoints, fake implementations."""
import ctypes
import os

import pytest
import torch

import gemlite_amd
from gemlite_amd import DType, ExpertPlan, GemLiteExperts, GemLiteLinear, GemLiteMoE, _ext
from gemlite_amd.helper import A16W4_HQQ_INT, A8W8_fp8_dynamic, A8W8_int8_dynamic

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_matches_header():
    header = open(os.path.join(ROOT, "include", "gemlite_amd.h")).read()
    body = header[header.index("typedef struct gla_experts_args {"): header.index("} gla_experts_args;")]
    names, comment = [], False
    for line in body.splitlines()[1:]:
        if comment:
            comment = "*/" not in line
            continue
        comment = "/*" in line and "*/" not in line
        line = line.split("/*")[0].strip()
        if not line.endswith(";"):
            continue
        for part in line[:-1].split(",") if "*" not in line else [line[:-1]]:
            names.append(part.strip().split()[-1].lstrip("*"))
    assert names == [f[0] for f in _ext.ExpertsArgs._fields_]


def _args(**kw):
    """Valid 4-bit arguments; the addresses are never dereferenced on the host."""
    a = _ext.ExpertsArgs()
    a.struct_size = ctypes.sizeof(_ext.ExpertsArgs)
    a.mode, a.R, a.T, a.top_k, a.E, a.N, a.K = 0, 8, 4, 2, 4, 64, 256
    a.x = a.w = a.out = a.offsets = a.order = a.places = a.weights = a.scales = a.zeros = 4096
    a.w_stride_e, a.meta_stride_e, a.x_stride_m, a.out_stride_m = 256 * 64 // 2, 2 * 64 * 2, 256, 64
    a.W_nbits, a.group_size, a.elements_per_sample = 4, 128, 8
    a.input_dtype = a.output_dtype = a.meta_dtype = a.x_dtype = DType.BF16.value
    a.W_group_mode, a.tile_config = 4, -1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(struct_size=4), -1), (dict(mode=3), -3), (dict(E=0), -1), (dict(E=2000), -1), (dict(R=-1), -1), (dict(N=60), -4), (dict(K=240), -4),
    (dict(mode=1, N=56, out_stride_m=28), -4), (dict(output_dtype=0), -2), (dict(x_dtype=1), -2), (dict(W_nbits=2), -3),
    (dict(channel_scale_mode=1), -3), (dict(group_size=48), -4), (dict(group_size=96), -4), (dict(W_group_mode=1), -3), (dict(meta_dtype=0), -2),
    (dict(scales=None), -1), (dict(K=1 << 21, N=8, out_stride_m=8, x_stride_m=1 << 21, w_stride_e=1 << 24), -1), (dict(zeros=None), -1), (dict(x=None), -1), (dict(offsets=None), -1), (dict(x=4104), -1), (dict(x_stride_m=252), -1),
    (dict(x_stride_m=128), -1), (dict(out_stride_m=32), -1), (dict(out=4100), -1), (dict(w_stride_e=16), -1), (dict(mode=1, order=None), -1),
    (dict(mode=2, places=None), -1), (dict(mode=2, weights=None), -1), (dict(mode=1, T=3), -1), (dict(mode=2, top_k=0), -1), (dict(tile_config=7), -1),
    (dict(tile_config=-3), -1), (dict(tile_config=99016), -1), (dict(N=1 << 20, K=1 << 14, w_stride_e=1 << 34, out_stride_m=1 << 20, x_stride_m=1 << 14), -3),
    (dict(W_nbits=8, elements_per_sample=1, input_dtype=3, channel_scale_mode=5, W_group_mode=0, meta_dtype=1), -1),
    (dict(W_nbits=8, elements_per_sample=1, input_dtype=3, channel_scale_mode=5, W_group_mode=0, K=96, meta_dtype=0), -4),
    (dict(W_nbits=8, elements_per_sample=1, input_dtype=4, channel_scale_mode=5, W_group_mode=0, meta_dtype=0), -3)])
def test_library_refuses(change, status):
    lib = _ext.load_library()
    good, bad = _args(), _args(**change)
    assert lib.gla_experts_workspace_bytes(ctypes.byref(good)) >= 0
    assert lib.gla_experts_workspace_bytes(ctypes.byref(bad)) == status
    assert lib.gla_experts_matmul(ctypes.byref(bad), None) == status
    assert lib.gla_last_error()


def test_library_refuses_a_small_workspace_and_null():
    lib = _ext.load_library()
    a = _args(mode=2)
    assert lib.gla_experts_workspace_bytes(ctypes.byref(a)) >= 8 * 64 * 4
    assert lib.gla_experts_matmul(ctypes.byref(a), None) == -5
    a.workspace, a.workspace_bytes = 4100, 1 << 20
    assert lib.gla_experts_matmul(ctypes.byref(a), None) == -5   # not aligned
    assert lib.gla_experts_matmul(None, None) == -1
    assert lib.gla_experts_matmul(ctypes.byref(_args(R=0, x=None, out=None)), None) == 0   # nothing to do


def test_library_refuses_routes():
    lib = _ext.load_library()
    p = 4096

    def route(logits=p, dtype=0, stride=8, T=4000, E=8, k=2, scoring=0, ws=p, n=1 << 20, offsets=p):
        return lib.gla_route_experts(logits, dtype, stride, T, E, k, scoring, 1, 1.0, p, p, offsets, p, p, ws, n, None)

    assert route(T=-1) == -1 and route(E=0) == -1 and route(E=1025) == -1 and route(k=0) == -1 and route(k=65, E=100) == -1
    assert route(k=9) == -1 and route(scoring=2) == -1 and route(dtype=4) == -2 and route(stride=7) == -1 and route(logits=None) == -1
    assert route(ws=None) == -5 and route(n=16) == -5 and route(ws=p + 4) == -5 and route(offsets=None) == -1
    assert route(T=1 << 30, k=4) == -1
    assert lib.gla_plan_experts(None, 4, 8, 2, p, p, p, p, 1 << 20, None) == -1
    assert lib.gla_plan_experts(p, 4000, 8, 2, p, p, p, p, 8, None) == -5
    assert lib.gla_route_workspace_bytes(4, 0, 1) == -1 and lib.gla_route_workspace_bytes(0, 8, 1) == 0
    assert lib.gla_route_workspace_bytes(4000, 8, 2) > 0


def _w4_layers(E=3, K=128, N=32, gs=64, bias=False, dtype=torch.float16):
    g = torch.Generator().manual_seed(0)
    out = []
    for _ in range(E):
        q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.int32).to(torch.uint8)
        n = N * K // gs
        out.append(A16W4_HQQ_INT(device="cpu", dtype=dtype).from_weights(q, torch.rand((n, 1), generator=g).to(dtype), torch.rand((n, 1), generator=g).to(dtype),
                                                                          bias=torch.rand(N, generator=g) if bias else None))
    return out


def test_stacking_keeps_the_layers_tensors():
    layers = _w4_layers(bias=True)
    e = GemLiteExperts.from_layers(layers)
    assert (e.num_experts, e.in_features, e.out_features) == (3, 128, 32)
    for i, layer in enumerate(layers):
        assert torch.equal(e.W_q[i], layer.W_q) and torch.equal(e.scales[i], layer.scales) and torch.equal(e.zeros[i], layer.zeros)
        assert torch.equal(e.bias[i], layer.bias.float())
    assert e.get_meta_args() == layers[0].get_meta_args()
    wide = [A8W8_fp8_dynamic(device="cpu", fp8=torch.float8_e4m3fn, block_quant=True).from_weights(torch.randn(160, 256).bfloat16()) for _ in range(2)]
    e = GemLiteExperts.from_layers(wide)
    assert e.W_q.shape == (2, 256, 160) and e.W_q.stride() == (256 * 160, 1, 256) and e.scales.shape == (2, 2, 2)
    raw = [GemLiteLinear(16, None, 64, 32, DType.BF16, DType.BF16).pack(torch.randn(32, 64).bfloat16(), None, None) for _ in range(2)]
    e = GemLiteExperts.from_layers(raw)
    assert e.W_q.stride() == (64 * 32, 1, 64) and torch.equal(e.W_q[1], raw[1].W_q)


def test_stacking_of_channelwise_layers_and_scalar_zeros():
    q = torch.randint(0, 16, (32, 64), dtype=torch.int32).to(torch.uint8)
    s = torch.rand((32, 1)).half()
    layer = A16W4_HQQ_INT(device="cpu").from_weights(q, s, 7 * torch.ones((32, 1)).half())
    e = GemLiteExperts.from_layers([layer])
    assert e.meta_args[2] == 64 and e.meta_args[9:11] == [0, 3] and torch.equal(e.zeros[0], 7 * torch.ones((1, 32)).half())
    layer = GemLiteLinear(4, 32, 64, 32, DType.FP16, DType.FP16).pack(q, torch.rand((64, 1)).half(), 8)
    e = GemLiteExperts.from_layers([layer])
    assert e.meta_args[10] == 3 and e.zeros.shape == e.scales.shape and bool((e.zeros == 8).all())
    layer = GemLiteLinear(4, 32, 64, 32, DType.BF16, DType.BF16).pack(q, torch.rand((64, 1)).bfloat16(), 259)
    with pytest.raises(NotImplementedError, match="zero point"):
        GemLiteExperts.from_layers([layer])


def test_stacking_refuses():
    layers = _w4_layers()
    with pytest.raises(ValueError, match="non-empty"):
        GemLiteExperts.from_layers([])
    with pytest.raises(ValueError, match="non-empty"):
        GemLiteExperts.from_layers([torch.nn.Linear(4, 4)])
    with pytest.raises(ValueError, match="kind or shape"):
        GemLiteExperts.from_layers(layers + _w4_layers(E=1, N=40))
    with pytest.raises(ValueError, match="kind or shape"):
        GemLiteExperts.from_layers(layers + _w4_layers(E=1, gs=32))
    with pytest.raises(ValueError, match="bias"):
        GemLiteExperts.from_layers(layers + _w4_layers(E=1, bias=True))
    int8 = A8W8_int8_dynamic(device="cpu", block_quant=True).from_weights(torch.randn(128, 128).half())
    with pytest.raises(NotImplementedError, match="not\\s+built"):
        GemLiteExperts.from_layers([int8])
    with pytest.raises(NotImplementedError, match="not\\s+built"):
        GemLiteExperts.from_layers([GemLiteLinear(2, 64, 64, 32).pack(torch.zeros((32, 64), dtype=torch.uint8), torch.ones((32, 1)).half(), 1)])


@pytest.mark.parametrize("kind", ["w4", "fp8", "h16"])
@pytest.mark.parametrize("strides", [True, False])
def test_state_dict_round_trip(kind, strides, tmp_path):
    if kind == "w4":
        layers = _w4_layers(bias=True)
    elif kind == "fp8":
        layers = [A8W8_fp8_dynamic(device="cpu", fp8=torch.float8_e4m3fn, block_quant=True).from_weights(torch.randn(160, 256).bfloat16()) for _ in range(2)]
    else:
        layers = [GemLiteLinear(16, None, 64, 32, DType.BF16, DType.BF16).pack(torch.randn(32, 64).bfloat16(), None, None) for _ in range(2)]
    e = GemLiteExperts.from_layers(layers)
    model = torch.nn.Sequential(e)
    sd = model.state_dict()
    if not strides:   # as a format without strides keeps it
        sd = {k: (v.view(torch.uint8).contiguous().view(v.dtype) if v.dtype == torch.float8_e4m3fn else v.contiguous()) for k, v in sd.items()}
    torch.save(sd, tmp_path / "m.pt")
    other = torch.nn.Sequential(GemLiteExperts())
    other.load_state_dict(torch.load(tmp_path / "m.pt", weights_only=True))
    o = other[0]
    assert o.meta_args == e.meta_args and o.W_q.stride() == e.W_q.stride() and (o.num_experts, o.in_features, o.out_features) == (
        e.num_experts, e.in_features, e.out_features)
    for name in ("W_q", "scales", "zeros", "bias"):
        a, b = getattr(e, name), getattr(o, name)
        assert (a is None and b is None) or torch.equal(a.float(), b.float())
    with pytest.raises(RuntimeError, match="missing|Missing"):
        torch.nn.Sequential(GemLiteExperts()).load_state_dict({})


def test_python_refuses():
    with pytest.raises(RuntimeError, match="GPU only"):
        gemlite_amd.route_experts(torch.zeros(2, 4), 1)
    with pytest.raises(ValueError, match="tokens, experts"):
        gemlite_amd.route_experts(torch.zeros(4), 1)
    with pytest.raises(ValueError, match="scoring"):
        gemlite_amd.route_experts(torch.zeros(2, 4), 1, scoring="tanh")
    with pytest.raises(ValueError, match="expert_ids"):
        gemlite_amd.plan_experts(torch.zeros(2, 4), torch.zeros(2, 4), 8)
    with pytest.raises(ValueError, match="weights"):
        gemlite_amd.plan_experts(torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 3), 8)
    e = GemLiteExperts.from_layers(_w4_layers())
    with pytest.raises(RuntimeError, match="GPU only"):
        e(torch.zeros(4, 128).half(), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="rows, K"):
        e(torch.zeros(128).half(), torch.zeros(4, dtype=torch.int32))
    down = GemLiteExperts.from_layers(_w4_layers(K=64, N=32))
    with pytest.raises(ValueError, match="belong together"):
        GemLiteMoE(e, down, 2)
    with pytest.raises(ValueError, match="scoring"):
        GemLiteMoE(GemLiteExperts.from_layers(_w4_layers(N=128)), down, 2, scoring="x")


def test_fake_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode

    e = GemLiteExperts.from_layers(_w4_layers(N=128))
    with FakeTensorMode(allow_non_fake_inputs=True):
        logits, x = torch.empty((5, 3)), torch.empty((5, 128), dtype=torch.float16)
        plan = torch.ops.gemlite.route_experts(logits, 2, "softmax", True, 1.0)
        assert [tuple(t.shape) for t in plan] == [(5, 2), (5, 2), (4,), (10,), (5, 2)] and plan[0].dtype == torch.float32
        h = torch.ops.gemlite.experts(1, x, None, e.get_tensor_args(), e.meta_args, plan[2], plan)
        assert h.shape == (10, 64) and h.dtype == torch.float16
        y = torch.ops.gemlite.experts(2, torch.empty((10, 128), dtype=torch.float16), None, e.get_tensor_args(), e.meta_args, plan[2], plan)
        assert y.shape == (5, 128)
        assert torch.ops.gemlite.experts(0, x, None, e.get_tensor_args(), e.meta_args, plan[2], []).shape == (5, 128)
