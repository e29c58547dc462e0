"""Mixture-of-experts calls without a GPU: operands that do not belong together, sizes at the limits, what a compiled call
hands on.  The device check and the launches are replaced, so nothing runs."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import gemlite_amd
from gemlite_amd import DType, ExpertPlan, GemLiteExperts, GemLiteLinear, GemLiteMoE, _ext, experts as experts_module

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def launches(monkeypatch):
    """Operands on the CPU pass the device check; what would be launched is recorded."""
    calls = []
    monkeypatch.setattr(_ext, "_require_cuda", lambda *tensors: None)
    monkeypatch.setattr(_ext, "experts_matmul", lambda args, need, x: calls.append((args, need)))
    return calls


def _raw_experts(dtype, E=2, K=64, N=32):
    code = {torch.float16: DType.FP16, torch.bfloat16: DType.BF16}[dtype]
    return GemLiteExperts.from_layers([GemLiteLinear(16, None, K, N, code, code).pack(torch.randn(N, K).to(dtype), None, None) for _ in range(E)])


@pytest.mark.parametrize("dtype,other", [(torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)])
def test_unquantised_weights_of_another_type_than_the_activations(launches, dtype, other):
    """A cast of the module changes its tensors and not what its meta_args say: the bits of one type are not read as the other."""
    x, off = torch.zeros((4, 64), dtype=dtype), torch.tensor([0, 2, 4], dtype=torch.int32)
    e = _raw_experts(dtype)
    assert e(x, off).shape == (4, 32) and len(launches) == 1
    cast = _raw_experts(dtype).to(other)
    for rows in (x, x.to(other)):
        with pytest.raises(NotImplementedError):
            cast(rows, off)
    with pytest.raises(NotImplementedError):
        gemlite_amd.experts_functional(x, None, [e.W_q.to(other), e.scales, e.zeros], e.get_meta_args(), off)
    assert len(launches) == 1


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


def test_tokens_without_slots_are_refused(launches):
    """Tokens whose plan has no slots have no rows: the combination would return memory that nothing has written."""
    lib = _ext.load_library()
    for mode in (1, 2):
        for top_k in (0, 2, -1):
            bad = _args(mode=mode, R=0, T=5, top_k=top_k)
            assert lib.gla_experts_workspace_bytes(ctypes.byref(bad)) == -1 and lib.gla_experts_matmul(ctypes.byref(bad), None) == -1
        assert lib.gla_experts_matmul(ctypes.byref(_args(mode=mode, R=0, T=0, top_k=2)), None) == 0
    e = _raw_experts(torch.bfloat16)
    none = torch.empty(0, dtype=torch.int32)
    plan = ExpertPlan(torch.empty((5, 0)), none.view(5, 0), torch.zeros(3, dtype=torch.int32), none, none.view(5, 0))
    with pytest.raises(ValueError):
        e.forward_combined(torch.empty((0, 64), dtype=torch.bfloat16), plan)
    assert not launches


def test_sizes_that_32_bits_cannot_hold(launches):
    """Sizes reach the library as 32-bit integers: larger ones are refused, not wrapped."""
    for T, E, k in ((2 ** 32 + 10, 8, 1), (2 ** 31, 8, 1), (2 ** 30, 8, 4), (4, 2 ** 32 + 8, 2), (4, 8, 2 ** 32 + 2)):
        with pytest.raises(ValueError):
            _ext._route_need(T, E, k)
    ids, w = torch.zeros((4, 2), dtype=torch.int32), torch.ones((4, 2))
    for experts in (2 ** 32 + 8, 1025, 0, -5):
        for rows in (4, 0):
            with pytest.raises(ValueError):
                gemlite_amd.plan_experts(ids[:rows], w[:rows], experts)
    lib = _ext.load_library()
    for R in (2 ** 31 - 1, 2 ** 31 - 256):   # row + tile height has to stay an int
        assert lib.gla_experts_workspace_bytes(ctypes.byref(_args(R=R))) == -1
    with pytest.raises(ValueError):
        meta = torch.empty((2 ** 32 + 8, 64), dtype=torch.bfloat16, device="meta")
        e = _raw_experts(torch.bfloat16)
        t = [v.to("meta") for v in e.get_tensor_args()]
        gemlite_amd.experts_functional(meta, None, t, e.get_meta_args(), torch.empty(3, dtype=torch.int32, device="meta"))
    assert not launches


def test_import_without_custom_ops():
    """A torch without torch.library.custom_op, or a name that is taken, costs the compiled nodes and not the package."""
    code = ("import torch; del torch.library.custom_op; import gemlite_amd; from gemlite_amd import experts; "
            "assert experts.experts_op is None and experts.route_experts_op is None; print('imported')")
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "imported" in run.stdout, run.stderr


def test_compiled_calls_without_custom_ops(launches, monkeypatch):
    e = _raw_experts(torch.bfloat16)
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    monkeypatch.setattr(experts_module, "experts_op", None)
    monkeypatch.setattr(experts_module, "route_experts_op", None)
    monkeypatch.setattr(_ext, "route_experts", lambda *args: None)
    assert gemlite_amd.route_experts(torch.zeros((4, 2)), 1).places.shape == (4, 1)
    assert e(torch.zeros((4, 64), dtype=torch.bfloat16), torch.tensor([0, 2, 4], dtype=torch.int32)).shape == (4, 32) and len(launches) == 1


def test_compiled_calls_hand_on_the_tile_configuration(launches, monkeypatch):
    e = _raw_experts(torch.bfloat16)
    x, off = torch.zeros((4, 64), dtype=torch.bfloat16), torch.tensor([0, 2, 4], dtype=torch.int32)
    eager = gemlite_amd.experts_functional(x, None, e.get_tensor_args(), e.get_meta_args(), off, tile_config=2064)
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    compiled = gemlite_amd.experts_functional(x, None, e.get_tensor_args(), e.get_meta_args(), off, tile_config=2064)
    assert compiled.shape == eager.shape and [args.tile_config for args, _ in launches] == [2064, 2064]
    with pytest.raises(ValueError):
        gemlite_amd.experts_functional(x, None, e.get_tensor_args(), e.get_meta_args(), off, tile_config=7)
    e(x, off)
    assert launches[-1][0].tile_config == -1


def test_compiled_routing_copies_nothing(monkeypatch):
    """The op returns what the kernel writes, in five allocations of their own (outputs of an op must not share memory)."""
    written = []

    def record(logits, top_k, scoring, renormalize, scale, *outputs):
        written.extend(outputs)
        for t in outputs:
            t.zero_()

    monkeypatch.setattr(_ext, "_require_cuda", lambda *tensors: None)
    monkeypatch.setattr(_ext, "route_experts", record)
    plan = torch.ops.gemlite.route_experts(torch.zeros((5, 3)), 2, "softmax", True, 1.0)
    assert [t.data_ptr() for t in plan] == [t.data_ptr() for t in written]
    assert len({t.untyped_storage().data_ptr() for t in plan}) == 5
    assert [tuple(t.shape) for t in plan] == [(5, 2), (5, 2), (4,), (10,), (5, 2)]


def test_a_block_is_loaded_from_a_checkpoint(launches, monkeypatch):
    """A block of empty experts takes their shapes from the checkpoint, like the experts alone."""
    monkeypatch.setattr(_ext, "route_experts", lambda *args: None)
    block = GemLiteMoE(_raw_experts(torch.bfloat16, N=128), _raw_experts(torch.bfloat16), 2)
    model, empty = torch.nn.Sequential(block), torch.nn.Sequential(GemLiteMoE(GemLiteExperts(), GemLiteExperts(), 2))
    x, logits = torch.zeros((3, 64), dtype=torch.bfloat16), torch.zeros((3, 2))
    with pytest.raises(ValueError, match="belong together"):
        empty[0](x, logits)
    empty.load_state_dict(model.state_dict())
    assert empty[0].gate_up.num_experts == 2 and empty[0](x, logits).shape == (3, 32) and len(launches) == 2
    other = torch.nn.Sequential(GemLiteMoE(GemLiteExperts(), GemLiteExperts(), 2))
    other.load_state_dict(torch.nn.Sequential(torch.nn.ModuleDict({"gate_up": _raw_experts(torch.bfloat16), "down": _raw_experts(torch.bfloat16)})).state_dict())
    with pytest.raises(ValueError, match="belong together"):
        other[0](x, logits)


def test_one_workgroup_routes_few_tokens():
    """One workgroup's 16 waves take the tokens one after the other: above a few per wave the launch over many blocks, which
    keeps counts, is the faster one at every number of experts."""
    lib = _ext.load_library()
    for E, k in ((8, 2), (64, 1), (128, 8), (1024, 16)):
        assert lib.gla_route_workspace_bytes(40, E, k) == 0 and lib.gla_route_workspace_bytes(41, E, k) > 0
        assert lib.gla_route_workspace_bytes(128, E, k) > 0
    assert lib.gla_route_workspace_bytes(17, 1024, 64) > 0   # more (token, slot) pairs than threads
    # given ids are sorted by a thread each
    assert lib.gla_plan_workspace_bytes(128, 128, 8) == 0 and lib.gla_plan_workspace_bytes(129, 128, 8) > 0
    assert lib.gla_plan_workspace_bytes(4, 0, 1) == -1


def _fp8_args(K, R, N=4096, E=4):
    return _args(mode=0, R=R, T=0, top_k=0, E=E, N=N, K=K, W_nbits=8, group_size=K, elements_per_sample=1, input_dtype=DType.FP8.value, zeros=None,
                 meta_dtype=DType.FP32.value, channel_scale_mode=5, W_group_mode=0, w_stride_e=K * N, meta_stride_e=K // 128 * N // 128 * 4,
                 x_stride_m=K, out_stride_m=N)


def test_few_rows_of_fp8_experts_are_streamed():
    """The streaming kernel quantises in registers, the tiled one in a launch that writes to the workspace."""
    lib = _ext.load_library()

    def streamed(K, R):
        return lib.gla_experts_workspace_bytes(ctypes.byref(_fp8_args(K, R))) == 0

    assert [streamed(K, 8) for K in (2048, 2176, 2560, 3584, 4096)] == [False, True, True, True, True]
    assert [streamed(K, 12) for K in (2048, 2560, 3584, 4096)] == [False, False, False, True]
    assert streamed(4096, 32) and not streamed(4096, 36)
