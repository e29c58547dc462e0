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
