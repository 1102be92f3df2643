"""Conversion under ``torch.inference_mode``: the same module as outside of it."""
import copy

import pytest
import torch
import torch.nn as nn

from glowq_b200 import CudaW8A8Linear, convert_to_cuda_w8a8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_conversion(device):
    for k in (40, 64):
        lin = nn.Linear(k, 24).to(device)
        want = CudaW8A8Linear.from_float(lin)
        with torch.inference_mode():
            model = convert_to_cuda_w8a8(nn.Sequential(copy.deepcopy(lin)))
            for mod in (model[0], copy.deepcopy(model)[0], nn.Sequential(model[0]).half()[0]):
                assert mod.qweight_i8.shape == (24, (k + 15) // 16 * 16) and mod.qweight_i8.is_contiguous()
                assert torch.equal(mod.qweight_i8, want.qweight_i8) and torch.equal(mod.scales_f32, want.scales_f32)
        fresh = CudaW8A8Linear(k, 24, bias=True)
        fresh.load_state_dict(model[0].state_dict())
        assert torch.equal(fresh.qweight_i8.to(device), want.qweight_i8)
