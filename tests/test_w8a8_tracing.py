"""Traces of torch's operations do not see the kernels: they are refused."""
import pytest
import torch
import torch.nn as nn
from torch.fx.experimental.proxy_tensor import make_fx

from glowq_b200 import CudaLayerNorm, CudaW8A8Linear, layer_norm, norm_quantize_tokens, quantize_channels, quantize_tokens, right_factor, w8a8_linear
from glowq_b200.cuda_w8a8 import kernels as K


def nothing(desc):
    raise AssertionError("launched")


def test_launches_are_refused_under_proxies():
    """(on the CPU: what all launches go through)"""
    seen = []

    def f(x):
        with pytest.raises(RuntimeError, match="traced"):
            K.call(nothing, torch.device("cuda", 0), b"", "glowq_w8a8_quantize")
        seen.append(1)
        return x + 1

    make_fx(f)(torch.zeros(2))
    assert len(seen) == 1


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_every_entry_point():
    x, res = torch.randn(4, 64, device="cuda").half(), torch.randn(4, 64, device="cuda").half()
    w = torch.ones(64, device="cuda").half()
    q, qs = quantize_channels(torch.randn(32, 64, device="cuda"))
    L, R = torch.randn(32, 8, device="cuda").half(), torch.randn(8, 64, device="cuda").half()
    t = quantize_tokens(x)
    lin, norm = CudaW8A8Linear.from_float(nn.Linear(64, 32).cuda().half()), CudaLayerNorm(64, device="cuda", dtype=torch.float16)
    calls = [lambda v: quantize_tokens(v)[:2], lambda v: norm_quantize_tokens(v, w, residual=res.reshape(v.shape))[1], lambda v: quantize_channels(v.flatten(0, -2))[0],
             lambda v: right_factor(v, R), lambda v: w8a8_linear(v, q, qs), lambda v: w8a8_linear(v, q, qs, L=L, R=R),
             lambda v: w8a8_linear(t, q, qs) + v.flatten(0, -2)[:, :32], lambda v: layer_norm(v, w),
             lambda v: layer_norm(v, w, None, 1e-5, res.reshape(v.shape))[0], lin, norm]
    for call in calls:
        call(x)
        for v in (x, x.t().contiguous().t(), x[None], x.expand(4, 64)):
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(call, v, check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(lambda v: call(v))(x)
        call(x)
