"""Types through a converted model: linears of shared codes return what linears of the activations return."""
import pytest
import torch
import torch.nn as nn

from glowq_b200 import AddSVDCorrection, TokenCodes, convert_to_cuda_w8a8, norm_quantize_tokens, quantize_tokens
from glowq_b200.cuda_w8a8 import read_status

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 6, 300])
def test_codes_and_activations_give_the_same(m, dtype):
    torch.manual_seed(0)
    model = convert_to_cuda_w8a8(nn.ModuleDict({n: nn.Linear(96, o) for n, o in (("q", 96), ("k", 40))}).cuda().to(dtype))
    wrapped = AddSVDCorrection(model["q"], 0.1 * torch.randn(96, 8).cuda(), 0.1 * torch.randn(8, 96).cuda(), "solo", False, None)
    x, res = (torch.randn(2, m, 96, device="cuda").to(dtype) for _ in range(2))
    w = torch.ones(96, device="cuda", dtype=dtype)
    for lin in model.values():
        y = lin(x)
        assert y.dtype == dtype and y.shape[:2] == (2, m)
        for t in (lin.tokens(x), quantize_tokens(x)):
            assert t.dtype == dtype
            z = lin(t)
            assert z.dtype == dtype and torch.equal(z, y.flatten(0, 1))
        for norm in ("rms", "layer"):
            t, h = norm_quantize_tokens(x, w, residual=res, norm=norm)
            assert t.dtype == dtype and lin(t).dtype == dtype and h.dtype == dtype
    y, t = wrapped(x), wrapped.tokens(x)
    assert y.dtype == dtype and wrapped(t).dtype == dtype
    assert t._replace(r=None).dtype == dtype
    # codes that say nothing of a type
    assert model["q"](TokenCodes(t.codes, t.scales)).dtype == torch.float16
    model["q"].out_dtype = torch.float32
    assert model["q"](t).dtype == torch.float32 and model["q"](x).dtype == torch.float32
    read_status()


def test_values_that_fp16_does_not_hold():
    for dtype in (torch.bfloat16, torch.float32):
        lin = convert_to_cuda_w8a8(nn.Sequential(nn.Linear(64, 32, bias=False).cuda().to(dtype)))[0]
        x = torch.full((2, 64), 3.0e6, device="cuda").to(dtype)
        y = lin(lin.tokens(x))
        assert torch.equal(y, lin(x)) and torch.isfinite(y).all() and (y.abs() > 65504).any()
