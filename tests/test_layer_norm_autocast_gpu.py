"""``CudaLayerNorm`` in the place of ``nn.LayerNorm`` where parameters and rows are of different types."""
import pytest
import torch
import torch.nn as nn

from glowq_b200 import CudaLayerNorm
from test_layer_norm_gpu import EPS, exact
from w8a8_reference import U, assert_within

pytestmark = pytest.mark.gpu


def modules(k, dtype, bias=True):
    torch.manual_seed(0)
    ref = nn.LayerNorm(k, eps=EPS, bias=bias).cuda()
    with torch.no_grad():
        for p in ref.parameters():
            p.add_(0.3 * torch.randn(k, device="cuda"))
    return ref.to(dtype), CudaLayerNorm.from_float(ref)


@pytest.mark.parametrize("cast", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("x_dtype,w_dtype", [(torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.float16),
                                             (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("bias", [True, False])
def test_autocast(x_dtype, w_dtype, cast, bias):
    m, k = 20, 200
    ref, mod = modules(k, w_dtype, bias)
    x, dy = torch.randn(m, k, device="cuda").to(x_dtype), torch.randn(m, k, device="cuda")
    w, b = ref.weight.detach().float(), ref.bias.detach().float() if bias else None
    (y, ey), dx, dw, db = exact(x.float(), w, b, dy)
    leaf = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=cast):
        want, got = ref(x), mod(leaf)
        assert got.dtype == want.dtype == torch.float32 and got.shape == want.shape
        with torch.no_grad():
            assert torch.equal(mod(x), got)
        z, h = mod(x, x)
        assert h.dtype == x_dtype and torch.equal(h, x + x) and z.dtype == torch.float32
    assert_within(got.detach(), y, ey)
    leaves = [leaf, *mod.parameters()]
    for g, (value, bound), p in zip(torch.autograd.grad(got, leaves, dy), (dx, dw, db), leaves):
        assert g.dtype == p.dtype
        # (rounded to fp32 first where the leaf is narrower)
        assert_within(g, value, bound + U * value.abs())


def test_one_type_under_autocast_stays_it():
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        _, mod = modules(96, dtype)
        x = torch.randn(4, 96, device="cuda").to(dtype)
        want = mod(x)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(mod(x), want) and mod(x).dtype == dtype


def test_types_that_differ_are_refused_outside():
    ref, mod = modules(96, torch.float32)
    x = torch.randn(4, 96, device="cuda").half()
    for call in (ref, mod):
        with pytest.raises(RuntimeError):
            call(x)
