"""Derivatives that the layer norm and the norm in front of codes have, and those that they refuse."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from glowq_b200 import CudaLayerNorm, layer_norm, norm_quantize_tokens

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused():
    """(a plain result would be a tangent of zero without a word)"""
    x, t, w = torch.randn(4, 64, device="cuda"), torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    norm = CudaLayerNorm(64, device="cuda")
    for frozen in (True, False):
        norm.requires_grad_(not frozen)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), fw.dual_level():
                d = fw.make_dual(x, t)
                for call in (lambda: norm(d), lambda: layer_norm(d, w), lambda: layer_norm(x, fw.make_dual(w, w)),
                             lambda: layer_norm(x, w, None, 1e-5, d), lambda: layer_norm(x, w, fw.make_dual(w, w))):
                    with pytest.raises(NotImplementedError):
                        call()
                assert torch.equal(norm(x), torch.no_grad()(norm)(x))        # without a tangent all is as ever
                y, h = norm(x, t)
                assert torch.equal(h, x + t)
    assert torch.isfinite(norm(x)).all()


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 37), (48,)])
def test_the_sum_in_front_of_codes_has_gradients(shape, norm):
    a, b, d = (torch.randn(shape, device="cuda") for _ in range(3))
    w = torch.ones(shape[-1], device="cuda", requires_grad=True)
    with torch.no_grad():
        codes, h0 = norm_quantize_tokens(a, w, residual=b, norm=norm)
    assert not h0.requires_grad and h0.shape == shape
    for ga, gb in ((True, True), (True, False), (False, True), (False, False)):
        x, res = a.clone().requires_grad_(ga), b.clone().requires_grad_(gb)
        t, h = norm_quantize_tokens(x, w, residual=res, norm=norm)
        assert torch.equal(h, a + b) and torch.equal(t.codes, codes.codes) and torch.equal(t.scales, codes.scales)
        assert h.shape == shape and h.requires_grad == (ga or gb) and not t.codes.requires_grad and not t.scales.requires_grad
        assert t.codes.shape == codes.codes.shape and t.codes.stride() == codes.codes.stride()
        if ga or gb:
            (h * 2).backward(d)
        for leaf, g in ((x, ga), (res, gb)):
            assert (leaf.grad is not None) == g
            if g:
                assert torch.equal(leaf.grad, 2 * d)
    x = a.clone().requires_grad_()
    t, h = norm_quantize_tokens(x, w, residual=x, norm=norm)      # the same tensor twice
    h = h.mul_(3.0)                                               # (what is changed in place goes on as any tensor)
    h.backward(d)
    assert torch.equal(x.grad, 6 * d)
    t, h = norm_quantize_tokens(x, w, norm=norm)
    assert h is x
    with torch.no_grad(), fw.dual_level():
        with pytest.raises(NotImplementedError):
            norm_quantize_tokens(fw.make_dual(a, b), w, residual=b, norm=norm)
        assert torch.equal(norm_quantize_tokens(a, w, residual=b, norm=norm)[1], a + b)


@pytest.mark.parametrize("shape", [(48,), (6, 48), (2, 3, 48), (2, 1, 3, 37)])
def test_outputs_that_are_changed_in_place(shape):
    x, res, d, e = (torch.randn(shape, device="cuda") for _ in range(4))
    w, b = torch.randn(shape[-1], device="cuda", requires_grad=True), torch.randn(shape[-1], device="cuda", requires_grad=True)
    leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
    layer_norm(leaf, w, b).mul_(2.0).add_(1.0).backward(d)
    want = torch.autograd.grad(layer_norm(other, w, b) * 2.0, other, d)[0]
    assert torch.equal(leaf.grad, want)
    leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
    y, _ = layer_norm(leaf, w, b, 1e-5, res)
    y.mul_(2.0).backward(d)
    y, _ = layer_norm(other, w, b, 1e-5, res)
    (y * 2.0).backward(d)
    assert y.shape == shape and torch.equal(leaf.grad, other.grad)
    y, h = layer_norm(leaf, w, b, 1e-5, res)
    h.add_(1.0)                               # h is what the gradients are taken from
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.backward((y, h), (d, e))
