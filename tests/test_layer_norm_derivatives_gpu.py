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
