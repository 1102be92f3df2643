"""Which factors belong to an 8-bit linear: those of its own error. The patchers say so where others are given."""
import warnings

import pytest
import torch
import torch.nn as nn

from glowq_b200 import AddSVDCorrection, CudaW8A8Linear, convert_to_cuda_w8a8, patch_svd_correction_wrappers, patch_svd_correction_wrappers_cumulative
from glowq_b200.cuda_w4a16.linear import _quantize_per_group_w4, _unpack_int4_i32


def weight(n=384, k=512):
    gen = torch.Generator().manual_seed(0)
    w = 0.02 * torch.randn(n, k, generator=gen)
    w[:, ::97] *= 5
    return w.half()


def four_bits(w, group=128):
    """The weight that the 4-bit path's codes stand for."""
    q, z, s, _ = _quantize_per_group_w4(w, group)
    n, k = w.shape
    codes, zeros = _unpack_int4_i32(q, k).float(), _unpack_int4_i32(z, s.shape[1]).float()
    groups = torch.arange(k) // group
    return (codes - zeros[:, groups]) * s.float()[:, groups]


def low_rank(e, rank):
    u, s, v = torch.linalg.svd(e, full_matrices=False)
    return u[:, :rank] * s[:rank], v[:rank]


def model_and_artefact(error, rank):
    w = weight()
    lin = nn.Linear(w.shape[1], w.shape[0], bias=False).half()
    lin.weight.data.copy_(w)
    model = convert_to_cuda_w8a8(nn.Sequential(lin))
    A, B = low_rank(error(w, model[0]), rank)
    return w, model, {"0.A": A, "0.B": B}, {"0.weight": "0.B"}


def of_eight(w, module):
    return w.float() - module.dequantized_weight()


def of_four(w, module):
    return w.float() - four_bits(w)


def test_dequantized_weight():
    w = weight()
    lin = nn.Linear(w.shape[1], w.shape[0]).half()
    lin.weight.data.copy_(w)
    mod = CudaW8A8Linear.from_float(lin)
    assert mod.dequantized_weight().shape == w.shape and mod.dequantized_weight(torch.bfloat16).dtype == torch.bfloat16
    assert ((mod.dequantized_weight() - w.float()).abs() <= 0.5001 * mod.scales_f32[:, None]).all()
    assert (four_bits(w) - w.float()).abs().max() < 0.1


@pytest.mark.parametrize("rank", [16, 64])
@pytest.mark.parametrize("cumulative", [False, True])
def test_the_patchers_warn_of_factors_of_another_error(rank, cumulative):
    def patch(model, shared, bmap, **kw):
        if cumulative:
            return patch_svd_correction_wrappers_cumulative(model, shared, bmap, {"0"}, **kw)
        return patch_svd_correction_wrappers(model, shared, bmap, **kw)
    w, model, shared, bmap = model_and_artefact(of_four, rank)
    with pytest.warns(UserWarning, match="8-bit modules"):
        patch(model, shared, bmap)
    assert isinstance(model[0], AddSVDCorrection)
    for kw in (dict(), dict(alpha_svd=0.9)):
        w, model, shared, bmap = model_and_artefact(of_eight, rank)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            patch(model, shared, bmap, **kw)
        assert isinstance(model[0], AddSVDCorrection)


def test_what_factors_do_to_the_error():
    """(the weights that the modules stand for, on the host)"""
    x = torch.randn(64, 512, generator=torch.Generator().manual_seed(1))
    errors = {}
    for name, error in (("own", of_eight), ("four", of_four)):
        w, model, shared, _ = model_and_artefact(error, 64)
        left = of_eight(w, model[0])
        errors["none"] = (x @ left.t()).norm()
        errors[name] = (x @ (left - shared["0.A"] @ shared["0.B"]).t()).norm()
    assert errors["own"] < errors["none"] < errors["four"]


@pytest.mark.gpu
def test_a_corrected_linear_comes_nearer():
    w, model, shared, bmap = model_and_artefact(of_eight, 64)
    x = torch.randn(40, 512, generator=torch.Generator().manual_seed(2))
    want = x.double() @ w.double().t()
    model = model.cuda()
    t = model[0].tokens(x.half().cuda())
    codes = (t.codes.double() * t.scales.double()[:, None]).cpu()
    plain = model[0](x.cuda()).double().cpu()
    patch_svd_correction_wrappers(model, shared, bmap)
    y = model[0](x.cuda()).double().cpu()
    # the weights' part of the error; that of the tokens' codes is there in both
    rest = (codes - x.double()) @ model[0].inner.dequantized_weight().cpu().double().t()
    assert (y - want - rest).norm() < 0.97 * (plain - want - rest).norm()
