"""The 8-bit path as it is used: models converted, patched with corrections, a decoder block's half run through it."""
import copy
import warnings

import pytest
import torch
import torch.nn as nn

from glowq_b200 import (AddSVDCorrection, CudaLayerNorm, CudaW4A16Linear, CudaW8A8Linear, TokenCodes, convert_to_cuda_w4a16,
                        convert_to_cuda_w8a8, norm_quantize_tokens, patch_svd_correction_wrappers_cumulative, quantize_tokens, right_factor)
from glowq_b200.cuda_w8a8 import read_status
from toy_model import ToyDecoder, make_artifacts
from w8a8_reference import U, assert_within, codes_of, norm_of, product_of


def patched(device, alpha=0.8, rank=16):
    model = ToyDecoder(seed=1)
    shared, bmap = make_artifacts(model, rank=rank)
    model = convert_to_cuda_w8a8(model.half().to(device))
    groups = {k.rsplit(".", 1)[0] for k in bmap.values()}
    return patch_svd_correction_wrappers_cumulative(model, shared, bmap, groups, alpha_svd=alpha)


def wrappers(model):
    return [m for m in model.modules() if isinstance(m, AddSVDCorrection)]


def test_patching_a_converted_model():
    model = patched("cpu")
    ws = wrappers(model)
    assert ws and all(isinstance(w.inner, CudaW8A8Linear) and w.group_launcher is None for w in ws)
    with pytest.raises(RuntimeError, match="CUDA"):
        ws[0](torch.randn(2, ws[0].inner.in_features))
    mixed = ToyDecoder(seed=1)
    mixed = convert_to_cuda_w4a16(mixed, 128)
    shared, bmap = make_artifacts(mixed, rank=8)
    lin = mixed.proj(0, ToyDecoder.PROJ[0])
    with pytest.raises(TypeError):
        AddSVDCorrection(lin, torch.zeros(lin.out_features, 8), torch.zeros(8, lin.in_features), "solo", False, None).tokens(torch.zeros(1, 4))
    with pytest.raises(TypeError):
        AddSVDCorrection(nn.Linear(4, 4), torch.zeros(4, 2), torch.zeros(2, 4), "solo", False, None)
    copy.deepcopy(model)


def linear_reference(w, x):
    """(y in 64 bits, bound) of a corrected module's fp16 call on x."""
    inner = w.inner if isinstance(w, AddSVDCorrection) else w
    codes, scales = codes_of(x)
    if inner is w:
        return product_of(codes, scales, inner.weight_codes, inner.scales_f32, inner.bias)
    exact = x.double() @ w.B_q.double().t()
    off = (2 * x.shape[1] + 4) * U * (x.double().abs() @ w.B_q.double().abs().t())
    off = off + 2.0 ** -11 * (exact.abs() + off) + 2.0 ** -25                    # r is held in fp16
    y, bound = product_of(codes, scales, inner.weight_codes, inner.scales_f32, inner.bias, w.alpha_svd, exact, w.A_q)
    return y, bound + abs(w.alpha_svd) * (off @ w.A_q.double().abs().t())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 20, 300])
def test_patched_modules(m):
    model = patched("cuda")
    gen = torch.Generator(device="cuda").manual_seed(m)
    for w in wrappers(model):
        x = torch.randn(m, w.inner.in_features, generator=gen, device="cuda").half()
        y = w(x)
        assert y.dtype == torch.float16
        assert_within(y, *linear_reference(w, x))
        t = w.tokens(x)
        assert isinstance(t, TokenCodes) and t.r.shape == (m, w.A_q.shape[1])
        assert_within(w(t), *linear_reference(w, x))
        w.alpha_svd = 0.0
        assert torch.equal(w(x), w.inner(x)) and torch.equal(w(t), w.inner(x))
    read_status()


@pytest.mark.gpu
def test_a_wrapper_whose_factors_do_not_fit():
    inner = CudaW8A8Linear.from_float(nn.Linear(64, 32).half().cuda())
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        w = AddSVDCorrection(inner, torch.zeros(32, 4).cuda(), torch.zeros(5, 64).cuda(), "solo", False, None)
    x = torch.randn(3, 64, device="cuda").half()
    assert torch.equal(w(x), inner(x)) and w.tokens(x).r is None and torch.equal(w(w.tokens(x)), inner(x))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 260])
@pytest.mark.parametrize("kind,dtype", [("layer", torch.float16), ("rms", torch.float16), ("rms", torch.bfloat16), ("layer", torch.float32)])
def test_half_a_block(m, kind, dtype):
    """residual -> norm -> codes -> three projections of one input -> quantised output projection, captured and replayed."""
    torch.manual_seed(0)
    h = 320
    norm_w, norm_b = (1 + 0.1 * torch.randn(h, device="cuda")).to(dtype), (0.1 * torch.randn(h, device="cuda")).to(dtype)
    b = norm_b if kind == "layer" else None
    qkv = [CudaW8A8Linear.from_float(nn.Linear(h, n, bias=kind == "layer").cuda().to(dtype), out_dtype=dtype) for n in (h, 128, 128)]
    o = CudaW8A8Linear.from_float(nn.Linear(h, h, bias=False).cuda().to(dtype))

    def block(x, res):
        t, hidden = norm_quantize_tokens(x, norm_w, b, residual=res, norm=kind)
        outs = [p(t) for p in qkv]
        return (*outs, o(outs[0]), hidden)

    x, res = torch.randn(m, h, device="cuda").to(dtype), torch.randn(m, h, device="cuda").to(dtype)
    got = block(x, res)
    hidden, y, _, _ = norm_of(x, res, norm_w, b, 1e-5, kind)
    assert torch.equal(got[4], hidden)
    for p, out in zip(qkv, got):
        assert out.dtype == dtype
        assert_within(out, *product_of(*codes_of(y), p.weight_codes, p.scales_f32, p.bias))
    assert_within(got[3], *product_of(*codes_of(got[0]), o.weight_codes, o.scales_f32, None))
    static = [x.clone(), res.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block(*static)
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for s in static:
            s.copy_(torch.randn(s.shape, generator=gen, device="cuda"))
        graph.replay()
        for a, c in zip(captured, block(*static)):
            assert torch.equal(a, c)
    read_status()


@pytest.mark.gpu
def test_beside_the_four_bit_modules():
    """4-bit and 8-bit launches one behind the other on a stream keep out of each other's way."""
    torch.manual_seed(0)
    lins = [nn.Linear(1024, 1024, bias=False).half().cuda() for _ in range(2)]
    four, eight = CudaW4A16Linear.from_float(lins[0], 128), CudaW8A8Linear.from_float(lins[1])
    for m in (1, 12, 40, 100, 300):
        x = torch.randn(m, 1024, device="cuda").half()
        want4 = four(x)
        torch.cuda.synchronize()
        want8 = eight(x)
        torch.cuda.synchronize()
        for _ in range(20):
            a, b = four(x), eight(x)
            c, d = eight(x), four(x)
        assert torch.equal(a, want4) and torch.equal(d, want4) and torch.equal(b, want8) and torch.equal(c, want8)


@pytest.mark.gpu
def test_converted_model_with_layer_norms():
    torch.manual_seed(0)
    model = nn.Sequential(nn.LayerNorm(96), nn.Linear(96, 64), nn.LayerNorm(64), nn.Linear(64, 48, bias=False)).cuda().half()
    x = torch.randn(10, 96, device="cuda").half()
    want = model(x)
    new = convert_to_cuda_w8a8(copy.deepcopy(model), layer_norms=True)
    assert isinstance(new[0], CudaLayerNorm) and isinstance(new[1], CudaW8A8Linear) and not new._w8a8_conversion_errors
    got = new(x)
    assert got.shape == want.shape and got.dtype == want.dtype
    step = x
    for mod in new:
        out = mod(step)
        if isinstance(mod, CudaLayerNorm):
            assert torch.equal(out, norm_of(step, None, mod.weight, mod.bias, mod.eps, "layer")[1])
        else:
            assert_within(out, *product_of(*codes_of(step), mod.weight_codes, mod.scales_f32, mod.bias))
        step = out
    assert torch.equal(step, got)
    r = right_factor(x, torch.randn(8, 96, device="cuda").half())
    assert quantize_tokens(x)._replace(r=r).r is r
