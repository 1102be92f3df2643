"""Host side of the 8-bit path on the CPU: codes of weights, modules, refusals, the C entry points' checks and layouts."""
import ctypes
import os
import re

import pytest
import torch
import torch.nn as nn

from glowq_b200 import cuda_w8a8 as w8
from glowq_b200.cuda_w4a16 import kernels as K4
from glowq_b200.cuda_w8a8 import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "glowq_w8a8.h")).read()


def test_codes_of_weights():
    gen = torch.Generator().manual_seed(0)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        w = torch.randn(6, 37, generator=gen).to(dtype)
        w[2] = 0
        w[4, 3] = float("inf")
        codes, scales = w8.quantize_channels(w)
        assert codes.shape == (6, 37) and codes.dtype == torch.int8 and codes.stride() == (48, 1)
        assert scales[2] == 0 and not codes[2].any() and torch.isnan(scales[4]) and not codes[4].any()
        for i in (0, 1, 3, 5):
            assert scales[i] == (w[i].double().abs().max() / 127).float()
            assert (codes[i].double() * scales[i].double() - w[i].double()).abs().max() <= scales[i].double() * 0.5 * (1 + 1e-6)
    with pytest.raises(RuntimeError):
        w8.quantize_channels(torch.randn(3))
    with pytest.raises(RuntimeError):
        w8.quantize_channels(torch.zeros(3, 4, dtype=torch.int32))


def test_module_and_conversion():
    lin = nn.Linear(40, 24).half()
    mod = w8.CudaW8A8Linear.from_float(lin)
    assert (mod.in_features, mod.out_features) == (40, 24) and mod.qweight_i8.shape == (24, 48)
    assert mod.bias.dtype == torch.float32 and torch.equal(mod.bias.data, lin.bias.data.float())
    assert torch.equal(mod.weight_codes, w8.quantize_channels(lin.weight)[0]) and not mod.qweight_i8[:, 40:].any()
    other = w8.CudaW8A8Linear(40, 24, bias=True)
    other.load_state_dict(mod.state_dict())
    assert torch.equal(other.qweight_i8, mod.qweight_i8) and torch.equal(other.scales_f32, mod.scales_f32)
    assert w8.CudaW8A8Linear.from_float(nn.Linear(32, 8, bias=False)).bias is None
    with pytest.raises(RuntimeError, match="CUDA"):
        mod(torch.randn(2, 40))

    class Model(nn.Module):
        def __init__(self):
            super().__init__()
            self.block = nn.ModuleList([nn.Linear(16, 16), nn.LayerNorm(16), nn.LayerNorm((4, 4)), nn.LayerNorm(16, elementwise_affine=False)])
            self.lm_head = nn.Linear(16, 8)

    model = w8.convert_to_cuda_w8a8(Model())
    assert isinstance(model.block[0], w8.CudaW8A8Linear) and type(model.block[1]) is nn.LayerNorm and type(model.lm_head) is nn.Linear
    assert model._w8a8_conversion_errors == {}
    model = Model()
    weight = model.block[1].weight
    w8.convert_to_cuda_w8a8(model, layer_norms=True)
    assert isinstance(model.block[1], w8.CudaLayerNorm) and model.block[1].weight is weight
    assert type(model.block[2]) is nn.LayerNorm and type(model.block[3]) is nn.LayerNorm
    assert set(model._w8a8_conversion_errors) == {"block.2", "block.3"}
    with pytest.raises(ValueError):
        w8.CudaLayerNorm((2, 3))


def test_modules_that_are_cast():
    """A model cast to another type: codes, scales and bias stay what they are."""
    mod = w8.CudaW8A8Linear.from_float(nn.Linear(24, 16))
    want = {k: v.clone() for k, v in mod.state_dict().items()}
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu")):
        model = cast(nn.Sequential(mod))
        for k, v in mod.state_dict().items():
            assert v.dtype == want[k].dtype and torch.equal(v, want[k])
        assert isinstance(model[0].bias, nn.Parameter)


def test_cpu_tensors_are_refused():
    x, w = torch.randn(2, 16), torch.ones(16)
    for call in (lambda: w8.quantize_tokens(x), lambda: w8.norm_quantize_tokens(x, w), lambda: w8.layer_norm(x, w),
                 lambda: w8.right_factor(x, torch.zeros(4, 16, dtype=torch.float16)),
                 lambda: w8.w8a8_linear(x, torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)),
                 lambda: w8.w8a8_linear(w8.TokenCodes(torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)),
                                        torch.zeros(4, 16, dtype=torch.int8), torch.ones(4))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError):
        w8.norm_quantize_tokens(x, w, norm="batch")
    with pytest.raises(ValueError):
        w8.norm_quantize_tokens(x, w, w, norm="rms")


@pytest.mark.parametrize("name,cls", [("glowq_w8a8_rows", K.Rows), ("glowq_layer_norm_grad", K.LayerNormGrad), ("glowq_w8a8_linear", K.Linear)])
def test_descriptors_match_the_header(name, cls):
    body = re.search(r"typedef struct %s \{(.*?)\} %s_t;" % (name, name), HEADER, re.S).group(1)
    fields = []
    for line in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        line = line.strip()
        if line:
            m = re.match(r"(?:const )?(\w+)(\s*\*)?\s+(.*)|(?:const )?(\w+)\* (.*)", line)
            kind = "ptr" if "*" in line else m.group(1)
            fields += [(n.strip().lstrip("*"), kind) for n in re.sub(r"^(const )?\w+\s*\**\s*", "", line).split(",")]
    types = {"ptr": ctypes.c_void_p, "int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "double": ctypes.c_double, "float": ctypes.c_float,
             "size_t": ctypes.c_size_t}
    assert fields and [(n, types[k]) for n, k in fields] == list(cls._fields_)


def test_exports():
    lib = K4.load_w4a16_extension().lib
    names = re.findall(r"^\w+ (glowq_\w+)\(", HEADER, re.M)
    assert sorted(names) == sorted(K.EXPORTS)
    for n in names:
        assert hasattr(lib, n)


A = 1 << 12     # an address that no call here gets to read


def rows_desc(**kw):
    d = dict(x=A, residual=0, weight=0, bias=0, hidden=0, y=0, codes=A, scales=A, mean=0, rstd=0, stream=0, eps=0.0, x_stride=64,
             residual_stride=64, hidden_stride=64, y_stride=64, code_stride=64, M=4, K=64, dtype=0, norm=0, constant=0, reserved=0)
    d.update(kw)
    return K.pack_rows.pack(*(d[n] for n, _ in K.Rows._fields_))


BAD, STRIDE, SPACE, DEVICE, CUDA, LARGE = 1, 3, 4, 5, 6, 9
NOT_HERE = (DEVICE, CUDA)      # past the checks: there is no device in this process


@pytest.mark.parametrize("change,status", [
    (dict(M=-1), BAD), (dict(K=0), BAD), (dict(reserved=1), BAD), (dict(dtype=3), BAD), (dict(norm=3), BAD), (dict(x=0), BAD),
    (dict(codes=0), BAD), (dict(scales=0), BAD), (dict(y=A), BAD), (dict(weight=A), BAD), (dict(residual=A), BAD), (dict(mean=A), BAD),
    (dict(norm=1), BAD), (dict(norm=2, weight=A, bias=A), BAD), (dict(norm=1, weight=A, eps=-1.0), BAD), (dict(norm=1, weight=A, eps=float("nan")), BAD),
    (dict(norm=1, weight=A, hidden=A), BAD), (dict(norm=1, weight=A, constant=1), BAD), (dict(x=A + 1), BAD), (dict(x_stride=63), STRIDE),
    (dict(code_stride=63), STRIDE), (dict(norm=1, weight=A, residual=A, residual_stride=1), STRIDE),
    (dict(norm=1, weight=A, residual=A, hidden=A, hidden_stride=1), STRIDE)])
def test_row_calls_are_refused(change, status):
    assert K.ext().quantize(rows_desc(**change)) == status


def test_layer_norm_calls_are_refused():
    ok = dict(codes=0, scales=0, y=A, norm=1, weight=A)
    for change, status in ((dict(norm=2), BAD), (dict(norm=0, weight=0), BAD), (dict(codes=A), BAD), (dict(scales=A), BAD), (dict(y=0), BAD),
                           (dict(y_stride=1), STRIDE)):
        assert K.ext().layer_norm_forward(rows_desc(**{**ok, **change})) == status
    g = dict(h=A, dy=A, dh=0, weight=A, mean=A, rstd=A, dx=A, dweight=A, dbias=A, workspace=A, workspace_bytes=1 << 30, stream=0, h_stride=64,
             dy_stride=64, dh_stride=64, dx_stride=64, M=4, K=64, dtype=0, reserved=0)
    for change, status in ((dict(h=0), BAD), (dict(M=0), BAD), (dict(K=-1), BAD), (dict(dweight=0), BAD), (dict(dx=0, dweight=0, dbias=0), BAD),
                           (dict(dx=0, dh=A), BAD), (dict(dtype=7), BAD), (dict(reserved=1), BAD), (dict(dy=A + 1), BAD), (dict(h_stride=3), STRIDE),
                           (dict(dx_stride=3), STRIDE), (dict(workspace=0), SPACE), (dict(workspace_bytes=100), SPACE)):
        d = {**g, **change}
        assert K.ext().layer_norm_backward(K.pack_grad.pack(*(d[n] for n, _ in K.LayerNormGrad._fields_))) == status
    assert K.ext().lib.glowq_layer_norm_workspace_bytes(0, 5) == 0


@pytest.mark.parametrize("change,status", [
    (dict(M=-1), BAD), (dict(K=0), BAD), (dict(OC=0), BAD), (dict(reserved=1), BAD), (dict(out_dtype=5), BAD), (dict(r_mode=3), BAD),
    (dict(K=131072, code_stride=131072, weight_stride=131072), LARGE), (dict(M=(1 << 22) + 1), LARGE), (dict(codes=0), BAD), (dict(codes=A + 8), BAD),
    (dict(weight=A + 1), BAD), (dict(scales=0), BAD), (dict(scales=A + 2), BAD), (dict(weight_scales=0), BAD), (dict(out=0), BAD), (dict(out=A + 1), BAD),
    (dict(bias=A + 2), BAD), (dict(code_stride=72), STRIDE), (dict(weight_stride=48), STRIDE), (dict(out_stride=31), STRIDE),
    (dict(x=A, x_dtype=4, x_stride=64), BAD), (dict(x=A, x_stride=3), STRIDE), (dict(r_mode=2), BAD), (dict(r_mode=2, rank=16), BAD),
    (dict(r_mode=2, rank=1025, L=A, r=A, L_stride=1032, r_stride=1032), LARGE), (dict(r_mode=2, rank=16, L=A, r=A, L_stride=12, r_stride=16), STRIDE),
    (dict(r_mode=2, rank=16, L=A, r=A + 2, L_stride=16, r_stride=16), BAD), (dict(r_mode=1, rank=16, L=A, r=A, L_stride=16, r_stride=16), BAD),
    (dict(r_mode=1, rank=16, L=A, r=A, R=A, r_x=A, L_stride=16, r_stride=16, R_stride=60, r_x_stride=64), STRIDE)])
def test_linear_calls_are_refused(change, status):
    d = dict(x=0, codes=A, scales=A, weight=A, weight_scales=A, bias=0, r_x=0, R=0, r=0, L=0, out=A, stream=0, x_stride=0, code_stride=64,
             weight_stride=64, r_x_stride=0, R_stride=0, r_stride=0, L_stride=0, out_stride=32, M=4, K=64, OC=32, rank=0, x_dtype=0, out_dtype=0,
             r_mode=0, alpha=1.0, reserved=0)
    d.update(change)
    assert K.ext().linear(K.pack_linear.pack(*(d[n] for n, _ in K.Linear._fields_))) == status


@pytest.mark.skipif(torch.cuda.is_available(), reason="the address is read where there is a device")
def test_without_a_device():
    assert K.ext().quantize(rows_desc()) in NOT_HERE
