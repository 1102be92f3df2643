"""Factors in wrappers around 8-bit linears: they stay fp16 in a model that is cast, and lie as the kernels read them."""
import copy

import pytest
import torch
import torch.nn as nn

from glowq_b200 import AddSVDCorrection, CudaW4A16Linear, CudaW8A8Linear
from glowq_b200.cuda_w8a8 import read_status
from w8a8_reference import assert_within
from test_w8a8_block import linear_reference


def wrapper(cls, k, n, rank, device="cpu"):
    torch.manual_seed(0)
    lin = nn.Linear(k, n).to(device).half()
    inner = CudaW8A8Linear.from_float(lin) if cls is CudaW8A8Linear else CudaW4A16Linear.from_float(lin, 32)
    return AddSVDCorrection(inner, 0.1 * torch.randn(n, rank).to(device), 0.1 * torch.randn(rank, k).to(device), "solo", False, None, 0.8)


CASTS = [lambda m: m.bfloat16(), lambda m: m.float(), lambda m: m.to("cpu", torch.float64), lambda m: m.half(), copy.deepcopy,
         lambda m: m.bfloat16().half().float()]


@pytest.mark.parametrize("cls,k,rank", [(CudaW8A8Linear, 64, 16), (CudaW8A8Linear, 36, 12), (CudaW8A8Linear, 64, 5), (CudaW4A16Linear, 64, 12)])
def test_casts_and_places(cls, k, rank):
    for cast in CASTS:
        w = wrapper(cls, k, 24, rank)
        want = {n: getattr(w, n).clone() for n in ("A_q", "B_q")}
        assert want["A_q"].shape == (24, rank) and want["B_q"].shape == (rank, k)
        w = cast(nn.Sequential(w))[0]
        for n, v in want.items():
            t = getattr(w, n)
            assert t.dtype == torch.float16 and torch.equal(t, v), n
            assert n in dict(w.named_buffers()) and n not in w.state_dict()
            if cls is CudaW8A8Linear:
                assert t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0
            else:
                assert t.is_contiguous()


def test_factors_that_are_parameters():
    for cls in (CudaW8A8Linear, CudaW4A16Linear):
        w = wrapper(cls, 64, 24, 12)
        want = w.A_q.clone()
        del w.A_q
        w.A_q = nn.Parameter(want.clone(), requires_grad=False)
        w = nn.Sequential(w).bfloat16()[0]
        assert isinstance(w.A_q, nn.Parameter) and w.A_q.dtype == torch.float16 and torch.equal(w.A_q, want)
        held = w.B_q
        assert nn.Sequential(w).half()[0].B_q is held


def test_factors_of_other_shapes():
    inner = CudaW8A8Linear.from_float(nn.Linear(64, 32))
    with pytest.warns(UserWarning):
        w = AddSVDCorrection(inner, torch.zeros(4), torch.zeros(5, 63), "solo", False, None)
    assert w.bfloat16().A_q.dtype == torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 20, 300])
def test_calls_of_a_model_that_was_cast(m, dtype):
    for k, rank in ((64, 12), (36, 16), (128, 64)):
        w = nn.Sequential(wrapper(CudaW8A8Linear, k, 24, rank)).to("cuda", dtype)[0]
        x = torch.randn(m, k, device="cuda").to(dtype)
        y = w(x)
        assert y.dtype == dtype
        assert_within(y, *linear_reference(w, x.half()) if dtype == torch.float16 else reference(w, x))
    read_status()


def reference(w, x):
    """As ``linear_reference``, of an x that r takes in fp16."""
    from w8a8_reference import U, codes_of, product_of
    half = x.half().double()
    exact = half @ w.B_q.double().t()
    off = (2 * x.shape[1] + 4) * U * (half.abs() @ w.B_q.double().abs().t())
    off = off + 2.0 ** -11 * (exact.abs() + off) + 2.0 ** -25
    y, bound = product_of(*codes_of(x), w.inner.weight_codes, w.inner.scales_f32, w.inner.bias, w.alpha_svd, exact, w.A_q)
    return y, bound + abs(w.alpha_svd) * (off @ w.A_q.double().abs().t())


@pytest.mark.gpu
def test_calls_copy_no_factor():
    from test_w8a8_order_gpu import early
    for rank in (12, 64):
        w = wrapper(CudaW8A8Linear, 64, 128, rank, "cuda")
        x = torch.randn(20, 64, device="cuda").half()
        assert early(lambda: w(x)) == [True, True]          # codes, r, product
