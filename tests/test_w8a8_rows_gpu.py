"""Token codes, alone and behind a norm, against their definition in 64 bits: the same codes and scales, bit for bit."""
import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from w8a8_reference import codes_of, norm_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def values(m, k, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=gen, device="cuda") * torch.exp(torch.randn(m, 1, generator=gen, device="cuda"))
    x[:, ::97] *= 20
    return x.to(dtype)


def assert_codes(t, x):
    codes, scales = codes_of(x)
    assert torch.equal(t.scales.view(torch.int32), scales.view(torch.int32)) or torch.equal(
        torch.nan_to_num(t.scales, nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
    assert t.codes.shape == x.shape and t.codes.dtype == torch.int8
    assert torch.equal(t.codes, codes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 7), (5, 128), (1, 1024), (9, 1032), (4, 2047), (2, 5120), (130, 520), (3, 18944),
                                 (2, 17001), (1, 32776), (2, 70000)])
def test_codes(m, k, dtype):
    x = values(m, k, dtype, seed=k)
    assert_codes(w8.quantize_tokens(x), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_special(dtype):
    x = values(12, 520, dtype)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 500] = float("nan")
    x[4] = float("-inf")
    x[5] = 0
    x[5, 519] = torch.finfo(dtype).smallest_normal
    x[6] = torch.finfo(dtype).max
    x[7] = 3.0
    x[8] = -0.0
    if dtype != torch.float16:          # scales that are subnormal numbers, or nothing at all
        x[9] *= 2.0 ** -133
        x[10] = 0
        x[10, 3] = 2.0 ** -133
    t = w8.quantize_tokens(x)
    assert_codes(t, x)
    assert torch.isnan(t.scales[2:5]).all() and not torch.isnan(t.scales[[0, 1, 5, 6, 7, 8, 9, 10, 11]]).any()


def test_borders():
    """Quotients that lie on a border between two codes, or next to one."""
    steps = torch.arange(-254, 255, device="cuda", dtype=torch.float32) * 0.5
    rows = []
    for top in (127.0, 254.0, 127.0 * 2 ** -9, 100.0, 63.5, 0.1):
        row = steps * (top / 127.0)
        row[0] = top
        rows += [row, row * (1 + 2.0 ** -23), row * (1 - 2.0 ** -23), row * (1 + 2.0 ** -22)]
    x = torch.stack(rows)
    for dtype in TYPES:
        y = x.to(dtype)
        assert_codes(w8.quantize_tokens(y), y)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dtype):
    big = values(6, 800, dtype)
    for x in (big[:, :640], big[:, 3:600], big[::2, :512], big[1:2], big[:, 8:520]):
        assert_codes(w8.quantize_tokens(x), x)
    t = w8.quantize_tokens(big.t())                       # unit stride the other way
    assert_codes(t, big.t().contiguous())
    t = w8.quantize_tokens(big.reshape(2, 3, 800))
    assert_codes(t, big)
    assert_codes(w8.quantize_tokens(big[0]), big[:1])
    row = big[:1].expand(4, 800)
    assert_codes(w8.quantize_tokens(row), row)
    t = w8.quantize_tokens(big[:0])
    assert t.codes.shape == (0, 800) and t.scales.shape == (0,)


def test_codes_behind_codes_stay_as_they_are():
    """Rows of 37 columns lie 48 bytes apart: what is between them is not written."""
    x = values(5, 37, torch.float16)
    room = torch.full((5, 48), 77, dtype=torch.int8, device="cuda")
    scales = torch.empty(7, device="cuda").fill_(9.0)
    from glowq_b200.cuda_w8a8 import functional as F
    F._quantize(x, room[:, :37], scales[:5], False)
    assert torch.equal(room[:, :37], codes_of(x)[0]) and (room[:, 37:] == 77).all() and (scales[5:] == 9).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("m,k", [(1, 1), (2, 7), (5, 96), (1, 2048), (3, 2049), (70, 1024), (2, 5120), (1, 20001), (2, 40000)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_codes_behind_a_norm(m, k, kind, with_residual, dtype):
    x, res = values(m, k, dtype, seed=1), values(m, k, dtype, seed=2) if with_residual else None
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = (1 + 0.3 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
    b = (0.3 * torch.randn(k, generator=gen, device="cuda")).to(dtype) if kind == "layer" else None
    t, hidden = w8.norm_quantize_tokens(x, w, b, eps=1e-5, residual=res, norm=kind)
    h, y, _, _ = norm_of(x, res, w, b, 1e-5, kind)
    assert torch.equal(hidden, h)
    assert_codes(t, y)
    if not with_residual:
        assert hidden is x


def test_norms_of_special_rows():
    """Constant rows, large means, an infinity, a NaN; a layer norm without a bias; strided rows."""
    for dtype in TYPES:
        x = values(8, 512, dtype)
        x[1] = 4.0
        x[2] = 0
        x[3] = (1000 + x[3].float()).to(dtype)
        x[4, 7] = float("inf")
        x[5, 9] = float("nan")
        w = torch.linspace(0.5, 1.5, 512, device="cuda").to(dtype)
        for kind in ("layer", "rms"):
            t, _ = w8.norm_quantize_tokens(x, w, eps=1e-5, norm=kind)
            _, y, _, _ = norm_of(x, None, w, None, 1e-5, kind)
            assert_codes(t, y)
            assert torch.isnan(t.scales[4:6]).all() and not torch.isnan(t.scales[[0, 1, 2, 3, 6, 7]]).any()
        wide = values(8, 700, dtype)
        t, h = w8.norm_quantize_tokens(wide[::2, 4:516], w, residual=wide[1::2, 5:517], norm="rms")
        hh, y, _, _ = norm_of(wide[::2, 4:516], wide[1::2, 5:517], w, None, 1e-5, "rms")
        assert torch.equal(h, hh)
        assert_codes(t, y)


def test_weights_take_the_same_codes_on_either_device():
    for k in (64, 37):
        w = values(9, k, torch.float16)
        w[3] = 0
        a, sa = w8.quantize_channels(w)
        b, sb = w8.quantize_channels(w.cpu())
        assert torch.equal(a.cpu(), b) and torch.equal(sa.cpu(), sb)
        assert a.stride(0) % 16 == 0 and torch.equal(a, codes_of(w)[0])


def test_many_rows_of_few_columns():
    x = values(200_003, 24, torch.float16)
    assert_codes(w8.quantize_tokens(x), x)
