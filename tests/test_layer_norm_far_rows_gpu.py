"""Layer norm's gradients on rows that lie far from zero against their deviation: the row's mean is taken off first, whatever its size."""
import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from w8a8_reference import U, assert_within, codes_of, norm_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS = 1e-5
# (of each plan: a group of warps, a CTA to a row, two pieces a thread, passes over the rows; odd widths)
WIDTHS = [64, 250, 1000, 2048, 2999, 5120, 9000, 12288, 40000]


def gradients(h, w, dy):
    """(dx, bound), (dw, bound), (db, bound) in 64 bits of rows whose mean is a number of 32 bits."""
    v, m = h.double(), h.shape[0]
    total = v.sum(dim=1, keepdim=True)                    # (exact: 24 bits and the count's)
    mean = total / torch.full_like(total, h.shape[1])     # (a scalar divisor would be taken as a product with its reciprocal)
    assert torch.equal(mean, mean.float().double())
    rstd = 1 / torch.sqrt((v - mean).square().mean(dim=1, keepdim=True) + EPS)
    xh = (v - mean) * rstd
    exh = 4 * U * xh.abs()                    # a difference, rstd, a product: the mean is exact
    d, g = dy.double(), dy.double() * w.double()
    c1, c2 = g.mean(dim=1, keepdim=True), (g * xh).mean(dim=1, keepdim=True)
    n = 140 * U                               # sums over a row: at most 128 additions in a thread, then a tree of 10
    ec1, ec2 = n * g.abs().mean(dim=1, keepdim=True), n * (g * xh).abs().mean(dim=1, keepdim=True) + (g.abs() * exh).mean(dim=1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    edx = rstd * (6 * U * (g.abs() + c1.abs() + (xh * c2).abs()) + ec1 + xh.abs() * ec2 + exh * (c2.abs() + ec2))
    rows = (m + 12) * U
    return ((dx, edx * 1.01), ((d * xh).sum(dim=0), 1.01 * (rows * (d * xh).abs().sum(dim=0) + (d.abs() * exh).sum(dim=0))),
            (d.sum(dim=0), 1.01 * rows * d.abs().sum(dim=0)))


def leaves(m, k, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return (1 + 0.3 * rand(k)).to(dtype).requires_grad_(), rand(k).to(dtype).requires_grad_(), rand(m, k).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_constant_rows(k, dtype):
    """What is normalised is zero: dweight gets nothing from such rows."""
    for value in (999.0, -0.7, 3.0e4):
        w, b, dy = leaves(9, k, dtype)
        x = torch.full((9, k), value, device="cuda").to(dtype).requires_grad_()
        gx, gw, gb = torch.autograd.grad(w8.layer_norm(x, w, b, EPS), (x, w, b), dy)
        assert not gw.any()
        dx, _, db = gradients(x.detach(), w.detach(), dy)
        assert_within(gx, *dx, "dx")
        assert_within(gb, *db, "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_rows_with_a_large_mean(k, dtype):
    """16384 +- a few steps of the type, in equal parts: the mean is exact, and some hundred deviations."""
    m, step = 21, {torch.float16: 16, torch.bfloat16: 128, torch.float32: 16}[dtype]
    w, b, dy = leaves(m, k, dtype, seed=k)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.full((m, k), 16384.0, device="cuda")
    for row in range(m):
        signs = 2 * (torch.randperm(k // 2 * 2, generator=gen, device="cuda") % 2) - 1
        x[row, k % 2:] += step * (3 + 2 * (row % 3)) * signs
    x = x.to(dtype)
    want = gradients(x, w.detach(), dy)
    x.requires_grad_()
    for got, (value, bound), name in zip(torch.autograd.grad(w8.layer_norm(x, w, b, EPS), (x, w, b), dy), want, ("dx", "dw", "db")):
        assert_within(got, value, bound, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [37, 96, 1001, 2999, 5121, 5128, 9001, 12290, 40001])
def test_rows_of_the_lowest_value(k, dtype):
    """Rows that a mask has filled with the type's lowest value (mean * rstd is above all numbers): what lies behind a row's end joins no sum."""
    lowest = torch.finfo(dtype).min
    w, b, dy = leaves(9, k, dtype, seed=k)
    x = torch.randn(9, k, device="cuda").to(dtype)
    x[::2] = lowest
    for res in (None, torch.zeros_like(x)):
        t, h = w8.norm_quantize_tokens(x, w.detach(), b.detach(), eps=EPS, residual=res, norm="layer")
        _, y, _, _ = norm_of(x, None, w.detach(), b.detach(), EPS, "layer")
        codes, scales = codes_of(y)
        assert torch.equal(h, x) and torch.equal(t.scales, scales) and torch.equal(t.codes, codes)
        assert torch.equal(y[0], b)
    leaf = x[::2].clone().requires_grad_()
    gx, gw, gb = torch.autograd.grad(w8.layer_norm(leaf, w, b, EPS), (leaf, w, b), dy[::2].contiguous())
    assert not gw.any() and torch.isfinite(gx).all()
    assert_within(gb, *gradients(leaf.detach(), w.detach(), dy[::2])[2], "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [37, 96, 1001, 2999, 5121, 5128, 9001, 12290, 40001])
def test_deviation_of_constant_rows(k, dtype):
    """It is nothing at any width, however large the value: dx is the projection of dy * weight, times 1 / sqrt(eps)."""
    w, b, dy = leaves(3, k, dtype, seed=k)
    for value in (torch.finfo(dtype).min, min(1e20, torch.finfo(dtype).max)):
        x = torch.full((3, k), value, dtype=dtype, device="cuda", requires_grad=True)
        gx, gw, gb = torch.autograd.grad(w8.layer_norm(x, w, b, EPS), (x, w, b), dy)
        dx, _, db = gradients(x.detach(), w.detach(), dy)
        assert_within(gx, *dx, "dx")
        assert_within(gb, *db, "db")
        assert not gw.any()


@pytest.mark.parametrize("ratio", [3, 20, 100, 900])
def test_statistics_are_rounded_once(ratio):
    """Rows whose mean is many deviations: rstd, and with it every scale and code, is that of 64-bit sums."""
    m, k = 200_000, 200
    gen = torch.Generator(device="cuda").manual_seed(ratio)
    x = torch.randn(m, k, generator=gen, device="cuda") + ratio * torch.randn(m, 1, generator=gen, device="cuda").sign()
    w, b = (1 + 0.3 * torch.randn(k, generator=gen, device="cuda")), 0.3 * torch.randn(k, generator=gen, device="cuda")
    t, _ = w8.norm_quantize_tokens(x, w, b, eps=EPS, norm="layer")
    _, y, mean, rstd = norm_of(x, None, w, b, EPS, "layer")
    out = w8.layer_norm(x.requires_grad_(), w, b, EPS)
    kept, root = out.grad_fn.saved_tensors[2:]
    assert torch.equal(kept, mean.flatten()) and torch.equal(root, rstd.flatten())
    codes, scales = codes_of(y)
    assert torch.equal(t.scales, scales) and torch.equal(t.codes, codes)


def test_rows_have_one_mean_wherever_they_lie():
    """fp32 rows of few columns, whose mean is often half way between two numbers of 32 bits: the kernels that take them round it alike."""
    for k in (96, 117, 150):
        m = 20_000
        gen = torch.Generator(device="cuda").manual_seed(k)
        x, res = (torch.randn(m, k, generator=gen, device="cuda") for _ in range(2))
        x += 5 * torch.randn(m, 1, generator=gen, device="cuda")
        w, b = torch.ones(k, device="cuda"), torch.zeros(k, device="cuda")
        room = torch.zeros(m, k + 3, device="cuda")
        room[:, 1:k + 1] = res
        far = room[:, 1:k + 1]                   # not where x lies within 16 bytes: passes over the rows
        kept = []
        for r in (res, far):
            out = w8.layer_norm(x.clone().requires_grad_(), w, b, EPS, r)
            kept.append([t.detach().clone() for t in (*out, *out[0].grad_fn.saved_tensors[2:])])
            t, h = w8.norm_quantize_tokens(x, w, b, eps=EPS, residual=r, norm="layer")
            kept[-1] += [t.codes, t.scales, h]
        for a, c in zip(*kept):
            assert torch.equal(a, c)
        _, _, mean, rstd = norm_of(x, res, w, b, EPS, "layer")
        assert torch.equal(kept[0][2], mean.flatten()) and torch.equal(kept[0][3], rstd.flatten())
