"""The 8-bit path's definitions in 64 bits, and the bounds of what fp32 arithmetic may differ from them."""
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}   # half the smallest subnormal
U = 2.0 ** -24


def codes_of(x):
    """(codes, fp32 scales) of the rows of x."""
    v = x.double()
    top = v.abs().amax(dim=1) if x.shape[1] else v.new_zeros(x.shape[0])
    scales = (top / 127.0).float()
    bad = ~torch.isfinite(v).all(dim=1)
    scales[bad] = float("nan")
    s = scales.double()[:, None]
    q = torch.where(s > 0, torch.round(v / s), torch.zeros_like(v))
    return q.clamp(-127, 127).to(torch.int8), scales


def norm_of(x, residual, w, b, eps, kind):
    """(h, rows of x's type, mean, rstd): the arithmetic that the entry points promise, every rounding in its place."""
    t = x.dtype
    h = x if residual is None else (x.double() + residual.double()).float().to(t)
    v = h.double()
    if kind == "rms":
        rstd = (1.0 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps)).float()
        n = (v * rstd.double()).float().to(t)
        return h, (n.double() * w.double()).float().to(t), None, rstd
    mean = v.mean(dim=1, keepdim=True)
    rstd = (1.0 / torch.sqrt((v - mean).square().mean(dim=1, keepdim=True) + eps)).float()
    mean = mean.float()
    n = ((v - mean.double()).float().double() * rstd.double()).float()
    y = n.double() * w.double()
    return h, (y + b.double() if b is not None else y).float().to(t), mean, rstd


def product_of(codes, scales, weight, weight_scales, bias, alpha=0.0, r=None, L=None):
    """(y in 64 bits, bound of the fp32 arithmetic before the last rounding)"""
    p = (codes.double() @ weight.double().t()) * scales.double()[:, None] * weight_scales.double()
    y, bound = p.clone(), 4 * U * p.abs()        # the integer's conversion, two factors, one sum
    if r is not None:
        y += alpha * (r.double() @ L.double().t())
        mag = abs(alpha) * (r.double().abs() @ L.double().abs().t())
        bound += (2 * r.shape[1] + 4) * U * mag  # sums of rank products whose adder may truncate: two half steps each
        # the products may be added to the scaled sum itself, held as sum / alpha (three more roundings: 1 / alpha, the quotient, the
        # product with alpha), by four MMAs for every 64 ranks, each of which may truncate the sum
        rest = p.abs() + (bias.double().abs() if bias is not None else 0)
        bound += (3 + 8 * ((r.shape[1] + 63) // 64)) * U * rest
    if bias is not None:
        y += bias.double()
        bound += 2 * U * bias.double().abs()
    return y, bound + 2 * U * y.abs()


def assert_within(got, want, bound, what=""):
    """got (of its own type) is want up to `bound` and one rounding to that type."""
    t = got.dtype
    g, w = got.double(), want.double()
    nan = torch.isnan(w)
    assert torch.equal(torch.isnan(g), nan), f"{what}: NaN in other places"
    limit = bound + HALF_STEP[t] * (w.abs() + bound) + SMALLEST[t]
    over = ((g - w).abs() - limit)[~nan]
    assert not over.numel() or over.max().item() <= 0.0, f"{what}: {over.max().item():.3e} over the bound"
