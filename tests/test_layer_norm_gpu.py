"""Layer norm and its gradients against 64 bits, against differences, and against the separate steps."""
import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from w8a8_reference import U, assert_within, norm_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS = 1e-5


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    w8.read_status()


def inputs(m, k, dtype, residual=False, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, w, b = rand(m, k) + 0.3 * rand(m, 1), 1 + 0.3 * rand(k), 0.3 * rand(k)
    out = [t.to(dtype) for t in (x, w, b)]
    return (*out, rand(m, k).to(dtype) if residual else None)


def exact(h, w, b, dy=None, dh=None):
    """(y, its bound), and with dy ((dx, bound), (dw, bound), (db, bound)) of the rows h, in 64 bits."""
    v, m, k = h.double(), h.shape[0], h.shape[1]
    mean = v.mean(dim=1, keepdim=True)
    rstd = 1 / torch.sqrt((v - mean).square().mean(dim=1, keepdim=True) + EPS)
    xh = (v - mean) * rstd
    # mean and rstd are held in fp32, one rounding each; a difference, a product, an fma
    exh = rstd * mean.abs() * U + 4 * U * xh.abs()
    y = xh * w.double() + (b.double() if b is not None else 0)
    ey = exh * w.double().abs() + U * y.abs()
    if dy is None:
        return y, ey * 1.01
    d, wd = dy.double(), w.double().abs()
    g = d * w.double()
    c1, c2 = g.mean(dim=1, keepdim=True), (g * xh).mean(dim=1, keepdim=True)
    # sums over a row: at most 128 additions in a thread, then a tree of 10 (fp32)
    n = 140 * U
    ec1, ec2 = n * g.abs().mean(dim=1, keepdim=True), n * (g * xh).abs().mean(dim=1, keepdim=True) + (g.abs() * exh).mean(dim=1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    terms = g.abs() + c1.abs() + (xh * c2).abs()
    edx = rstd * (6 * U * terms + ec1 + xh.abs() * ec2 + exh * (c2.abs() + ec2))
    if dh is not None:
        dx = dx + dh.double()
        edx = edx + U * dx.abs()
    dw, db = (d * xh).sum(dim=0), d.sum(dim=0)
    rows = (m + 12) * U
    return (y, ey * 1.01), (dx, edx * 1.01), (dw, 1.01 * (rows * (d * xh).abs().sum(dim=0) + (d.abs() * exh).sum(dim=0))), \
        (db, 1.01 * rows * d.abs().sum(dim=0))


SIZES = [(1, 1), (1, 8), (2, 7), (5, 96), (3, 1000), (1, 2048), (70, 2048), (9, 1023), (33, 5120), (1300, 64), (4, 12000), (2, 16384), (3, 18945),
         (2, 40000), (601, 40), (1200, 8), (700, 1027), (333, 6001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", SIZES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_forward_and_gradients(m, k, with_residual, dtype):
    x, w, b, res = inputs(m, k, dtype, with_residual, seed=m + k)
    gen = torch.Generator(device="cuda").manual_seed(7)
    dy = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
    dh = torch.randn(m, k, generator=gen, device="cuda").to(dtype) if with_residual else None
    h = norm_of(x, res, w, b, EPS, "layer")[0]
    with torch.no_grad():
        out = w8.layer_norm(x, w, b, EPS, res)
    y = out[0] if with_residual else out
    (wy, ey), dx, dw, db = exact(h, w, b, dy, dh)
    assert_within(y, wy, ey, "y")
    if with_residual:
        assert torch.equal(out[1], h)
    leaves = [t.requires_grad_() for t in (x, w, b, *([res] if with_residual else []))]
    out2 = w8.layer_norm(x, w, b, EPS, res)
    assert torch.equal(out2[0] if with_residual else out2, y)
    grads = torch.autograd.grad(out2, leaves, (dy, dh) if with_residual else dy)
    for got, (want, bound), name in zip(grads, (dx, dw, db, dx), ("dx", "dw", "db", "dresidual")):
        assert got.dtype == dtype
        assert_within(got, want, bound, name)


def test_gradients_against_differences():
    m, k = 3, 24
    x, w, b, res = inputs(m, k, torch.float32, True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    a, c = (torch.randn(m, k, generator=gen, device="cuda") for _ in range(2))
    leaves = [t.requires_grad_() for t in (x, w, b, res)]
    y, h = w8.layer_norm(x, w, b, EPS, res)
    grads = torch.autograd.grad((y * a).sum() + (h * c).sum(), leaves)

    def value(*t):                            # the same function in 64 bits
        x, w, b, res = t
        h = x + res
        v = h - h.mean(dim=1, keepdim=True)
        y = v / torch.sqrt(v.square().mean(dim=1, keepdim=True) + EPS) * w + b
        return ((y * a.double()).sum() + (h * c.double()).sum()).item()

    base = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        for at in range(0, g.numel(), 5):
            step, vals = 1e-5, []
            for sign in (1, -1):
                t = [u.clone() for u in base]
                t[i].view(-1)[at] += sign * step
                vals.append(value(*t))
            # central differences: off by step^2 times a third derivative, which is some hundreds at most here
            assert abs((vals[0] - vals[1]) / (2 * step) - g.reshape(-1)[at].item()) < 1e-5 * (1 + g.abs().max().item())


def test_some_gradients_only():
    x, w, b, res = inputs(20, 256, torch.float32, True)
    dy = torch.randn_like(x)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(w8.layer_norm(*full, EPS), full, dy)
    for mask in range(1, 8):
        t = [u.clone().requires_grad_(bool(mask >> i & 1)) for i, u in enumerate((x, w, b))]
        w8.layer_norm(*t, EPS).backward(dy)
        for i in range(3):
            assert (t[i].grad is not None) == bool(mask >> i & 1)
            if t[i].grad is not None:
                assert torch.equal(t[i].grad, want[i])
    # only one of the outputs is used
    t = [u.clone().requires_grad_() for u in (x, w, b, res)]
    y, h = w8.layer_norm(t[0], t[1], t[2], EPS, t[3])
    g = torch.autograd.grad(h, t, dy, retain_graph=True)
    assert torch.equal(g[0], dy) and torch.equal(g[3], dy) and not g[1].any() and not g[2].any()
    g = torch.autograd.grad(y, t, dy, retain_graph=True)
    (y * dy).sum().backward()
    assert t[0].grad.data_ptr() != t[3].grad.data_ptr() and torch.equal(t[0].grad, t[3].grad)
    assert_within(g[0], *exact((x.double() + res.double()).float(), w, b, dy)[1])
    # without a bias
    t = [u.clone().requires_grad_() for u in (x, w)]
    torch.autograd.grad(w8.layer_norm(*t, eps=EPS), t, dy)


def test_shapes_strides_and_gradients_that_are_broadcast():
    x, w, b, _ = inputs(24, 130, torch.float16)
    want = w8.layer_norm(x, w, b, EPS)
    for v in (x.reshape(2, 3, 4, 130), x.t().contiguous().t()):
        assert torch.equal(w8.layer_norm(v, w, b, EPS).reshape(24, 130), want)
    wide = torch.full((24, 140), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 3:133] = x
    assert torch.equal(w8.layer_norm(wide[:, 3:133], w, b, EPS), want)
    assert w8.layer_norm(x[:0], w, b, EPS).shape == (0, 130)
    v = wide[:, 3:133].detach().requires_grad_()
    w2, b2 = w.clone().requires_grad_(), b.clone().requires_grad_()
    w8.layer_norm(v, w2, b2, EPS).float().sum().backward()            # a gradient of stride zero
    (_, _), dx, dw, db = exact(x, w, b, torch.ones_like(x))
    assert_within(v.grad, *dx)
    assert_within(w2.grad, *dw)
    assert_within(b2.grad, *db)
    e = x[:0].clone().requires_grad_()
    g = torch.autograd.grad(w8.layer_norm(e, w2, b2, EPS), (e, w2, b2), x[:0])
    assert g[0].shape == (0, 130) and not g[1].any() and not g[2].any()


def test_module_and_captured_training_step():
    torch.manual_seed(0)
    ref = torch.nn.LayerNorm(192, eps=1e-5).cuda()
    mod = w8.CudaLayerNorm.from_float(ref)
    assert mod.weight is ref.weight and isinstance(mod, torch.nn.LayerNorm) and mod.eps == ref.eps
    x = torch.randn(40, 192, device="cuda")
    (want, bound) = exact(x, ref.weight.detach(), ref.bias.detach())
    assert_within(mod(x).detach(), want, bound)
    # a training step of a module of its own, captured and replayed with other inputs
    mod = w8.CudaLayerNorm(192).cuda()
    static, dy = x.clone(), torch.randn_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.autograd.grad(mod(static), (mod.weight, mod.bias), dy)
        del g
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mod(static)
        g = torch.autograd.grad(y, (mod.weight, mod.bias), dy)
    for seed in (3, 4):
        z = inputs(40, 192, torch.float32, seed=seed)[0]
        static.copy_(z)
        graph.replay()
        (wy, ey), _, dw, db = exact(z, mod.weight.detach(), mod.bias.detach(), dy)
        assert_within(y.detach(), wy, ey)
        assert_within(g[0], *dw)
        assert_within(g[1], *db)


def test_same_bits_every_time():
    for m, k in ((3000, 512), (50, 18945)):
        x, w, b, _ = inputs(m, k, torch.float16)
        dy = torch.randn_like(x)
        t = [u.requires_grad_() for u in (x, w, b)]
        first = torch.autograd.grad(w8.layer_norm(*t, EPS), t, dy)
        for _ in range(4):
            for a, c in zip(first, torch.autograd.grad(w8.layer_norm(*t, EPS), t, dy)):
                assert torch.equal(a, c)
