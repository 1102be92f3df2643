"""Layer norm's gradients where the matrices of a call begin at different places within 16 bytes: pieces of a row are shifted between lanes."""
import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from test_layer_norm_gpu import EPS, TYPES, exact, inputs
from w8a8_reference import assert_within

pytestmark = pytest.mark.gpu
# (a warp, several warps, a CTA, two pieces a thread; whole pieces and others)
WIDTHS = [13, 300, 512, 1027, 2048, 5001, 12000, 16383]


def placed(t, offset, pitch):
    """`t` with its rows `pitch` elements apart from `offset` on, NaN around them."""
    room = torch.full((t.shape[0], pitch), float("nan"), dtype=t.dtype, device=t.device)
    room[:, offset:offset + t.shape[1]] = t
    return room[:, offset:offset + t.shape[1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("offset,more", [(1, 9), (2, 8), (3, 11), (4, 16), (5, 10), (6, 7), (7, 13), (0, 5)])
def test_gradients(k, offset, more, dtype):
    m = 37
    x, w, b, _ = inputs(m, k, dtype, seed=k)
    dy = torch.randn(m, k, generator=torch.Generator(device="cuda").manual_seed(offset), device="cuda").to(dtype)
    _, dx, dw, db = exact(x, w, b, dy)
    leaves = [placed(x, offset, k + more).detach().requires_grad_(), w.requires_grad_(), b.requires_grad_()]
    for d in (dy, placed(dy, more - offset, k + more + 1)):
        got = torch.autograd.grad(w8.layer_norm(*leaves, EPS), leaves, d)
        for g, (want, bound), name in zip(got, (dx, dw, db), ("dx", "dw", "db")):
            assert_within(g, want, bound, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_gradients_with_a_residual(k, dtype):
    m = 21
    x, w, b, res = inputs(m, k, dtype, True, seed=k)
    gen = torch.Generator(device="cuda").manual_seed(1)
    dy, dh = (torch.randn(m, k, generator=gen, device="cuda").to(dtype) for _ in range(2))
    h = (x.double() + res.double()).float().to(dtype)
    _, dx, dw, db = exact(h, w, b, dy, dh)
    leaves = [placed(x, 3, k + 5).detach().requires_grad_(), w.requires_grad_(), b.requires_grad_(), placed(res, 1, k + 2).detach().requires_grad_()]
    for o in (0, 1, 5):
        out = w8.layer_norm(leaves[0], leaves[1], leaves[2], EPS, leaves[3])
        assert torch.equal(out[1], h)
        got = torch.autograd.grad(out, leaves, (placed(dy, 7 - o, k + 7), placed(dh, o, k + 6)))
        for g, (want, bound), name in zip(got, (dx, dw, db, dx), ("dx", "dw", "db", "dresidual")):
            assert_within(g, want, bound, name)
