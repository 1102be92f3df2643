"""The largest sizes of the 8-bit entry points: what 32 bits do not number is refused, what they do works."""
import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from glowq_b200.cuda_w8a8 import kernels as K
from w8a8_reference import assert_within, codes_of, product_of
from test_w8a8_host import A, LARGE, rows_desc


def linear_desc(**kw):
    d = dict(x=0, codes=A, scales=A, weight=A, weight_scales=A, bias=0, r_x=A, R=A, r=A, L=A, out=A, stream=0, x_stride=0, code_stride=64,
             weight_stride=64, r_x_stride=64, R_stride=64, r_stride=16, L_stride=16, out_stride=32, M=4, K=64, OC=32, rank=16, x_dtype=0, out_dtype=0,
             r_mode=0, alpha=1.0, reserved=0)
    d.update(kw)
    return K.pack_linear.pack(*(d[n] for n, _ in K.Linear._fields_))


# (the calls are refused before an address of theirs is looked at; what is in range is not called with these addresses)
@pytest.mark.parametrize("sizes", [dict(M=(1 << 30) + 1), dict(M=(1 << 31) - 1), dict(K=(1 << 29) + 1, x_stride=1 << 40, code_stride=1 << 40)])
def test_rows_past_32_bits_are_refused(sizes):
    assert K.ext().quantize(rows_desc(**sizes)) == LARGE
    assert K.ext().layer_norm_forward(rows_desc(codes=0, scales=0, y=A, norm=1, weight=A, y_stride=1 << 40, **sizes)) == LARGE
    g = dict(h=A, dy=A, dh=0, weight=A, mean=A, rstd=A, dx=A, dweight=A, dbias=A, workspace=A, workspace_bytes=1 << 60, stream=0, h_stride=1 << 40,
             dy_stride=1 << 40, dh_stride=0, dx_stride=1 << 40, M=4, K=64, dtype=0, reserved=0)
    g.update({n: v for n, v in sizes.items() if n in g})
    assert K.ext().layer_norm_backward(K.pack_grad.pack(*(g[n] for n, _ in K.LayerNormGrad._fields_))) == LARGE


def test_linears_past_32_bits_are_refused():
    assert K.ext().linear(linear_desc(OC=(1 << 29) + 1, out_stride=1 << 40)) == LARGE
    assert K.ext().right_factor(linear_desc(K=(1 << 29) + 1, r_x_stride=1 << 34, R_stride=1 << 34)) == LARGE
    assert K.ext().right_factor(linear_desc(M=(1 << 22) + 1)) == LARGE


@pytest.mark.gpu
def test_as_many_tokens_as_are_taken():
    m, k, n, rank = 1 << 22, 16, 24, 3
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(m, k, generator=gen, device="cuda").half()
    q, qs = w8.quantize_channels(torch.randn(n, k, generator=gen, device="cuda"))
    L, R = (torch.randn(*s, generator=gen, device="cuda").half() for s in ((n, rank), (rank, k)))
    t = w8.quantize_tokens(x)._replace(r=w8.right_factor(x, R))
    y = w8.w8a8_linear(t, q, qs, L=L, alpha=0.5)
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        codes, scales = codes_of(x[rows])
        assert torch.equal(t.codes[rows], codes)
        assert (t.r[rows].double() - x[rows].double() @ R.double().t()).abs().max() < 0.02
        assert_within(y[rows], *product_of(codes, scales, q, qs, None, 0.5, t.r[rows], L))
    with pytest.raises(RuntimeError, match="tokens"):
        w8.right_factor(torch.empty(m + 1, 8, dtype=torch.float16, device="cuda"), R[:, :8])
    w8.read_status()
