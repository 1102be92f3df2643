"""The 8-bit linear against its definition in 64 bits."""
import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from w8a8_reference import HALF_STEP, U, assert_within, codes_of, product_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    w8.read_status()


def operands(m, k, n, rank=0, bias=True, seed=0, dtype=torch.float16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = (rand(m, k) * torch.exp(0.5 * rand(m, 1))).to(dtype)
    q, qs = w8.quantize_channels((0.02 * rand(n, k)).to(torch.float16))
    b = 0.1 * rand(n) if bias else None
    if not rank:
        return x, q, qs, b
    return x, q, qs, b, (0.05 * rand(n, rank)).to(torch.float16), (rand(rank, k) / k ** 0.5).to(torch.float16)


SIZES = [(1, 16, 8), (1, 1, 1), (1, 129, 130), (2, 2048, 2048), (5, 37, 300), (16, 1000, 128), (17, 640, 512), (33, 512, 257), (64, 2048, 130),
         (65, 256, 384), (100, 777, 999), (128, 1024, 256), (129, 384, 640), (256, 512, 512), (300, 1536, 768), (777, 321, 511)]


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_products(m, k, n, out):
    x, q, qs, b = operands(m, k, n, seed=m + k)
    t = w8.quantize_tokens(x)
    y = w8.w8a8_linear(t, q, qs, b, out_dtype=out)
    want, bound = product_of(*codes_of(x), q, qs, b)
    assert y.dtype == out and y.shape == (m, n)
    assert_within(y, want, bound)
    assert torch.equal(w8.w8a8_linear(x, q, qs, b, out_dtype=out), y)      # codes made in the call
    y = w8.w8a8_linear(t, q, qs, out_dtype=out)
    assert_within(y, *product_of(*codes_of(x), q, qs, None))


def right_factor_of(x, R):
    """(r in 64 bits, bound before rounding to fp16)"""
    a = x.to(torch.float16).double()
    mag = a.abs() @ R.double().abs().t()
    return a @ R.double().t(), (2 * x.shape[1] + 4) * U * mag


@pytest.mark.parametrize("m,k,n,rank", [(1, 512, 300, 16), (1, 5120, 128, 128), (3, 333, 200, 40), (20, 2048, 512, 64), (64, 640, 130, 256),
                                        (77, 1024, 384, 7), (130, 512, 640, 128), (300, 768, 257, 100), (257, 520, 520, 1024), (1, 8, 8, 1), (16, 5120, 256, 128), (15, 264, 130, 33), (2, 18944, 64, 256)])
@pytest.mark.parametrize("out", [torch.float16, torch.float32])
def test_corrected(m, k, n, rank, out):
    x, q, qs, b, L, R = operands(m, k, n, rank, seed=rank)
    r = w8.right_factor(x, R)
    assert r.shape == (m, rank) and r.dtype == torch.float16
    assert_within(r, *right_factor_of(x, R))
    for bias in (b, None):
        want, bound = product_of(*codes_of(x), q, qs, bias, 0.7, r, L)
        t = w8.quantize_tokens(x)._replace(r=r)
        assert_within(w8.w8a8_linear(t, q, qs, bias, out_dtype=out, L=L, alpha=0.7), want, bound)
        # r made in the call, whose sums may be taken in another order (of a few tokens): each r_j is off by the bound of right_factor_of
        # and its rounding, here and above
        exact, off = right_factor_of(x, R)
        off = 2 * (off + HALF_STEP[torch.float16] * (exact.abs() + off) + 2.0 ** -25)
        y = w8.w8a8_linear(x, q, qs, bias, out_dtype=out, L=L, R=R, alpha=0.7)
        assert_within(y, want, bound + 0.7 * (off @ L.double().abs().t()))


@pytest.mark.parametrize("m", [9, 300])
def test_alpha_zero_small_and_large(m):
    x, q, qs, b, L, R = operands(m, 512, 256, 64)
    plain = w8.w8a8_linear(x, q, qs, b, out_dtype=torch.float32)
    assert torch.equal(w8.w8a8_linear(x, q, qs, b, out_dtype=torch.float32, L=L, R=R, alpha=0.0), plain)
    r = w8.right_factor(x, R)
    t = w8.quantize_tokens(x)._replace(r=r)
    for alpha in (-1e4, 1e-20):
        y = w8.w8a8_linear(t, q, qs, b, out_dtype=torch.float32, L=L, alpha=alpha)
        assert_within(y, *product_of(*codes_of(x), q, qs, b, alpha, r, L))


@pytest.mark.parametrize("m", [1, 3, 70, 300])
def test_sums_are_exact_at_the_largest_codes(m):
    """Codes of -128 (which no quantiser here makes) and 127 over long rows: sums near 2^31."""
    k, n = 131071, 256
    t = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    t[0] = 127
    q = torch.full((n, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    q[1::2] = 127
    ones = torch.ones(max(m, n), device="cuda")
    y = w8.w8a8_linear(w8.TokenCodes(t, ones[:m]), q, ones[:n], out_dtype=torch.float32)
    want = (t[:, :1].double() * q[:, 0].double()) * k
    assert torch.equal(y, want.float())


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_tokens_with_nan_and_infinity(m, dtype):
    x, q, qs, b, L, R = operands(m + 3, 512, 256, 32, dtype=dtype)
    x[0, 3] = float("nan")
    x[2, 5] = float("-inf")
    x[1] = 0
    y = w8.w8a8_linear(x, q, qs, b, out_dtype=torch.float32, L=L, R=R)
    assert torch.isnan(y[0]).all() and torch.isnan(y[2]).all()
    assert torch.equal(y[1], b)
    assert torch.isfinite(y[1]).all() and torch.isfinite(y[3:]).all()
    clean = x.clone()
    clean[[0, 2]] = 0
    z = w8.w8a8_linear(clean, q, qs, b, out_dtype=torch.float32, L=L, R=R)
    keep = [1, *range(3, m + 3)]
    assert torch.equal(y[keep], z[keep])


@pytest.mark.parametrize("m", [2, 70, 260])
def test_strides_alignment_and_neighbours(m):
    """Operands that are parts of larger tensors; columns behind K and rows behind the last token hold what must not be used."""
    k, n, rank = 500, 200, 24
    x, q, qs, b, L, R = operands(m, k, n, rank)
    want = w8.w8a8_linear(x, q, qs, b, L=L, R=R, alpha=0.5)
    wide = torch.full((m + 2, k + 13), float("nan"), dtype=torch.float16, device="cuda")
    wide[1:m + 1, 5:k + 5] = x
    assert torch.equal(w8.w8a8_linear(wide[1:m + 1, 5:k + 5], q, qs, b, L=L, R=R, alpha=0.5), want)
    wide = torch.full((n + 1, k + 28), 99, dtype=torch.int8, device="cuda")     # rows 528 bytes apart
    wide[:n, :k] = q
    odd = torch.full((n + 1, k + 27), 99, dtype=torch.int8, device="cuda")      # rows that do not begin on 16 bytes
    odd[1:, 3:k + 3] = q
    wideL = torch.full((n, rank + 5), float("nan"), dtype=torch.float16, device="cuda")
    wideL[:, 2:rank + 2] = L
    for weight in (wide[:n, :k], odd[1:, 3:k + 3]):
        assert torch.equal(w8.w8a8_linear(x, weight, qs, b, L=wideL[:, 2:rank + 2], R=R, alpha=0.5), want)
    t = w8.quantize_tokens(x)
    odd = torch.full((m, k + 7), 55, dtype=torch.int8, device="cuda")
    odd[:, 1:k + 1] = t.codes
    t = t._replace(r=w8.right_factor(x, R))
    assert torch.equal(w8.w8a8_linear(t._replace(codes=odd[:, 1:k + 1]), q, qs, b, L=L, alpha=0.5),
                       w8.w8a8_linear(t, q, qs, b, L=L, alpha=0.5))
    y = w8.w8a8_linear(x.reshape(1, m, k), q, qs, b, L=L, R=R, alpha=0.5)
    assert y.shape == (1, m, n) and torch.equal(y[0], want)


def test_outputs_keep_to_their_rows():
    """The C call with a wider output: columns behind the last channel and rows behind the last token stay as they were."""
    from glowq_b200.cuda_w4a16.kernels import current_stream_ptr
    from glowq_b200.cuda_w8a8 import kernels as K
    for m, n, pitch in ((3, 130, 137), (70, 257, 264), (300, 259, 300), (300, 256, 264)):
        x, q, qs, b = operands(m, 256, n)
        t = w8.quantize_tokens(x)
        for dtype in (torch.float16, torch.float32):
            out = torch.full((m + 2, pitch), 7.0, dtype=dtype, device="cuda")
            desc = K.pack_linear.pack(0, t.codes.data_ptr(), t.scales.data_ptr(), q.data_ptr(), qs.data_ptr(), b.data_ptr(), 0, 0, 0, 0,
                                      out.data_ptr(), current_stream_ptr(out.device), 0, t.codes.stride(0), q.stride(0), 0, 0, 0, 0, pitch,
                                      m, 256, n, 0, 0, K.DTYPES[dtype], K.R_NONE, 0.0, 0)
            K.call(K.ext().linear, out.device, desc, "glowq_w8a8_linear")
            assert torch.equal(out[:m, :n], w8.w8a8_linear(t, q, qs, b, out_dtype=dtype))
            assert (out[m:] == 7).all() and (out[:, n:] == 7).all()


def test_types_of_outputs():
    x, q, qs, b = operands(4, 256, 64)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        assert w8.w8a8_linear(x.to(dtype), q, qs, b).dtype == dtype
    assert w8.w8a8_linear(w8.quantize_tokens(x), q, qs, b).dtype == torch.float16
    assert w8.w8a8_linear(x[:0], q, qs, b).shape == (0, 64)
    assert w8.w8a8_linear(x, q[:0], qs[:0]).shape == (4, 0)


@pytest.mark.parametrize("m", [1, 200])
def test_graphs_and_streams(m):
    """A captured call replayed with other inputs, and two streams at once."""
    x, q, qs, b, L, R = operands(m, 1024, 512, 64)
    x2 = operands(m, 1024, 512, seed=9)[0]
    call = lambda v: w8.w8a8_linear(v, q, qs, b, L=L, R=R, alpha=0.9)  # noqa: E731
    want, want2 = call(x), call(x2)
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(static)
    for v, w in ((x2, want2), (x, want)):
        static.copy_(v)
        graph.replay()
        assert torch.equal(y, w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, v in zip(streams, (x, x2)):
            with torch.cuda.stream(s):
                got.append(call(v))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, (want, want2)[i & 1])
    w8.read_status()


def test_threads():
    """Calls from several threads at once, each on a stream of its own."""
    import threading
    jobs = []
    for i, m in enumerate((1, 3, 60, 300)):
        x, q, qs, b, L, R = operands(m, 1024, 512, 64, seed=i)
        jobs.append((x, q, qs, b, L, R, w8.w8a8_linear(x, q, qs, b, L=L, R=R)))
    torch.cuda.synchronize()
    wrong = []

    def work(x, q, qs, b, L, R, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                y = w8.w8a8_linear(x, q, qs, b, L=L, R=R)
            torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want):
                wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_weights_made_right_before_they_are_used():
    """Weights that the call in front quantised: the product does not read them early."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, 2048, generator=gen, device="cuda", dtype=torch.float16)
    t = w8.quantize_tokens(x)
    ws = [torch.randn(2048, 2048, generator=gen, device="cuda", dtype=torch.float16) for _ in range(2)]
    want = []
    for w in ws:
        q, qs = w8.quantize_channels(w)
        torch.cuda.synchronize()
        want.append(w8.w8a8_linear(t, q, qs))
    for i in range(20):
        q, qs = w8.quantize_channels(ws[i & 1])
        assert torch.equal(w8.w8a8_linear(t, q, qs), want[i & 1])
        q.zero_()
        del q, qs


@pytest.mark.parametrize("m,k,n", [(260, 256, 2000), (260, 256, 4000), (260, 256, 5000), (260, 256, 9000), (600, 384, 20000), (1500, 130, 9000),
                                   (70, 640, 30000), (40, 256, 20001)])
def test_tiles_of_every_width_and_rounds_of_them(m, k, n):
    """Pairs on tiles of 64 to 256 channels, one and several to a pair (a corrected tile ends among the next one's steps), two CTAs to an SM."""
    x, q, qs, b, L, R = operands(m, k, n, 72)
    t = w8.quantize_tokens(x)._replace(r=w8.right_factor(x, R))
    for out in (torch.float16, torch.float32):
        assert_within(w8.w8a8_linear(t, q, qs, b, out_dtype=out), *product_of(*codes_of(x), q, qs, b))
        assert_within(w8.w8a8_linear(t, q, qs, b, out_dtype=out, L=L, alpha=0.6), *product_of(*codes_of(x), q, qs, b, 0.6, t.r, L))


def test_many_channels_and_tokens():
    for m, k, n in ((5000, 128, 300), (9, 128, 40_000), (1, 64, 70_001)):
        x, q, qs, b = operands(m, k, n)
        assert_within(w8.w8a8_linear(x, q, qs, b), *product_of(*codes_of(x), q, qs, b))


def test_same_bits_every_time():
    for m in (1, 33, 500):
        x, q, qs, b, L, R = operands(m, 3000, 700, 128)
        first = w8.w8a8_linear(x, q, qs, b, L=L, R=R)
        for _ in range(5):
            assert torch.equal(w8.w8a8_linear(x, q, qs, b, L=L, R=R), first)


def test_how_far_eight_bits_are():
    """Against the 16-bit linear: two roundings to 8 bits, each of half a step at most."""
    x, q, qs, b = operands(32, 2048, 512)
    w = q.double() * qs.double()[:, None]
    y = w8.w8a8_linear(x, q, qs, out_dtype=torch.float32)
    s = codes_of(x)[1].double()
    limit = 0.5 * s[:, None] * w.abs().sum(dim=1)            # the tokens' rounding; the weights are their codes here
    assert ((y.double() - x.double() @ w.t()).abs() <= limit * (1 + 1e-5) + HALF_STEP[torch.float32]).all()


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows' codes, norms, products and r."""
    m, k, n = 131_104, 16_400, 72
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 40 GB")
    x = torch.zeros(m, k, dtype=torch.float16, device="cuda")
    rows = torch.tensor([0, 5, m // 2, m - 200, m - 1], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    some = torch.randn(len(rows), k, generator=gen, device="cuda").half()
    x[rows] = some
    t = w8.quantize_tokens(x)
    codes, scales = codes_of(some)
    assert torch.equal(t.codes[rows], codes) and torch.equal(t.scales[rows], scales)
    _, q, qs, b, L, R = operands(1, k, n, 24)
    r = w8.right_factor(x, R)
    assert_within(r[rows], *right_factor_of(some, R))
    y = w8.w8a8_linear(t._replace(r=r), q, qs, b, L=L, alpha=0.5)
    want, bound = product_of(codes, scales, q, qs, b, 0.5, r[rows], L)
    assert_within(y[rows], want, bound)
    assert_within(y[1:5], *product_of(torch.zeros_like(codes[:4]), torch.zeros_like(scales[:4]), q, qs, b, 0.5, r[1:5], L))
    del t, y
    w = torch.ones(k, dtype=torch.float16, device="cuda")
    ln = w8.layer_norm(x, w)
    assert torch.equal(ln[rows], w8.layer_norm(some, w)) and not ln[1].any()
    del ln
    leaf, wl = x.requires_grad_(), w.clone().requires_grad_()
    dy = torch.zeros(m, k, dtype=torch.float16, device="cuda")
    dy[rows] = some.flip(0)
    gx, gw = torch.autograd.grad(w8.layer_norm(leaf, wl), (leaf, wl), dy)
    small = some.clone().requires_grad_()
    sx, _ = torch.autograd.grad(w8.layer_norm(small, wl), (small, wl), some.flip(0))
    # (row sums in the same order whatever the number of rows)
    assert torch.equal(gx[rows], sx) and not gx[1].any()
