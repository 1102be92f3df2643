"""What a launch may read before the one in front of it is complete: constants, never what the operation right in front has made.  Captured
calls show how a launch hangs on the one in front: fully, or so that it may begin early."""
import ctypes

import pytest
import torch

from glowq_b200 import cuda_w8a8 as w8
from glowq_b200.cuda_w8a8 import kernels as K

pytestmark = pytest.mark.gpu


def early(call):
    """For every kernel behind the first one of a captured call, in order: may it begin while the one in front of it runs?"""
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        kept = call()
    runtime, raw = ctypes.CDLL("libcudart.so.12"), ctypes.c_void_p(graph.raw_cuda_graph())
    nodes, edges = ctypes.c_size_t(), ctypes.c_size_t()
    assert runtime.cudaGraphGetNodes(raw, None, ctypes.byref(nodes)) == 0
    assert runtime.cudaGraphGetEdges_v2(raw, None, None, None, ctypes.byref(edges)) == 0
    n = edges.value
    assert n == nodes.value - 1                                        # a chain
    tails, heads, data = (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)(), (ctypes.c_uint8 * (8 * n))()
    assert runtime.cudaGraphGetEdges_v2(raw, tails, heads, data, ctypes.byref(edges)) == 0
    edges = {tails[i]: (heads[i], data[8 * i + 2]) for i in range(n)}  # (two ports, then the type: 1 of a programmatic edge)
    at = (set(tails) - set(heads)).pop()
    order = []
    while at in edges:
        at, kind = edges[at]
        order.append(kind == 1)
    del kept
    return order


def operands(m, k, n, rank):
    gen = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    q, qs = w8.quantize_channels(rand(n, k).half())
    return rand(m, k).half(), q, qs, rand(n, rank).half(), rand(rank, k).half()


def moved(t):
    """The same matrix in rows that do not begin on 16 bytes."""
    room = torch.zeros(t.shape[0], t.shape[1] + 19, dtype=t.dtype, device="cuda")
    room[:, 1:t.shape[1] + 1] = t
    return room[:, 1:t.shape[1] + 1]


@pytest.mark.parametrize("m", [1, 3, 20, 600])
def test_constants_are_read_early_and_copies_are_not(m):
    x, q, qs, L, R = operands(m, 512, 1024, 64)
    t = w8.quantize_tokens(x)._replace(r=w8.right_factor(x, R))
    plain, corrected = w8.w8a8_linear(t, q, qs), w8.w8a8_linear(t, q, qs, L=L)
    whole = w8.w8a8_linear(x, q, qs, L=L, R=R)
    # (a copy, then the launch)
    assert early(lambda: w8.w8a8_linear(t, moved(q), qs))[-1] is False
    assert early(lambda: w8.w8a8_linear(t, q, qs, L=moved(L)))[-1] is False
    assert early(lambda: w8.right_factor(x, moved(R)))[-1] is False
    order = early(lambda: w8.w8a8_linear(x, q, qs, L=L, R=moved(R)))
    launches = 2 if m <= 4 else 3                # (codes and r of a few tokens are one)
    assert order[-launches + 1:] == [True] * (launches - 1)
    if m <= 4:
        assert order[-launches] is False
    # what a call of ours in front has made
    y = early(lambda: (w8.quantize_tokens(x), w8.w8a8_linear(t, q, qs)))
    assert y == [True]
    assert early(lambda: (w8.quantize_tokens(x), w8.w8a8_linear(t, q, qs, constant=False))) == [False]
    assert early(lambda: (w8.quantize_tokens(x), w8.right_factor(x, R, constant=False))) == [False]
    assert early(lambda: (w8.quantize_tokens(x), w8.w8a8_linear(x, q, qs, L=L, R=R, constant=False)))[:1] == [m > 4]
    for _ in range(10):
        assert torch.equal(w8.w8a8_linear(t, moved(q), qs), plain)
        assert torch.equal(w8.w8a8_linear(t, moved(q), qs, L=moved(L)), corrected)
        assert torch.equal(w8.w8a8_linear(t, q, qs, L=moved(L), constant=False), corrected)
        assert torch.equal(w8.w8a8_linear(x, q, qs, L=L, R=moved(R)), whole)
        assert torch.equal(w8.right_factor(x, moved(R)), t.r)
    w8.read_status()


def test_weights_are_complete_for_what_comes_behind_them():
    """Between the codes of a weight and the next launch stands one that waits for their end."""
    x, q, qs, _, _ = operands(4, 512, 256, 8)
    t, w = w8.quantize_tokens(x), torch.randn(256, 512, device="cuda").half()
    order = early(lambda: w8.w8a8_linear(t, *w8.quantize_channels(w)))
    assert order[-2:] == [False, True]
    want, scales = w8.quantize_channels(w)
    assert torch.equal(w8.w8a8_linear(t, *w8.quantize_channels(w)), w8.w8a8_linear(t, want, scales))


def test_weights_that_torch_has_just_made():
    x, q, qs, L, R = operands(2, 512, 2048, 32)
    t = w8.quantize_tokens(x)
    t = t._replace(r=w8.right_factor(x, R))
    for i in range(20):
        room = torch.empty_like(q)
        room.copy_(q if i % 2 else -q)
        y = w8.w8a8_linear(t, room, qs, out_dtype=torch.float32, constant=False)
        assert torch.equal(y, w8.w8a8_linear(t, q, qs, out_dtype=torch.float32) * (1 if i % 2 else -1))
        factor = L * (1.0 if i % 2 else -1.0)
        y = w8.w8a8_linear(t, q, qs, L=factor, alpha=1.0, constant=False)
        assert torch.equal(y, w8.w8a8_linear(t, q, qs, L=L, alpha=1.0 if i % 2 else -1.0))


def test_the_mode_with_the_flag():
    from test_w8a8_host import BAD
    from test_w8a8_limits import linear_desc
    assert K.ext().linear(linear_desc(r_mode=K.FRESH | 3)) == BAD
    assert K.ext().linear(linear_desc(r_mode=K.FRESH, M=0)) == 0
