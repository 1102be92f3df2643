"""The operators of the 8-bit path that are measured, as a user's program calls them, and their plain forms.

A case is one pass through one operator:

  layer_norm   layer norm, forward alone (serving) or with its gradients (tuning norms)
  quantize     int8 codes and a scale for every token
  norm         residual add, layer norm or RMSNorm, and the codes of the result (what a decoder block does in front of a linear)
  product      the product of token codes and channel codes, scaled, with or without a bias
  corrected    a whole linear from its 16-bit input: codes, the right factor's product, the int8 product, the left factor's part

Codes are whole numbers (a scale lies beside them), so both sides have to give the same ones: a code is the nearest integer of the exact
quotient of a value and its token's fp32 scale.  Behind a norm every rounding on the way there is part of the definition, and the
statistics are taken in 64 bits and rounded once.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-5


def listed():
    return [
        # one token through the norm of an OPT block, in front of its projections: nothing but latency
        dict(name="layer-norm-2048-m1", op="layer_norm", m=1, k=2048, dtype="fp16", residual=True, train=False),
        # sixteen sequences of 2048 tokens while norms are tuned: forward and all gradients
        dict(name="layer-norm-2048-m32768-grad", op="layer_norm", m=32768, k=2048, dtype="fp16", residual=False, train=True),
        # one token's activations in front of a 13B projection
        dict(name="quantize-5120-m1", op="quantize", m=1, k=5120, dtype="fp16"),
        # the input of a 13B down projection for a long prompt, a bf16 model
        dict(name="quantize-13824-m4096", op="quantize", m=4096, k=13824, dtype="bf16"),
        # a decode step of seven requests of an OPT model: residual, layer norm, codes
        dict(name="norm-layer-2048-m7", op="norm", m=7, k=2048, dtype="fp16", kind="layer", residual=True),
        # a prompt of a 13B Llama: residual, RMSNorm, codes
        dict(name="norm-rms-5120-m4000", op="norm", m=4000, k=5120, dtype="fp16", kind="rms", residual=True),
        # an OPT projection for one token, with its bias
        dict(name="product-2048-2048-m1", op="product", m=1, k=2048, n=2048, out="fp16", bias=True),
        # gate and up of a 13B layer for a batch of sixteen decoding requests
        dict(name="product-5120-27648-m16", op="product", m=16, k=5120, n=27648, out="fp16", bias=False),
        # a 13B up projection for a long prompt, a bf16 model
        dict(name="product-5120-13824-m4096", op="product", m=4096, k=5120, n=13824, out="bf16", bias=False),
        # a corrected 13B output projection for one token
        dict(name="corrected-5120-5120-m1", op="corrected", m=1, k=5120, n=5120, rank=128, out="fp16", bias=False),
        # a corrected 7B down projection for a short prompt of odd length, long rows
        dict(name="corrected-18944-3584-m77", op="corrected", m=77, k=18944, n=3584, rank=128, out="fp16", bias=True),
        # gate and up of a 13B layer, corrected, for a prompt
        dict(name="corrected-5120-27648-m2048", op="corrected", m=2048, k=5120, n=27648, rank=128, out="fp16", bias=False),
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    op = rng.choice(["layer_norm", "quantize", "norm", "product", "product", "corrected", "corrected"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    if op in ("layer_norm", "quantize", "norm"):
        k = _log_int(rng, 96, 20000)
        m = _log_int(rng, 1, max(1, min(32768, 60_000_000 // k)))
        if op == "layer_norm":
            return dict(op=op, m=m, k=k, dtype=dtype, residual=rng.random() < 0.5, train=rng.random() < 0.5)
        if op == "quantize":
            return dict(op=op, m=m, k=k, dtype=dtype)
        return dict(op=op, m=m, k=k, dtype=dtype, kind=rng.choice(["layer", "rms"]), residual=rng.random() < 0.5)
    k, n = _log_int(rng, 512, 19000), _log_int(rng, 512, 28000)
    if rng.random() < 0.5:      # most models' sizes are multiples of 64
        k, n = max(512, k // 64 * 64), max(512, n // 64 * 64)
    m = _log_int(rng, 1, max(1, min(4096, 280_000_000_000 // (k * n))))
    if op == "product":
        return dict(op=op, m=m, k=k, n=n, out=rng.choice(["fp16", "bf16", "fp32"]), bias=rng.random() < 0.5)
    return dict(op=op, m=m, k=k, n=n, rank=rng.choice([16, 40, 64, 128, 256]), out=rng.choice(["fp16", "fp32"]), bias=rng.random() < 0.5)


def _activations(m, k, gen, dtype):
    """Activations with the few large channels that make tokens' scales differ."""
    x = torch.randn(m, k, generator=gen, device="cuda")
    loud = torch.rand(k, generator=gen, device="cuda") < 0.004
    x *= torch.where(loud, 20.0, 1.0) * torch.exp(0.3 * torch.randn(m, 1, generator=gen, device="cuda"))
    return x.to(dtype)


def _codes(rows, k, gen):
    """int8 codes as a quantiser leaves them, rows at a multiple of 16 bytes, and fp32 scales."""
    pitch = (k + 15) // 16 * 16
    w = torch.randn(rows, pitch, generator=gen, device="cuda")
    w[:, k:] = 0
    top = w.abs().amax(dim=1, keepdim=True)
    codes = torch.round(w / top * 127.0).to(torch.int8)
    return codes[:, :k], (top[:, 0] * 0.02 / 127.0).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = dict(case)
    op, m, k = c["op"], c["m"], c["k"]
    if op in ("layer_norm", "quantize", "norm"):
        dtype = _DTYPES[c["dtype"]]
        c["x"] = _activations(m, k, gen, dtype)
        if op == "quantize":
            return c
        c["res"] = _activations(m, k, gen, dtype) if c["residual"] else None
        c["w"] = (1.0 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
        with_bias = op == "layer_norm" or c["kind"] == "layer"
        c["b"] = (0.1 * torch.randn(k, generator=gen, device="cuda")).to(dtype) if with_bias else None
        if op == "layer_norm" and c["train"]:
            c["dy"] = (0.1 * torch.randn(m, k, generator=gen, device="cuda")).to(dtype)
            c["dh"] = (0.1 * torch.randn(m, k, generator=gen, device="cuda")).to(dtype) if c["residual"] else None
            for name in ("x", "w", "b"):
                c[name].requires_grad_()
            if c["residual"]:
                c["res"].requires_grad_()
        return c
    c["q"], c["qs"] = _codes(c["n"], k, gen)
    c["bias"] = 0.1 * torch.randn(c["n"], generator=gen, device="cuda") if case["bias"] else None
    if op == "product":
        c["t"], c["ts"] = _codes(m, k, gen)
        return c
    c["x"] = _activations(m, k, gen, torch.float16)
    c["R"] = (torch.randn(c["rank"], k, generator=gen, device="cuda") / math.sqrt(k)).to(torch.float16)
    c["L"] = (0.02 * torch.randn(c["n"], c["rank"], generator=gen, device="cuda")).to(torch.float16)
    c["alpha"] = 0.9
    return c


# ---------------------------------------------------------------- plain forms
def _plain_quantize(x):
    x = x.float()
    top = x.abs().amax(dim=1)
    scales = top / torch.full_like(top, 127.0)      # (a scalar divisor would be taken as a product with its reciprocal)
    # the quotient lies next to a border where 32 bits cannot tell the side
    q = torch.round(x.double() / scales.double()[:, None]).clamp(-127, 127)
    codes = torch.where(scales[:, None] > 0, q, torch.zeros_like(q)).to(torch.int8)
    return codes, scales


def _plain_norm(x, res, w, b, kind):
    """(what is normalised, the normalised rows in x's type, mean, reciprocal deviation)"""
    dtype = x.dtype
    h = x if res is None else (x.float() + res.float()).to(dtype)
    v = h.double()
    if kind == "rms":
        rstd = (1.0 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS)).float()
        t = (h.float() * rstd).to(dtype)
        return h, (w.float() * t.float()).to(dtype), None, rstd
    mean64 = v.mean(dim=1, keepdim=True)
    rstd = (1.0 / torch.sqrt(((v - mean64) ** 2).mean(dim=1, keepdim=True) + EPS)).float()
    mean = mean64.float()
    t = (h.float() - mean) * rstd
    return h, (t.double() * w.double() + b.double()).float().to(dtype), mean, rstd


def _plain_product(codes, scales, q, qs):
    return (codes.double() @ q.double().t()) * scales.double()[:, None] * qs.double()


def _run_plain(s):
    op = s["op"]
    if op == "quantize":
        return _plain_quantize(s["x"])
    if op == "norm":
        h, y, _, _ = _plain_norm(s["x"], s["res"], s["w"], s["b"], s["kind"])
        codes, scales = _plain_quantize(y)
        return (codes, scales, h) if s["residual"] else (codes, scales)
    if op == "layer_norm":
        x, w, b = s["x"], s["w"], s["b"]
        h, y, mean, rstd = _plain_norm(x, s["res"], w, b, "layer")
        if not s["train"]:
            return (y, h) if s["residual"] else (y,)
        dy, xh = s["dy"].float(), (h.float() - mean) * rstd
        g = dy * w.float()
        dx = rstd * (g - g.mean(dim=1, keepdim=True) - xh * (g * xh).mean(dim=1, keepdim=True))
        dw, db = (dy * xh).sum(dim=0), dy.sum(dim=0)
        if s["residual"]:
            dx = dx + s["dh"].float()
            return y, h, dx.to(x.dtype), dx.to(x.dtype), dw.to(x.dtype), db.to(x.dtype)
        return y, dx.to(x.dtype), dw.to(x.dtype), db.to(x.dtype)
    out = _DTYPES[s["out"]]
    if op == "product":
        y = _plain_product(s["t"], s["ts"], s["q"], s["qs"])
    else:
        codes, scales = _plain_quantize(s["x"])
        r = (s["x"].float() @ s["R"].float().t()).to(torch.float16)
        y = _plain_product(codes, scales, s["q"], s["qs"]) + s["alpha"] * (r.float() @ s["L"].float().t()).double()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return (y.to(out),)


# ---------------------------------------------------------------- the framework's calls
def _run_own(s):
    from glowq_b200 import cuda_w8a8 as w8
    op = s["op"]
    if op == "quantize":
        t = w8.quantize_tokens(s["x"])
        return t.codes, t.scales
    if op == "norm":
        t, h = w8.norm_quantize_tokens(s["x"], s["w"], s["b"], eps=EPS, residual=s["res"], norm=s["kind"])
        return (t.codes, t.scales, h) if s["residual"] else (t.codes, t.scales)
    if op == "layer_norm":
        out = w8.layer_norm(s["x"], s["w"], s["b"], eps=EPS, residual=s["res"])
        if not s["residual"]:
            return (out, *torch.autograd.grad(out, (s["x"], s["w"], s["b"]), s["dy"])) if s["train"] else (out,)
        if not s["train"]:
            return out
        grads = torch.autograd.grad(out, (s["x"], s["res"], s["w"], s["b"]), (s["dy"], s["dh"]))
        return (*out, *grads)
    out = _DTYPES[s["out"]]
    if op == "product":
        return (w8.w8a8_linear(w8.TokenCodes(s["t"], s["ts"]), s["q"], s["qs"], s["bias"], out_dtype=out),)
    return (w8.w8a8_linear(s["x"], s["q"], s["qs"], s["bias"], out_dtype=out, L=s["L"], R=s["R"], alpha=s["alpha"]),)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    if op in ("layer_norm", "quantize", "norm"):
        e = _SIZE[case["dtype"]]
        if op == "quantize":
            return {"bytes": m * k * (e + 1) + 4 * m, "flops": 6 * m * k}
        both = 2 if case["residual"] else 1
        if op == "norm":
            return {"bytes": m * k * (e * (2 * both - 1) + 1) + 4 * m + 2 * k * e, "flops": 16 * m * k}
        forward = m * k * e * 2 * both + 2 * k * e
        if not case["train"]:
            return {"bytes": forward, "flops": 10 * m * k}
        # the gradients read what was normalised and dy (and the gradient of the sum), and write dx, dw, db
        return {"bytes": forward + m * k * e * (2 + both) + 3 * k * e, "flops": 28 * m * k}
    n = case["n"]
    out = _SIZE[case["out"]]
    bias = 4 * n if case["bias"] else 0
    if op == "product":
        return {"bytes": n * k + m * k + m * n * out + 4 * (m + n) + bias, "flops": 2 * m * n * k}
    rank = case["rank"]
    return {"bytes": n * k + 2 * m * k + 2 * rank * (k + n) + m * n * out + 4 * n + bias, "flops": 2 * m * n * k + 2 * m * rank * (k + n)}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_codes(y):
    """Codes of rows that are held in their own type: s = fp32(max / 127), the nearest integer of y / s."""
    v = y.to(torch.float64)
    s32 = (torch.max(torch.abs(v), dim=-1).values / 127.0).to(torch.float32)
    s = s32.to(torch.float64).unsqueeze(-1)
    ratio = torch.where(s > 0, torch.divide(v, torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(v))
    return torch.round(ratio).to(torch.int8), s32


def _exact_stats(h):
    v = h.to(torch.float64)
    mean = torch.einsum("mk->m", v) / v.shape[1]
    dev = v - mean.unsqueeze(-1)
    return v, mean, torch.einsum("mk,mk->m", dev, dev) / v.shape[1]


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    with torch.no_grad():
        if op == "quantize":
            return _exact_codes(s["x"])
        if op in ("norm", "layer_norm"):
            x = s["x"].detach()
            h = x if s["res"] is None else torch.add(x.to(torch.float64), s["res"].detach().to(torch.float64)).to(torch.float32).to(x.dtype)
        if op == "norm":
            v, mean, var = _exact_stats(h)
            w = s["w"].to(torch.float64)
            if s["kind"] == "rms":
                rs = torch.rsqrt(torch.einsum("mk,mk->m", v, v) / v.shape[1] + EPS).to(torch.float32).to(torch.float64)
                t = (v * rs.unsqueeze(-1)).to(torch.float32).to(h.dtype).to(torch.float64)
                y = (t * w).to(torch.float32).to(h.dtype)
            else:
                mu = mean.to(torch.float32).to(torch.float64)
                rs = torch.rsqrt(var + EPS).to(torch.float32).to(torch.float64)
                t = (v - mu.unsqueeze(-1)).to(torch.float32).to(torch.float64)
                t = (t * rs.unsqueeze(-1)).to(torch.float32).to(torch.float64)
                y = torch.addcmul(s["b"].to(torch.float64), t, w).to(torch.float32).to(h.dtype)
            codes, scales = _exact_codes(y)
            return (codes, scales, h) if s["residual"] else (codes, scales)
        if op == "layer_norm":
            v, mean, var = _exact_stats(h)
            rs = torch.rsqrt(var + EPS).unsqueeze(-1)
            xh = (v - mean.unsqueeze(-1)) * rs
            w, b = s["w"].detach().to(torch.float64), s["b"].detach().to(torch.float64)
            y = xh * w + b
            if not s["train"]:
                return (y, h.to(torch.float64)) if s["residual"] else (y,)
            dy = s["dy"].to(torch.float64)
            g = dy * w
            k = g.shape[1]
            dx = (g - torch.einsum("mk->m", g).unsqueeze(-1) / k - xh * (torch.einsum("mk,mk->m", g, xh).unsqueeze(-1) / k)) * rs
            dw, db = torch.einsum("mk,mk->k", dy, xh), torch.einsum("mk->k", dy)
            if s["residual"]:
                dx = dx + s["dh"].to(torch.float64)
                return y, h.to(torch.float64), dx, dx, dw, db
            return y, dx, dw, db
        qf = s["q"].to(torch.float64) * s["qs"].to(torch.float64).unsqueeze(-1)
        if op == "product":
            y = torch.nn.functional.linear(s["t"].to(torch.float64) * s["ts"].to(torch.float64).unsqueeze(-1), qf)
        else:
            codes, scales = _exact_codes(s["x"])
            y = torch.nn.functional.linear(codes.to(torch.float64) * scales.to(torch.float64).unsqueeze(-1), qf)
            x = s["x"].to(torch.float64)
            y = y + s["alpha"] * torch.einsum("mr,nr->mn", torch.einsum("mk,rk->mr", x, s["R"].to(torch.float64)), s["L"].to(torch.float64))
        return (y if s["bias"] is None else y + s["bias"].to(torch.float64),)
