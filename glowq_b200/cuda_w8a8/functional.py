"""Token codes and the 8-bit linear as functions of tensors.

    scale_t = fp32(max_k |x_tk| / 127)        code_tk = the integer nearest to x_tk / scale_t, ties to even, of the exact quotient
    y_to    = scale_t * weight_scale_o * sum_k code_tk weight_ok  +  alpha * sum_j r_tj L_oj  (+ bias_o),      r = x R^T

The sums of products are exact; the rest is fp32, rounded once to the output's type.  A token with a NaN or an infinity has scale NaN and
all its outputs are NaN; other tokens do not see it.  Everything runs on the current stream of the tensors' device, allocates its outputs
and its scratch through PyTorch, and works under a captured graph.  There are no gradients here (as in ``CudaW4A16Linear``); the layer
norm has them (``layer_norm``)."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from ..cuda_w4a16.kernels import current_stream_ptr
from . import kernels as K

_NORMS = {"layer": K.NORM_LAYER, "rms": K.NORM_RMS}
_pack_rows, _pack_linear = K.pack_rows.pack, K.pack_linear.pack
_TYPES = {code: dtype for dtype, code in K.DTYPES.items()}


class TokenCodes(NamedTuple):
    """A linear's input as int8 codes [tokens, in_features] with an fp32 scale per token [tokens].  ``r``: the right factor's product
    with the same input, fp16 [tokens, rank], for corrected linears that share one.  ``dtype``: the input's type, which a linear's output
    takes by default.  Rows of codes lie a multiple of 16 bytes apart."""
    codes: torch.Tensor
    scales: torch.Tensor
    r: Optional[torch.Tensor] = None
    dtype: Optional[torch.dtype] = None


# (Small calls cost what the host does: sizes in the place of a tuple and a known device take a third off an allocation, 0.8 us.)
_empty, _int8, _float32, _float16 = torch.empty, torch.int8, torch.float32, torch.float16


def _pitch(k: int) -> int:
    return (k + 15) & ~15


def _new_codes(m: int, k: int, device) -> torch.Tensor:
    pitch = (k + 15) & ~15
    t = _empty(m, pitch, dtype=_int8, device=device)
    return t if pitch == k else t[:, :k]


def _matrix(x: torch.Tensor, name: str):
    """``x`` as [rows, columns] with unit column stride and rows that do not overlap: (the matrix, rows, columns, row stride, device, the
    library's code of the type).  What is asked of a tensor costs up to 0.1 us each time, so it is asked once."""
    code = K.DTYPES.get(x.dtype)
    if code is not None and x.is_cuda:      # (mostly all is well)
        shape = x.shape
        if len(shape) == 2:
            (m, k), (s0, s1) = shape, x.stride()
            if m.__class__ is not int:      # (sizes are tensors under a trace)
                K.refuse_trace()
            if s1 == 1 and k > 0 and (s0 >= k or m <= 1):
                return x, m, k, s0, x.device, code
    if K.tracing():
        K.refuse_trace()
    x = _rows(x, name)
    return x, x.shape[0], x.shape[1], x.stride()[0], x.device, K.DTYPES[x.dtype]


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be CUDA (sm_100); there is no CPU path")
    if x.dtype not in K.DTYPES:
        raise RuntimeError(f"{name} must be fp16, bf16 or fp32, got {x.dtype}")
    if x.dim() != 2:
        if x.dim() == 0:
            raise RuntimeError(f"{name} must have a last dimension")
        x = x.reshape(-1, x.shape[-1])
    if x.shape[1] == 0:
        raise RuntimeError(f"{name} must have columns")
    stride = x.stride()
    if (stride[1] != 1 and x.shape[1] > 1) or (stride[0] < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


def _place(t: torch.Tensor, e: int, rows: int, cols: int):
    """(tensor, address, row stride, flag) of a matrix [rows, cols] of ``e``-byte elements as the copy engine reads it: rows that begin on 16 bytes.
    (Others are copied; what the package makes lies so.  Of a single row the stride may be anything: the library is told one that it
    accepts.)  The flag is ``K.FRESH`` for a copy, which a launch right behind it may not read early, else 0."""
    at, (s0, s1) = t.data_ptr(), t.stride()
    if not at & 15 and s1 == 1:
        if rows > 1:
            if s0 >= cols and not s0 * e & 15:
                return t, at, s0, 0
        else:
            per = 16 // e
            return t, at, (cols + per - 1) // per * per, 0
    per = 16 // e
    pitch = (cols + per - 1) // per * per
    room = _empty(rows, pitch, dtype=t.dtype, device=t.device)
    room[:, :cols].copy_(t)
    return room, room.data_ptr(), pitch, K.FRESH


def _quantize(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, constant: bool) -> None:
    desc = _pack_rows(x.data_ptr(), 0, 0, 0, 0, 0, codes.data_ptr(), scales.data_ptr(), 0, 0, current_stream_ptr(x.device), 0.0,
                      x.stride()[0], 0, 0, 0, codes.stride()[0], x.shape[0], x.shape[1], K.DTYPES[x.dtype], K.NORM_NONE, constant, 0)
    K.call(K.ext().quantize, x.device, desc, "glowq_w8a8_quantize")


def quantize_tokens(x: torch.Tensor) -> TokenCodes:
    """int8 codes and a scale for every row of ``x`` [..., in_features] (fp16, bf16 or fp32), in one launch."""
    x, m, k, stride, dev, code = _matrix(x, "x")
    pitch = (k + 15) & ~15
    codes = _empty(m, pitch, dtype=_int8, device=dev)
    scales = _empty(m, dtype=_float32, device=dev)
    if m:
        # (_quantize, without the calls)
        desc = _pack_rows(x.data_ptr(), 0, 0, 0, 0, 0, codes.data_ptr(), scales.data_ptr(), 0, 0, current_stream_ptr(dev), 0.0, stride,
                          0, 0, 0, pitch, m, k, code, 0, 0, 0)
        K.call(K.ext().quantize, dev, desc, "glowq_w8a8_quantize")
    return TokenCodes(codes if pitch == k else codes[:, :k], scales, None, _TYPES[code])


def quantize_channels(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a weight [out_features, in_features], a scale for every output channel.  The codes are a view of rows that lie a
    multiple of 16 bytes apart.  On the CPU the same codes with torch expressions, so that a model can be converted there."""
    rows, scales = channel_rows(weight)
    return rows[:, :weight.shape[1]], scales


def channel_rows(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes in whole rows [out_features, in_features rounded up to 16] with zeros at the end, scales)"""
    if weight.dim() != 2 or weight.dtype not in K.DTYPES:
        raise RuntimeError("weight must be [out_features, in_features] in fp16, bf16 or fp32")
    weight = weight.detach()
    oc, ic = weight.shape
    rows = torch.zeros((oc, _pitch(ic)), dtype=torch.int8, device=weight.device)
    codes = rows[:, :ic]
    scales = torch.empty(oc, dtype=torch.float32, device=weight.device)
    if oc == 0:
        return rows, scales
    if weight.is_cuda:
        _quantize(_matrix(weight, "weight")[0], codes, scales, True)
        return rows, scales
    top = weight.float().abs().amax(dim=1)
    torch.div(top, torch.full_like(top, 127.0), out=scales)
    bad = ~torch.isfinite(top)
    scales[bad] = float("nan")
    q = torch.round(weight.double() / scales.double()[:, None]).clamp_(-127, 127)
    codes.copy_(torch.where((scales > 0)[:, None], q, torch.zeros_like(q)))
    return rows, scales


def norm_quantize_tokens(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                         residual: Optional[torch.Tensor] = None, norm: str = "rms") -> Tuple[TokenCodes, torch.Tensor]:
    """Residual add, norm and codes in one launch: (codes of norm(h), h) with h = x + residual (h is ``x`` itself without a residual).

    ``norm``: "layer" (``nn.LayerNorm``'s arithmetic, ``bias`` may be None) or "rms" (the models' RMSNorm modules: fp32 statistics, the
    normalised value rounded to the input's type before the weight).  All tensors have one type; h and the normalised values are
    rounded to it, so the codes are those of the separate steps.  h has the gradients of the sum that it is (and no forward-mode
    derivatives: a dual tensor raises); the codes have none, as the linears that take them."""
    kind = _NORMS.get(norm)
    if kind is None:
        raise ValueError(f'norm must be "layer" or "rms", got {norm!r}')
    if kind == K.NORM_RMS and bias is not None:
        raise ValueError("RMSNorm has no bias")
    x2, m, k, stride, dev, code = _matrix(x, "x")
    dtype = _TYPES[code]
    check_norm(k, dtype, dev, weight, bias, eps)
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != dtype or residual.device != dev:
            raise RuntimeError("residual must have x's shape, type and device")
        if forward_ad._current_level >= 0 or ((x.requires_grad or residual.requires_grad) and torch.is_grad_enabled()):
            hidden, codes, scales = _NormCodes.apply(x, residual, weight, bias, eps, kind)
            return TokenCodes(codes, scales, None, dtype), hidden
    codes, scales, hidden = _norm_codes(x, (x2, m, k, stride, dev, code), weight, bias, eps, residual, kind)
    return TokenCodes(codes, scales, None, dtype), hidden


class _NormCodes(torch.autograd.Function):
    """The sum of a call with a residual, with its gradients."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, kind):
        codes, scales, hidden = _norm_codes(x, _matrix(x, "x"), weight, bias, eps, residual, kind)
        ctx.mark_non_differentiable(codes, scales)
        return hidden, codes, scales

    @staticmethod
    def backward(ctx, dh, *_):
        return dh, dh, None, None, None, None


def _norm_codes(x, matrix, weight, bias, eps, residual, kind):
    x2, m, k, stride, dev, code = matrix
    res_at = res_stride = hid_at = 0
    hidden = x
    if residual is not None:
        res, _, _, res_stride, _, _ = _matrix(residual, "residual")
        # (of x's shape from the start: autograd takes no change in place of a view that a function returns)
        hidden = _empty(m, k, dtype=_TYPES[code], device=dev) if x2 is x else _empty(*x.shape, dtype=_TYPES[code], device=dev)
        res_at, hid_at = res.data_ptr(), hidden.data_ptr()
    codes = _new_codes(m, k, dev)
    scales = _empty(m, dtype=_float32, device=dev)
    if m:
        weight = weight.contiguous()
        b_at = 0
        if bias is not None:
            bias = bias.contiguous()
            b_at = bias.data_ptr()
        desc = _pack_rows(x2.data_ptr(), res_at, weight.data_ptr(), b_at, hid_at, 0, codes.data_ptr(), scales.data_ptr(), 0, 0,
                          current_stream_ptr(dev), eps, stride, res_stride, k, 0, (k + 15) & ~15, m, k, code, kind, 0, 0)
        K.call(K.ext().quantize, dev, desc, "glowq_w8a8_quantize")
    return codes, scales, hidden


def check_norm(k: int, dtype: torch.dtype, dev: torch.device, weight: torch.Tensor, bias: Optional[torch.Tensor], eps: float) -> None:
    shape = (k,)
    if weight is None or weight.shape != shape or weight.dtype != dtype or weight.device != dev:
        raise RuntimeError(f"weight must be [{shape[0]}] of x's type on x's device")
    if bias is not None and (bias.shape != shape or bias.dtype != dtype or bias.device != dev):
        raise RuntimeError(f"bias must be [{shape[0]}] of x's type on x's device")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")


def _factor(t: torch.Tensor, name: str, rows: int, cols: Optional[int], device):
    """(``_place`` of a factor)"""
    shape = t.shape
    if t.dtype != _float16 or t.device != device or len(shape) != 2 or shape[0] != rows or (cols is not None and shape[1] != cols):
        raise RuntimeError(f"{name} must be fp16 [{rows}, {'rank' if cols is None else cols}] on {device}, got {t.dtype} {tuple(shape)}")
    return _place(t.detach() if t.requires_grad else t, 2, rows, shape[1])


def right_factor(x: torch.Tensor, R: torch.Tensor, constant: bool = True) -> torch.Tensor:
    """r = x R^T, fp16 [tokens, rank], for corrected linears that share a right factor (``TokenCodes.r``).  ``x`` is taken in fp16, as the
    W4A16 path takes it; sums in fp32.  ``constant``: as for ``w8a8_linear``."""
    x, m, k, _, dev, code = _matrix(x.detach(), "x")
    if R.dim() != 2 or not 0 < R.shape[0] <= K.MAX_RANK:
        raise RuntimeError(f"R must be [rank, in_features] with a rank of 1 to {K.MAX_RANK}")
    if m > K.MAX_TOKENS:
        raise RuntimeError(f"at most {K.MAX_TOKENS} tokens")
    R, R_at, R_stride, fresh = _factor(R, "R", R.shape[0], k, dev)
    rank = R.shape[0]
    if not constant:
        fresh = K.FRESH
    pitch = (rank + 7) & ~7
    r = _empty(m, pitch, dtype=_float16, device=dev)
    if m:
        x, x_at, x_stride, _ = _place(x if code == K.F16 else x.to(_float16), 2, m, k)
        desc = _pack_linear(0, 0, 0, 0, 0, 0, x_at, R_at, r.data_ptr(), 0, 0, current_stream_ptr(dev), 0, 0, 0, x_stride, R_stride, pitch, 0,
                            0, m, k, 0, rank, 0, 0, K.R_COMPUTE | fresh, 0.0, 0)
        K.call(K.ext().right_factor, dev, desc, "glowq_w8a8_right_factor")
    return r if pitch == rank else r[:, :rank]


def w8a8_linear(x: Union[torch.Tensor, TokenCodes], weight: torch.Tensor, weight_scales: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, out_dtype: Optional[torch.dtype] = None, L: Optional[torch.Tensor] = None,
                R: Optional[torch.Tensor] = None, alpha: float = 1.0, constant: bool = True) -> torch.Tensor:
    """One 8-bit linear.  ``x``: activations [..., in_features] (their codes are made here), or ``TokenCodes`` -> [tokens, out_features].
    ``weight`` int8 [out_features, in_features] and ``weight_scales`` fp32 [out_features] as ``quantize_channels`` gives them, ``bias`` fp32
    [out_features].  ``out_dtype``: fp16, bf16 or fp32; by default the activations' type, that which codes
    were made of (fp16 where ``TokenCodes.dtype`` is None).  ``L`` fp16 [out_features, rank]:
    the linear is corrected by alpha * r L^T, with r = x R^T (``R`` fp16 [rank, in_features]) or the codes' ``r``.  r is made of x in fp16 and
    held in fp16, as the W4A16 path has it: of a bf16 or fp32 token whose values or r pass 65504 the corrected outputs are not finite.

    ``constant``: ``weight``, ``L`` and ``R`` may be read before what is in front of this call on the stream is complete.  Pass False where
    the operation right in front made one of them (a merge, a cast, a copy; what ``quantize_channels`` gives may be used at once)."""
    x2 = lead = r = None
    if isinstance(x, TokenCodes):
        codes, scales, r, made_of = x
        shape, dev = codes.shape, codes.device
        if not codes.is_cuda or codes.dtype != _int8 or len(shape) != 2:
            raise RuntimeError("codes must be int8 [tokens, in_features] on a CUDA device")
        m, k = shape
        if m.__class__ is not int:
            K.refuse_trace()
        if scales.dtype != _float32 or scales.shape != (m,) or scales.device != dev:
            raise RuntimeError(f"scales must be fp32 [{m}] on {dev}")
        if R is not None:
            raise RuntimeError("codes have no right factor's product to be made from: pass TokenCodes.r (right_factor(x, R))")
        if out_dtype is None:
            out_dtype = made_of or _float16
    else:
        x2, m, k, x_stride, dev, x_code = _matrix(x, "x")
        if x2 is not x and x.dim() != 2:
            lead = x.shape[:-1]
        if (L is None) != (R is None):
            raise RuntimeError("a correction needs L and R")
        if out_dtype is None:
            out_dtype = _TYPES[x_code]
    out_code = K.DTYPES.get(out_dtype)
    if out_code is None:
        raise RuntimeError(f"out_dtype must be fp16, bf16 or fp32, got {out_dtype}")
    shape = weight.shape
    if weight.dtype != _int8 or len(shape) != 2 or weight.device != dev:
        raise RuntimeError(f"weight must be int8 [out_features, in_features] on {dev}")
    oc, ic = shape
    if ic != k:
        raise ValueError(f"Input dim mismatch: got {k}, expected {ic}")
    if not 0 < k <= K.MAX_EXACT_K:
        raise RuntimeError(f"in_features must be 1 to {K.MAX_EXACT_K} (sums are exact in 32 bits)")
    if weight_scales.dtype != _float32 or weight_scales.shape != (oc,) or weight_scales.device != dev:
        raise RuntimeError(f"weight_scales must be fp32 [{oc}] on {dev}")
    if bias is not None and (bias.dtype != _float32 or bias.shape != (oc,) or bias.device != dev):
        raise RuntimeError(f"bias must be fp32 [{oc}] on {dev}")
    if m > K.MAX_TOKENS:
        raise RuntimeError(f"at most {K.MAX_TOKENS} tokens")
    out = _empty(m, oc, dtype=out_dtype, device=dev)
    if m and oc:
        weight, w_at, w_stride, fresh = _place(weight, 1, oc, ic)
        if not constant:
            fresh = K.FRESH
        weight_scales = weight_scales.contiguous()
        b_at = 0
        if bias is not None:
            bias = bias.contiguous()
            b_at = bias.data_ptr()
        rank = mode = L_at = L_stride = R_at = R_stride = r_at = r_stride = rx_at = rx_stride = x_at = 0
        if L is not None:
            rank = L.shape[1] if L.dim() == 2 else 0
            L, L_at, L_stride, copied = _factor(L, "L", oc, None, dev)
            fresh |= copied
            if not 0 < rank <= K.MAX_RANK:
                raise RuntimeError(f"the rank must be 1 to {K.MAX_RANK}")
            if x2 is None:
                if r is None:
                    raise RuntimeError("a corrected linear of codes needs TokenCodes.r (right_factor(x, R))")
                r, r_at, r_stride, _ = _factor(r, "r", m, rank, dev)
                mode = K.R_LOAD
            else:
                R, R_at, R_stride, copied = _factor(R, "R", rank, k, dev)
                fresh |= copied
                rx, rx_at, rx_stride, _ = _place((x2 if x_code == K.F16 else x2.to(_float16)).detach(), 2, m, k)
                mode = K.R_COMPUTE
        if x2 is None:
            codes, code_at, code_stride, _ = _place(codes, 1, m, k)
            x_stride = x_code = 0
            scales = scales.contiguous()
            scale_at = scales.data_ptr()
        else:
            # codes, scales and r of this call: one piece of memory
            x_at = x2.data_ptr()
            code_stride, r_stride = (k + 15) & ~15, (rank + 7) & ~7
            scale_off = m * code_stride
            r_off = scale_off + (4 * m + 15 & ~15)
            room = _empty(r_off + 2 * m * r_stride, dtype=_int8, device=dev)
            code_at = room.data_ptr()
            scale_at, r_at = code_at + scale_off, code_at + r_off
        desc = _pack_linear(x_at, code_at, scale_at, w_at, weight_scales.data_ptr(), b_at, rx_at, R_at, r_at, L_at, out.data_ptr(),
                            current_stream_ptr(dev), x_stride, code_stride, w_stride, rx_stride, R_stride, r_stride, L_stride, oc, m, k, oc,
                            rank, x_code, out_code, mode | fresh, alpha, 0)
        K.call(K.ext().linear, dev, desc, "glowq_w8a8_linear")
    return out if lead is None else out.reshape(*lead, oc)


def read_status(device: Optional[torch.device] = None) -> None:
    """Raises if a bounded wait of the 8-bit kernels has run out on the device since the last call.  Synchronises the current stream."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        K.ext().check(K.ext().lib.glowq_w8a8_read_status(torch.cuda.current_stream().cuda_stream), "device status")
