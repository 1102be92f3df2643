"""Layer norm with its gradients, and with the residual add in front of it.

    h = x + residual (rounded to the type of x),  y = (h - mean) * rstd * weight + bias

Statistics are taken in 64 bits and held in fp32, sums of gradients in fp32 in an order that the sizes (and the
rows' places within 16 bytes) fix; each output is rounded once."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from ..cuda_w4a16.kernels import current_stream_ptr
from . import kernels as K
from .functional import _TYPES, _empty, _float32, _matrix, _pack_rows, _rows, check_norm


def _forward(x, matrix, residual, weight, bias, eps, statistics: bool):
    """(``matrix``: what ``_matrix`` gave of x.)  Outputs have x's shape from the start: autograd takes no change in place of a view that a
    function returns."""
    x2, m, k, stride, dev, code = matrix
    dtype, shape = _TYPES[code], (m, k) if x2 is x else x.shape
    y = _empty(*shape, dtype=dtype, device=dev)
    hidden = mean = rstd = None
    res_at = res_stride = hid_at = mean_at = rstd_at = 0
    if residual is not None:
        res, _, _, res_stride, _, _ = _matrix(residual, "residual")
        hidden = _empty(*shape, dtype=dtype, device=dev)
        res_at, hid_at = res.data_ptr(), hidden.data_ptr()
    if statistics:
        mean, rstd = _empty(m, dtype=_float32, device=dev), _empty(m, dtype=_float32, device=dev)
        mean_at, rstd_at = mean.data_ptr(), rstd.data_ptr()
    if m:
        weight, bias = weight.contiguous(), bias.contiguous() if bias is not None else None
        desc = _pack_rows(x2.data_ptr(), res_at, weight.data_ptr(), bias.data_ptr() if bias is not None else 0, hid_at, y.data_ptr(), 0, 0,
                          mean_at, rstd_at, current_stream_ptr(dev), eps, stride, res_stride, k, k, 0, m, k, code,
                          K.NORM_LAYER, 0, 0)
        K.call(K.ext().layer_norm_forward, dev, desc, "glowq_layer_norm_forward")
    return y, hidden, mean, rstd


def _backward(h, dy, dh, weight, mean, rstd, need_dx: bool, need_dw: bool):
    m, k = h.shape
    dev = h.device
    dx = _empty(m, k, dtype=h.dtype, device=dev) if need_dx else None
    dw, db = (_empty(k, dtype=h.dtype, device=dev), _empty(k, dtype=h.dtype, device=dev)) if need_dw else (None, None)
    need = K.ext().lib.glowq_layer_norm_workspace_bytes(m, k)
    room = torch.empty(need, dtype=torch.uint8, device=dev)
    if not need_dx:
        dh = None
    desc = K.pack_grad.pack(h.data_ptr(), dy.data_ptr(), dh.data_ptr() if dh is not None else 0, weight.data_ptr(), mean.data_ptr(),
                            rstd.data_ptr(), dx.data_ptr() if need_dx else 0, dw.data_ptr() if need_dw else 0,
                            db.data_ptr() if need_dw else 0, room.data_ptr(), need, current_stream_ptr(dev), h.stride()[0], dy.stride()[0],
                            dh.stride()[0] if dh is not None else 0, k, m, k, K.DTYPES[h.dtype], 0)
    K.call(K.ext().layer_norm_backward, dev, desc, "glowq_layer_norm_backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        ctx.set_materialize_grads(False)
        y, hidden, mean, rstd = _forward(x, _matrix(x, "x"), residual, weight, bias, eps, True)
        if residual is None:
            ctx.save_for_backward(x, weight, mean, rstd)
            return y
        ctx.save_for_backward(hidden, weight, mean, rstd)
        return y, hidden

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        need_dx, need_dw = need_x or need_res, need_w or need_b
        shape = h.shape
        if dy is None or h.numel() == 0:
            # the normalised rows were not used (or there are none): only the sum's own gradient is left
            dx = dh if dh is not None else (torch.zeros_like(h) if need_dx else None)
            dw = torch.zeros_like(weight) if need_dw else None
            db = torch.zeros_like(weight) if need_dw else None
        else:
            h2, dy2 = _rows(h, "h"), _rows(dy, "grad")
            dh2 = _rows(dh, "grad") if dh is not None else None
            dx, dw, db = _backward(h2, dy2, dh2, weight.contiguous(), mean, rstd, need_dx, need_dw)
            dx = dx.reshape(shape) if dx is not None else None
        return dx if need_x else None, dw if need_w else None, db if need_b else None, dx if need_res else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Layer norm over the last dimension (fp16, bf16 or fp32; ``weight`` and ``bias`` [columns] of the same type): y, or with ``residual``
    (y, h) for h = x + residual.  Differentiable once in all tensors; the gradient of h as an output joins that of y.  There are no
    forward-mode derivatives: a dual tensor raises."""
    matrix = _matrix(x, "x")
    _, _, k, _, dev, code = matrix
    dtype = _TYPES[code]
    check_norm(k, dtype, dev, weight, bias, eps)
    if residual is not None and (residual.shape != x.shape or residual.dtype != dtype or residual.device != dev):
        raise RuntimeError("residual must have x's shape, type and device")
    # (under a level of forward-mode derivatives autograd looks at the tensors, and refuses those with a tangent)
    if forward_ad._current_level >= 0 or (
            torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                         or (residual is not None and residual.requires_grad))):
        return _LayerNorm.apply(x, weight, bias, residual, float(eps))
    y, hidden, _, _ = _forward(x, matrix, residual, weight, bias, eps, False)
    return y if residual is None else (y, hidden)


class CudaLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension on the kernels of this package.  ``forward(x, residual)`` returns (y, x + residual).

    Under autocast rows and parameters may be of different types, and y is then fp32 as ``nn.LayerNorm``'s there; outside of it they are
    refused, as ``nn.LayerNorm`` refuses them on this device."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1 or self.weight is None:
            raise ValueError("CudaLayerNorm normalises the last dimension and has a weight")

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        weight, bias = self.weight, self.bias
        if x.dtype != weight.dtype and torch.is_autocast_enabled("cuda"):
            if residual is not None:
                h = x + residual
                return self.forward(h), h
            x, weight, bias = x.float(), weight.float(), bias.float() if bias is not None else None
        return layer_norm(x, weight, bias, self.eps, residual)

    @classmethod
    def from_float(cls, norm: nn.LayerNorm) -> "CudaLayerNorm":
        """The module around the same parameters."""
        if len(norm.normalized_shape) != 1 or norm.weight is None:
            raise ValueError("CudaLayerNorm normalises the last dimension and has a weight")
        mod = cls(norm.normalized_shape, norm.eps, bias=norm.bias is not None, device="meta")
        mod.weight, mod.bias = norm.weight, norm.bias
        mod.train(norm.training)
        return mod
