"""``CudaW8A8Linear``: an ``nn.Linear`` in 8 bits (a scale for each output channel, codes of its input made in the call), and the
conversion pass ``convert_to_cuda_w8a8``; the counterparts of ``CudaW4A16Linear`` and ``convert_to_cuda_w4a16``."""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn as nn

from .functional import TokenCodes, _pitch, channel_rows, quantize_tokens, right_factor, w8a8_linear
from .norms import CudaLayerNorm


class CudaW8A8Linear(nn.Module):
    """Buffers: ``qweight_i8`` int8 [out_features, in_features rounded up to 16], ``scales_f32`` [out_features]; ``bias`` fp32."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False, out_dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.in_features, self.out_features, self.out_dtype = int(in_features), int(out_features), out_dtype
        self.register_buffer("qweight_i8", torch.zeros(self.out_features, _pitch(self.in_features), dtype=torch.int8))
        self.register_buffer("scales_f32", torch.zeros(self.out_features, dtype=torch.float32))
        self.bias = nn.Parameter(torch.zeros(self.out_features, dtype=torch.float32), requires_grad=False) if bias else None

    def _apply(self, fn, recurse: bool = True):
        """Moves with the model; scales and bias stay fp32 whatever type the model is cast to."""
        scales, bias = self.scales_f32, self.bias.data if self.bias is not None else None   # (a parameter is cast in place)
        super()._apply(fn, recurse)
        if self.scales_f32.dtype != torch.float32:
            self.scales_f32 = scales.to(self.scales_f32.device)
        if bias is not None and self.bias.dtype != torch.float32:
            self.bias.data = bias.to(self.bias.device)
        return self

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

    @property
    def weight_codes(self) -> torch.Tensor:
        w = self.qweight_i8
        return w if w.shape[1] == self.in_features else w[:, :self.in_features]

    def dequantized_weight(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight that the codes stand for, [out_features, in_features]: what is left of the original, ``W - dequantized_weight()``, is what
        a correction's factors are fitted to."""
        return (self.weight_codes.float() * self.scales_f32[:, None]).to(dtype)

    def launch(self, x: Union[torch.Tensor, TokenCodes], *, L=None, R=None, alpha: float = 1.0) -> torch.Tensor:
        """The linear, optionally with its low-rank correction folded in."""
        return w8a8_linear(x, self.weight_codes, self.scales_f32, self.bias, out_dtype=self.out_dtype, L=L, R=R, alpha=alpha)

    def forward(self, x: Union[torch.Tensor, TokenCodes]) -> torch.Tensor:
        return self.launch(x)

    def tokens(self, x: torch.Tensor, R: Optional[torch.Tensor] = None) -> TokenCodes:
        """``x`` as linears that share it take it: its codes, and r = x R^T for the corrected ones."""
        t = quantize_tokens(x)
        return t if R is None else t._replace(r=right_factor(x, R))

    @classmethod
    def from_float(cls, linear_layer: nn.Linear, out_dtype: Optional[torch.dtype] = None) -> "CudaW8A8Linear":
        weight = linear_layer.weight.data
        rows, scales = channel_rows(weight)
        with torch.device("meta"):
            mod = cls(linear_layer.in_features, linear_layer.out_features, bias=linear_layer.bias is not None, out_dtype=out_dtype)
        mod.qweight_i8 = rows
        mod.scales_f32 = scales
        if linear_layer.bias is not None:
            mod.bias = nn.Parameter(linear_layer.bias.data.to(torch.float32).clone(), requires_grad=False)
        return mod


def convert_to_cuda_w8a8(model: nn.Module, layer_norms: bool = False) -> nn.Module:
    """Replace every ``nn.Linear`` whose qualified name does not contain "lm_head" by a ``CudaW8A8Linear``, and with ``layer_norms`` every
    ``nn.LayerNorm`` over the last dimension by a ``CudaLayerNorm`` around the same parameters.  A layer whose conversion raises keeps its
    original module; the failures are collected in ``model._w8a8_conversion_errors`` (as ``convert_to_cuda_w4a16`` does)."""
    errors = {}
    for name, mod in list(model.named_modules()):
        if isinstance(mod, nn.Linear) and "lm_head" not in name:
            make = CudaW8A8Linear.from_float
        elif layer_norms and isinstance(mod, nn.LayerNorm) and not isinstance(mod, CudaLayerNorm):
            make = CudaLayerNorm.from_float
        else:
            continue
        parent = model
        *path, leaf = name.split(".")
        for part in path:
            parent = getattr(parent, part)
        try:
            setattr(parent, leaf, make(mod))
        except Exception as exc:  # noqa: BLE001 - as the 4-bit pass: the others are converted
            errors[name] = repr(exc)
    try:
        model._w8a8_conversion_errors = errors
    except Exception:  # noqa: BLE001
        pass
    if torch.cuda.is_available():
        torch.cuda.empty_cache()
    return model


__all__ = ["CudaW8A8Linear", "convert_to_cuda_w8a8"]
