"""8-bit linears beside ``cuda_w4a16``: token codes, products of int8 codes with a scale for each token and channel (with the low-rank
correction, if there is one), and the norms in front of them.  The reference project has no 8-bit path; names and manners follow
``cuda_w4a16``.

    tokens, hidden = norm_quantize_tokens(x, ln.weight, ln.bias, residual=residual, norm="layer")
    q, k, v = q_proj(tokens), k_proj(tokens), v_proj(tokens)           # CudaW8A8Linear modules
"""
from .functional import (TokenCodes, norm_quantize_tokens, quantize_channels, quantize_tokens, read_status, right_factor, w8a8_linear)
from .norms import CudaLayerNorm, layer_norm
from .linear import CudaW8A8Linear, convert_to_cuda_w8a8

__all__ = ["TokenCodes", "quantize_tokens", "norm_quantize_tokens", "quantize_channels", "right_factor", "w8a8_linear", "layer_norm",
           "CudaLayerNorm", "CudaW8A8Linear", "convert_to_cuda_w8a8", "read_status"]
