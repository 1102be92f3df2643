"""glowq_b200: B200 (sm_100a) implementation of GlowQ's corrected W4A16 linear behind GlowQ's own Python surface, and 8-bit linears and
norms beside it (``cuda_w8a8``)."""
from .cuda_w4a16 import CudaW4A16Linear, convert_to_cuda_w4a16, load_w4a16_extension
from .correction import (AddSVDCorrection, MiniGroupCache, clear_group_cache, patch_svd_correction_wrappers,
                         patch_svd_correction_wrappers_cumulative)
from .cuda_w8a8 import (CudaLayerNorm, CudaW8A8Linear, TokenCodes, convert_to_cuda_w8a8, layer_norm, norm_quantize_tokens,
                        quantize_channels, quantize_tokens, right_factor, w8a8_linear)
from .artifacts import load_packed, save_packed

__all__ = ["load_w4a16_extension", "CudaW4A16Linear", "convert_to_cuda_w4a16", "AddSVDCorrection", "MiniGroupCache",
           "patch_svd_correction_wrappers", "patch_svd_correction_wrappers_cumulative", "clear_group_cache",
           "save_packed", "load_packed", "CudaW8A8Linear", "convert_to_cuda_w8a8", "CudaLayerNorm", "TokenCodes", "quantize_tokens",
           "norm_quantize_tokens", "quantize_channels", "right_factor", "w8a8_linear", "layer_norm"]
