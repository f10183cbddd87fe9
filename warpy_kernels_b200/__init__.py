"""B200 (sm_100a) implementation of the warpy-kernels hot path behind the reference's Python surface."""

from .arch import device_arch, supports
from .attn import attn_fwd_shared_prefix
from .interface import attn_bwd, attn_fwd, autotune_gemm, gemm, make_gemm
from .quant import quantize_mx
from .rotary import qk_norm_rope, qk_norm_rope_bwd, rope

__all__ = [
    "attn_bwd",
    "attn_fwd",
    "attn_fwd_shared_prefix",
    "autotune_gemm",
    "device_arch",
    "gemm",
    "make_gemm",
    "qk_norm_rope",
    "qk_norm_rope_bwd",
    "quantize_mx",
    "rope",
    "supports",
]
