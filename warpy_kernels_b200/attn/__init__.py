from .bwd_api import attn_bwd, autotune_attn_bwd, make_attn_bwd
from .fwd_api import attn_fwd, autotune_attn_fwd, make_attn_fwd
from .prefix_api import attn_fwd_shared_prefix

__all__ = [
    "attn_bwd",
    "attn_fwd",
    "attn_fwd_shared_prefix",
    "autotune_attn_bwd",
    "autotune_attn_fwd",
    "make_attn_bwd",
    "make_attn_fwd",
]
