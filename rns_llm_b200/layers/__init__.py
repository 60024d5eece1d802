from .rns_attention import QuantizedCacheAttention, QuantizedDecoderCache
from .rns_linear import RNSLinear
from .rns_qkv import (
    CachedRNSQKV,
    InstalledQKVFusion,
    RNSQKVProjection,
    install_opt_qkv_fusion,
)

__all__ = [
    "RNSLinear",
    "RNSQKVProjection",
    "CachedRNSQKV",
    "InstalledQKVFusion",
    "QuantizedCacheAttention",
    "QuantizedDecoderCache",
    "install_opt_qkv_fusion",
]
