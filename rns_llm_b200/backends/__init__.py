from .cuda_backend import (
    AdaptiveMetadata,
    CudaRNSBackend,
    PreparedAdaptiveRNSWeight,
    PreparedRNSWeight,
    RNSRequestBatchWorkspace,
    RNSWorkspace,
    cuda_extension_available,
)
from .kv_cache import QuantizedKVCache

__all__ = [
    "AdaptiveMetadata",
    "CudaRNSBackend",
    "PreparedRNSWeight",
    "PreparedAdaptiveRNSWeight",
    "QuantizedKVCache",
    "RNSWorkspace",
    "RNSRequestBatchWorkspace",
    "cuda_extension_available",
]
