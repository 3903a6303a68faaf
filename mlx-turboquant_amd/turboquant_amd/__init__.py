"""TurboQuant KV-cache compression and compressed-cache attention for AMD
MI355X (gfx950), with the public API of mlx-turboquant
(mlx_turboquant/__init__.py:45-59): apply_turboquant, enable_turboquant,
TurboQuantKVCache, TurboQuantMSE, TurboQuantProd; and, with no counterpart there,
an 8-bit KV cache (KV8Cache, KV8Batch and the kv8_* functions below them) and
attention with a sliding window (window_attention).

All compute runs in the hand-written HIP kernels of ``libtq_hip.so``; there is
no CPU fallback.
"""

__version__ = "0.1.0"

from .cache import TurboQuantKVCache
from .kv8 import KV8Batch, KV8Cache, KV8Store, kv8_attention, kv8_read, kv8_write
from .patch import apply_turboquant, detect_outlier_layers, enable_turboquant
from .quantizer import QuantizedTensor, TurboQuantMSE, TurboQuantProd
from .window import window_attention

__all__ = [
    "__version__",
    "apply_turboquant",
    "enable_turboquant",
    "TurboQuantKVCache",
    "TurboQuantMSE",
    "TurboQuantProd",
    "QuantizedTensor",
    "detect_outlier_layers",
    "KV8Store",
    "KV8Cache",
    "KV8Batch",
    "kv8_write",
    "kv8_read",
    "kv8_attention",
    "window_attention",
]
