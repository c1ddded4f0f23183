"""piper_kernels_b200 — B200-native (sm_100a) fused quantized attention.

Drop-in for the attention operators of Boffee/piper-kernels:
``piper_attention`` and ``sage_attention_2pp`` keep the reference's signatures and
validation and dispatch through ``torch.library`` operators into ``libpiper_b200.so``.  Beside
them, for serving: ``window_attention`` (prompts over a sliding window with sinks) and
``cache_attention`` (tokens and drafted trees over a :class:`PageCache`).
"""

from .attention import cache_attention, piper_attention, sage_attention_2pp, window_attention
from .cache import PageCache

__all__ = ["PageCache", "cache_attention", "piper_attention", "sage_attention_2pp", "window_attention"]
__version__ = "0.1.0"
