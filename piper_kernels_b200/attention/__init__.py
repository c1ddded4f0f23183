"""Fused attention operators: the quantized ones (same names as ``piper_kernels.attention``), and 16-bit
attention over a sliding window and over a paged cache."""

from .cached import cache_attention
from .piper import piper_attention
from .sage2pp import sage_attention_2pp
from .window import window_attention

__all__ = ["cache_attention", "piper_attention", "sage_attention_2pp", "window_attention"]
