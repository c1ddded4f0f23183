"""Public ``window_attention``: causal attention over a sliding window, with sink tokens."""

from __future__ import annotations

import torch

from ._validation import check_lengths, check_rows, check_scale, check_window

_OP = "Window Attention"


def window_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    *,
    window: int,
    sinks: int = 0,
    scale: float | None = None,
    lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of a prompt, or of a chunk at its end, over the keys near each token and the first ones.

    ``query`` is ``[batch, heads, q_len, head_dim]``, ``key`` and ``value`` ``[batch, kv_heads, kv_len,
    head_dim]``; FP16/BF16, contiguous head dimension of 64 or 128, any other strides; ``heads`` is a
    multiple of ``kv_heads`` and query head ``h`` reads key head ``h // (heads // kv_heads)``.  Query row
    ``i`` stands at position ``p = i + kv_len - q_len`` and sees key ``j`` when ``j <= p`` and either
    ``p - j < window`` or ``j < sinks``.  ``lengths`` (int32 ``[batch]``) says how many keys of each batch
    element exist (a right-padded batch); keys behind them are never looked at.  Rows that see no key and
    rows at or behind their length are zero.  ``scale`` defaults to ``head_dim**-0.5``.  Can be captured in a CUDA
    graph once it has run on the device outside of one.  Inference only.
    """
    for name, tensor in (("query", query), ("key", key), ("value", value)):
        check_rows(_OP, name, tensor)
    if query.device != key.device or query.device != value.device:
        raise ValueError(f"{_OP} query, key, and value must share a device, got {query.device}/{key.device}/{value.device}")
    if query.dtype is not key.dtype or query.dtype is not value.dtype:
        raise ValueError(f"{_OP} query, key, and value must share a dtype, got {query.dtype}/{key.dtype}/{value.dtype}")
    if key.shape != value.shape:
        raise ValueError(f"{_OP} key and value shapes must match, got {tuple(key.shape)}/{tuple(value.shape)}")
    if query.shape[0] != key.shape[0]:
        raise ValueError(f"{_OP} requires equal batch dimensions, got {query.shape[0]}/{key.shape[0]}")
    if 0 in query.shape[:3] or 0 in key.shape[:3]:
        raise ValueError(f"{_OP} does not accept empty query or key sequences")
    if query.shape[1] % key.shape[1]:
        raise ValueError(f"{_OP} query heads must be a multiple of the key heads, got {query.shape[1]}/{key.shape[1]}")
    if query.shape[3] != key.shape[3]:
        raise ValueError(f"{_OP} head dimensions must match, got {query.shape[3]}/{key.shape[3]}")
    window, sinks = check_window(_OP, window, sinks)
    check_lengths(_OP, "lengths", lengths, query.shape[0], query.device)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        raise RuntimeError(f"{_OP} is an inference-only operator and does not support autograd")
    converted_scale = check_scale(_OP, scale, query.shape[3])
    from .. import _ops

    return _ops.window_attention_op(query, key, value, lengths, window, sinks, converted_scale)

