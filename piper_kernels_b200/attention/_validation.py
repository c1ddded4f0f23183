"""Input validation shared by both public functions.

Same checks, in the same order and with the same message fragments, as the reference's
``_validate_inputs`` (src/piper_kernels/attention/piper/dispatch.py:22-89 and
src/piper_kernels/attention/sage2pp/dispatch.py:22-89).
"""

from __future__ import annotations

import math

import torch

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16)
SUPPORTED_HEAD_DIMS = (64, 128)


def validate_inputs(op: str, query, key, value, scale, is_causal) -> float:
    tensors = {"query": query, "key": key, "value": value}
    for name, tensor in tensors.items():
        if tensor.ndim != 4:
            raise ValueError(
                f"{op} {name} must have shape [batch, heads, sequence, head_dim], got {tuple(tensor.shape)}")
        if tensor.dtype not in SUPPORTED_DTYPES:
            raise ValueError(f"{op} {name} must use float16 or bfloat16, got {tensor.dtype}")
        if tensor.layout is not torch.strided:
            raise ValueError(f"{op} {name} must use strided layout")
        if tensor.stride(-1) != 1:
            raise ValueError(f"{op} {name}'s head dimension must be contiguous")
    if query.device != key.device or query.device != value.device:
        raise ValueError(
            f"{op} query, key, and value must share a device, got {query.device}/{key.device}/{value.device}")
    if query.dtype is not key.dtype or query.dtype is not value.dtype:
        raise ValueError(
            f"{op} query, key, and value must share a dtype, got {query.dtype}/{key.dtype}/{value.dtype}")
    if query.shape[:2] != key.shape[:2] or key.shape[:2] != value.shape[:2]:
        raise ValueError(
            f"{op} currently requires equal batch and head dimensions, got "
            f"{query.shape[:2]}/{key.shape[:2]}/{value.shape[:2]}")
    if key.shape[2] != value.shape[2]:
        raise ValueError(f"{op} key/value lengths must match, got {key.shape[2]}/{value.shape[2]}")
    if query.shape[3] != key.shape[3] or key.shape[3] != value.shape[3]:
        raise ValueError(
            f"{op} head dimensions must match, got {query.shape[3]}/{key.shape[3]}/{value.shape[3]}")
    if query.shape[3] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"{op} currently supports head dimensions 64 and 128, got {query.shape[3]}")
    if query.shape[2] == 0 or key.shape[2] == 0:
        raise ValueError(f"{op} does not accept empty query or key sequences")
    if is_causal and query.shape[2] != key.shape[2]:
        raise ValueError(
            f"Causal {op} currently requires equal query and key lengths, got "
            f"{query.shape[2]}/{key.shape[2]}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors.values()):
        raise RuntimeError(f"{op} is an inference-only operator and does not support autograd")
    converted = query.shape[-1] ** -0.5 if scale is None else float(scale)
    if not math.isfinite(converted) or converted <= 0:
        raise ValueError(f"{op} scale must be finite and positive, got {scale}")
    return converted


# Checks of the 16-bit operators (window_attention, cache_attention, PageCache), which have no counterpart
# in the reference; same fragments of messages.


def check_rows(op: str, name: str, tensor, ndim: int = 4) -> None:
    if tensor.ndim != ndim:
        shape = "[layers, batch, heads, sequence, head_dim]" if ndim == 5 else "[batch, heads, sequence, head_dim]"
        raise ValueError(f"{op} {name} must have shape {shape}, got {tuple(tensor.shape)}")
    if tensor.dtype not in SUPPORTED_DTYPES:
        raise ValueError(f"{op} {name} must use float16 or bfloat16, got {tensor.dtype}")
    if tensor.layout is not torch.strided:
        raise ValueError(f"{op} {name} must use strided layout")
    if tensor.shape[-1] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"{op} currently supports head dimensions 64 and 128, got {tensor.shape[-1]}")
    if tensor.stride(-1) != 1:
        raise ValueError(f"{op} {name}'s head dimension must be contiguous")


def check_lengths(op: str, name: str, tensor, batch: int, device, *, optional: bool = True) -> None:
    """Per-sequence counts: int32 [batch] on the operator's device."""
    if tensor is None and optional:
        return
    if not isinstance(tensor, torch.Tensor) or tensor.dtype is not torch.int32 or tensor.shape != (batch,):
        got = f"{tensor.dtype} {tuple(tensor.shape)}" if isinstance(tensor, torch.Tensor) else repr(tensor)
        raise ValueError(f"{op} {name} must be int32 of shape [{batch}], got {got}")
    if tensor.device != device:
        raise ValueError(f"{op} {name} must be on {device}, got {tensor.device}")
    if batch > 1 and tensor.stride(0) != 1:
        raise ValueError(f"{op} {name} must be contiguous")


def check_window(op: str, window, sinks) -> tuple[int, int]:
    for name, number, least in (("window", window, 1), ("sinks", sinks, 0)):
        if isinstance(number, bool) or not isinstance(number, int) or number < least:
            raise ValueError(f"{op} {name} must be an integer of at least {least}, got {number!r}")
    return min(window, 2**30), min(sinks, 2**30)


def check_scale(op: str, scale, head_dim: int) -> float:
    converted = head_dim**-0.5 if scale is None else float(scale)
    if not math.isfinite(converted) or converted <= 0:
        raise ValueError(f"{op} scale must be finite and positive, got {scale}")
    return converted
