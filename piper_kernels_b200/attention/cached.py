"""Public ``cache_attention``: attention of single tokens, chains and trees of drafted tokens over a paged cache."""

from __future__ import annotations

import ctypes as C
from typing import TYPE_CHECKING

import torch

from .. import _cabi
from ._validation import check_rows, check_scale, check_window

if TYPE_CHECKING:
    from ..cache import PageCache

_OP = "Cache Attention"
MAX_TREE_TOKENS = 64


def cache_attention(
    query: torch.Tensor,
    cache: PageCache,
    *,
    layer: int = 0,
    window: int | None = None,
    sinks: int = 0,
    tree: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of the tokens that :meth:`PageCache.extend` added last over one layer of the cache.

    ``query`` is ``[batch, heads, tokens, head_dim]`` (FP16/BF16, any strides but a contiguous head
    dimension); ``heads`` is a multiple of the cache's ``kv_heads``.  Token ``t`` of sequence ``b`` stands at
    row ``cache.starts[b] + t``; tokens at or behind ``cache.lengths[b]`` do not exist and give zeros.  A
    token sees every row up to its own.

    ``tree`` (int32 ``[batch, tokens]`` or ``[tokens]``, at most 64 tokens) makes the added rows a tree of
    drafted tokens: ``tree[b, t]`` is the token under which ``t`` hangs, one before it, or -1 where it hangs
    under the context itself (any other value counts as -1).  A token then sees the context, itself and
    the tokens above it.  ``window`` and ``sinks`` limit what is seen as in :func:`window_attention`, by
    positions: a drafted token's position is ``cache.starts[b]`` plus the number of tokens above it.

    Rows of an 8-bit cache enter as ``code * scale``.  The result is ``[batch, heads, tokens, head_dim]`` in
    the query's dtype.  Inference only.
    """
    check_rows(_OP, "query", query)
    batch, heads, tokens, head_dim = query.shape
    if query.device != cache.device:
        raise ValueError(f"{_OP} query and cache must share a device, got {query.device}/{cache.device}")
    if cache.dtype is not torch.int8 and query.dtype is not cache.dtype:
        raise ValueError(f"{_OP} query and cache must share a dtype, got {query.dtype}/{cache.dtype}")
    if batch != cache.batch:
        raise ValueError(f"{_OP} requires one query row per sequence of the cache, got {batch}/{cache.batch}")
    if tokens == 0 or heads == 0:
        raise ValueError(f"{_OP} does not accept empty queries")
    if heads % cache.kv_heads:
        raise ValueError(f"{_OP} query heads must be a multiple of the cache's heads, got {heads}/{cache.kv_heads}")
    if head_dim != cache.head_dim:
        raise ValueError(f"{_OP} head dimensions must match, got {head_dim}/{cache.head_dim}")
    layer = cache.check_layer(layer)
    limit, sinks = check_window(_OP, 2**30 if window is None else window, sinks)
    tree_stride = 0
    if tree is not None:
        if tokens > MAX_TREE_TOKENS:
            raise ValueError(f"{_OP} trees have at most {MAX_TREE_TOKENS} tokens, got {tokens}")
        if tree.dtype is not torch.int32 or tree.shape not in ((batch, tokens), (tokens,)):
            raise ValueError(f"{_OP} tree must be int32 of shape [{batch}, {tokens}] or [{tokens}], got {tree.dtype} {tuple(tree.shape)}")
        if tree.device != query.device:
            raise ValueError(f"{_OP} tree must be on {query.device}, got {tree.device}")
        if tokens > 1 and tree.stride(-1) != 1:
            raise ValueError(f"{_OP} tree's last dimension must be contiguous")
        tree_stride = tree.stride(0) if tree.ndim == 2 else 0
    if torch.is_grad_enabled() and query.requires_grad:
        raise RuntimeError(f"{_OP} is an inference-only operator and does not support autograd")
    converted_scale = check_scale(_OP, scale, head_dim)
    from .. import _ops

    _ops._require_cuda(query, "cache_attention")
    _ops.poll_device_fault(query.device.index)
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    q = _cabi.PkCacheQuery(heads, tokens, layer, _ops._DTYPE[query.dtype], 0 if window is None else limit, sinks, converted_scale, query.data_ptr(),
                           query.stride()[:3], None if tree is None else tree.data_ptr(), tree_stride, out.data_ptr(), None, 0)
    c = cache.mapped_handle()
    lib = _cabi.lib()
    nbytes = cache.workspaces.get((heads, tokens))
    if nbytes is None:
        n = C.c_uint64(0)
        _cabi.check(lib.pk_cache_attention_workspace_bytes(C.byref(c), C.byref(q), C.byref(n)))
        nbytes = cache.workspaces[heads, tokens] = n.value
    # allocated on the stream that uses it
    ws = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
    q.workspace, q.workspace_bytes = ws.data_ptr(), nbytes
    _cabi.check(lib.pk_cache_attention_fwd(C.byref(c), C.byref(q)))
    return out
