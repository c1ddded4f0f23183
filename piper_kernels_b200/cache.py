"""A paged K/V cache whose bookkeeping lives on the device.

A decoding step is a run of calls without a host round trip, which can be captured in a CUDA graph::

    cache.extend(counts)                          # room for the new tokens of every sequence
    for layer in range(layers):
        ...
        cache.write(key, value, layer=layer)      # their rows
        out = cache_attention(query, cache, layer=layer, tree=tree)
    cache.compact(paths, accepted)                # of a drafted tree, keep the accepted path
"""

from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _cabi
from ._ops import raw_stream
from .attention._validation import check_lengths, check_rows

_DTYPE = {torch.float16: _cabi.PK_F16, torch.bfloat16: _cabi.PK_BF16, torch.int8: _cabi.PK_I8, torch.float32: _cabi.PK_F32}
PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_BATCH = 4096
_OP = "PageCache"
_STRIDES = C.c_int64 * 4
_MAKING_MAPS = threading.Lock()


class PageCache:
    """Keys and values of ``batch`` sequences in pages of ``page_size`` rows, for all layers of a model.

    All state is in plain tensors, which a program may read, save, and restore in place (``copy_``; their
    addresses are kept):

    ``keys``, ``values``              ``[layers, pages, kv_heads, page_size, head_dim]`` in ``dtype``
    ``key_scales``, ``value_scales``  ``[layers, pages, kv_heads, page_size]`` float32 for ``dtype=torch.int8`` (a
                                      row is ``code * scale``; scales are not negative), else ``None``
    ``table``                         int32 ``[batch, width]``: page of each ``page_size`` rows of a sequence, or -1
    ``lengths``, ``starts``           int32 ``[batch]``: rows of each sequence, and where those added last begin
    ``uses``                          int32 ``[pages]``: how many table entries name a page (0: free)
    ``refused``                       int32 ``[batch]``: 1 where the latest extend, fork or compact left a sequence
                                      alone because it could not be done

    Calls run on the current stream of the cache's device.  They change the cache in place, so calls on
    one cache from several streams need the caller's events between them.  They can be captured in a CUDA
    graph once :func:`cache_attention` has run on the device outside of one.
    """

    def __init__(self, batch: int, pages: int, page_size: int, kv_heads: int, head_dim: int, *, max_length: int | None = None,
                 layers: int = 1, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        for name, n in (("batch", batch), ("pages", pages), ("page_size", page_size), ("kv_heads", kv_heads), ("layers", layers)):
            if n < 1:
                raise ValueError(f"{_OP} {name} must be positive, got {n}")
        length = pages * page_size if max_length is None else max_length
        if length < 1:
            raise ValueError(f"{_OP} max_length must be positive, got {max_length}")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        zeros = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
        eight_bit = dtype is torch.int8
        self._adopt(zeros(*shape, dtype=dtype), zeros(*shape, dtype=dtype),
                    torch.full((batch, -(-length // page_size)), -1, dtype=torch.int32, device=device),
                    zeros(batch), zeros(batch), zeros(pages),
                    zeros(*shape[:-1], dtype=torch.float32) if eight_bit else None,
                    zeros(*shape[:-1], dtype=torch.float32) if eight_bit else None)

    @classmethod
    def from_tensors(cls, keys, values, table, lengths, starts, uses, key_scales=None, value_scales=None) -> PageCache:
        """A cache on existing state (no copy); the tensors are described above, all contiguous."""
        self = cls.__new__(cls)
        self._adopt(keys, values, table, lengths, starts, uses, key_scales, value_scales)
        return self

    def _adopt(self, keys, values, table, lengths, starts, uses, key_scales, value_scales):
        if keys.ndim != 5 or keys.shape != values.shape:
            raise ValueError(f"{_OP} keys and values must have one shape [layers, pages, kv_heads, page_size, head_dim], got "
                             f"{tuple(keys.shape)}/{tuple(values.shape)}")
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = keys.shape
        self.dtype, self.device = keys.dtype, keys.device
        if self.dtype not in (torch.float16, torch.bfloat16, torch.int8) or values.dtype is not self.dtype:
            raise ValueError(f"{_OP} keys and values must use float16, bfloat16 or int8, got {keys.dtype}/{values.dtype}")
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"{_OP} page_size must be one of {PAGE_SIZES}, got {self.page_size}")
        if self.head_dim not in (64, 128):
            raise ValueError(f"{_OP} currently supports head dimensions 64 and 128, got {self.head_dim}")
        if table.ndim != 2 or 0 in table.shape:
            raise ValueError(f"{_OP} table must have shape [batch, width], got {tuple(table.shape)}")
        self.batch, self.width = table.shape
        if self.batch > MAX_BATCH:
            raise ValueError(f"{_OP} holds at most {MAX_BATCH} sequences, got {self.batch}")
        if self.width * self.page_size >= 2**30:
            raise ValueError(f"{_OP} sequences must stay below 2^30 rows, got {self.width * self.page_size}")
        if self.batch * self.width >= 2**31:
            raise ValueError(f"{_OP} table must have fewer than 2^31 entries, got {self.batch} x {self.width}")
        scales = (self.layers, self.pages, self.kv_heads, self.page_size) if self.dtype is torch.int8 else None
        wanted = {"keys": (keys, self.dtype, keys.shape), "values": (values, self.dtype, keys.shape),
                  "table": (table, torch.int32, (self.batch, self.width)), "lengths": (lengths, torch.int32, (self.batch,)),
                  "starts": (starts, torch.int32, (self.batch,)), "uses": (uses, torch.int32, (self.pages,)),
                  "key_scales": (key_scales, torch.float32, scales), "value_scales": (value_scales, torch.float32, scales)}
        for name, (tensor, dtype, shape) in wanted.items():
            if shape is None:
                if tensor is not None:
                    raise ValueError(f"{_OP} {name} belongs to an int8 cache, not to {self.dtype}")
            elif tensor is None or tensor.dtype is not dtype or tensor.shape != shape or not tensor.is_contiguous():
                got = "none" if tensor is None else f"{tensor.dtype} {tuple(tensor.shape)}"
                raise ValueError(f"{_OP} {name} must be contiguous {dtype} of shape {tuple(shape)}, got {got}")
            elif tensor.device != self.device:
                raise ValueError(f"{_OP} tensors must share a device, got {self.device}/{tensor.device} for {name}")
            setattr(self, name, tensor)
        self.refused = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        self.workspaces: dict[tuple[int, int], int] = {}  # bytes that cache_attention needs, by (heads, tokens)
        self._scratch = torch.zeros(4 * self.batch + 4, dtype=torch.int32, device=self.device)
        c = self._c = _cabi.PkCache()
        c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim = keys.shape
        c.batch, c.width, c.dtype = self.batch, self.width, _DTYPE[self.dtype]
        for name in wanted:
            if getattr(self, name) is not None:
                setattr(c, name, getattr(self, name).data_ptr())
        c.refused, c.scratch = self.refused.data_ptr(), self._scratch.data_ptr()
        c.device = self.device.index or 0
        self._maps = None  # the pool's copy maps, made at the first attention

    @property
    def max_length(self) -> int:
        """Rows that one sequence can hold."""
        return self.width * self.page_size

    def handle(self) -> _cabi.PkCache:
        """The cache for the C ABI, on the current stream of its device (one struct per call: callers may be threads)."""
        if self.device.type != "cuda":
            raise RuntimeError("PageCache runs only on CUDA tensors (B200, sm_100a); there is no CPU path")
        c = _cabi.PkCache.from_buffer_copy(self._c)
        c.stream = raw_stream(c.device)
        return c

    def mapped_handle(self) -> _cabi.PkCache:
        """The same with the copy maps of keys and values, which are made once for the cache's life."""
        c = self.handle()
        maps = self._maps
        if maps is None:
            memory = C.create_string_buffer(_cabi.PK_CACHE_MAP_BYTES + 64)
            at = -(-C.addressof(memory) // 64) * 64
            _cabi.check(_cabi.lib().pk_cache_maps(C.byref(c), at))
            with _MAKING_MAPS:  # of two threads that made maps the first one's stay: they may be in use already
                if self._maps is None:
                    self._maps = (memory, at)
                maps = self._maps
        c.maps = maps[1]
        return c

    def check_layer(self, layer: int) -> int:
        if isinstance(layer, bool) or not isinstance(layer, int) or not 0 <= layer < self.layers:
            raise ValueError(f"{_OP} layer must be in [0, {self.layers}), got {layer!r}")
        return layer

    def extend(self, counts: torch.Tensor) -> None:
        """Makes room for ``counts[b]`` (int32 ``[batch]``; negative counts as 0) more rows of each sequence.

        ``starts`` becomes the old and ``lengths`` the new length.  New pages are the lowest free ones, in the
        order of the sequences.  A partly filled last page that other sequences also use is replaced by a copy;
        when all of its owners are extended, the longest of them (the first of these) keeps it.  A sequence that
        would pass ``max_length``, or that the free pages (counted from the first sequence on) do not reach, is refused.
        """
        check_lengths(_OP, "counts", counts, self.batch, self.device, optional=False)
        _cabi.check(_cabi.lib().pk_cache_extend(C.byref(self.handle()), counts.data_ptr()))

    def write(self, key: torch.Tensor, value: torch.Tensor, *, layer: int | None = None) -> None:
        """Stores the rows that the last :meth:`extend` made room for.

        ``key`` and ``value`` are ``[batch, kv_heads, tokens, head_dim]`` for one ``layer``, or ``[layers, batch,
        kv_heads, tokens, head_dim]`` for all (``layer=None``); FP16/BF16, the cache's dtype unless it is int8.
        Sequence ``b`` takes its first ``lengths[b] - starts[b]`` rows; ``tokens`` has to reach the largest of
        these.  Int8 rows: ``scale = max|x| / 127 + 1e-7``, codes rounded to nearest even; a row with a value
        that is not finite reads back as NaN.
        """
        ndim = 5 if layer is None else 4
        check_rows(_OP, "key", key, ndim)
        check_rows(_OP, "value", value, ndim)
        if key.shape != value.shape or key.dtype is not value.dtype:
            raise ValueError(f"{_OP} key and value must match, got {key.dtype} {tuple(key.shape)}/{value.dtype} {tuple(value.shape)}")
        lead = (self.layers, self.batch, self.kv_heads) if layer is None else (self.batch, self.kv_heads)
        if key.shape[:-2] != lead or key.shape[-1] != self.head_dim:
            raise ValueError(f"{_OP} key and value must have shape [{', '.join(map(str, lead))}, tokens, {self.head_dim}], got {tuple(key.shape)}")
        if key.shape[-2] == 0:
            raise ValueError(f"{_OP} does not accept empty rows")
        if self.dtype is not torch.int8 and key.dtype is not self.dtype:
            raise ValueError(f"{_OP} rows and cache must share a dtype, got {key.dtype}/{self.dtype}")
        if key.device != self.device or value.device != self.device:
            raise ValueError(f"{_OP} rows and cache must share a device, got {key.device}/{value.device}/{self.device}")
        if torch.is_grad_enabled() and (key.requires_grad or value.requires_grad):
            raise RuntimeError(f"{_OP} is inference-only and does not support autograd")
        ks, vs = (t.stride()[:4] if layer is None else (0, *t.stride()[:3]) for t in (key, value))
        at = -1 if layer is None else self.check_layer(layer)
        _cabi.check(_cabi.lib().pk_cache_write(C.byref(self.handle()), at, key.data_ptr(), value.data_ptr(),
                                               _STRIDES(*ks), _STRIDES(*vs), _DTYPE[key.dtype], key.shape[-2]))

    def read(self, first: torch.Tensor, count: int, *, layer: int | None = None,
             dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Copies rows ``first[b] + [0, count)`` of every sequence out of the cache.

        Returns key and value, ``[batch, kv_heads, count, head_dim]`` for one ``layer`` or ``[layers, ...]`` for all,
        in ``dtype`` (float16, bfloat16 or float32; default: the cache's own, float32 of an int8 cache).  Rows
        that a sequence does not have read as zero.
        """
        check_lengths(_OP, "first", first, self.batch, self.device, optional=False)
        if isinstance(count, bool) or not isinstance(count, int) or not 1 <= count < 2**30:
            raise ValueError(f"{_OP} count must be a positive integer, got {count!r}")
        if dtype is None:
            dtype = torch.float32 if self.dtype is torch.int8 else self.dtype
        if dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise ValueError(f"{_OP} reads as float16, bfloat16 or float32, got {dtype}")
        lead = () if layer is not None else (self.layers,)
        at = -1 if layer is None else self.check_layer(layer)
        handle = self.handle()
        shape = (*lead, self.batch, self.kv_heads, count, self.head_dim)
        key, value = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        _cabi.check(_cabi.lib().pk_cache_read(C.byref(handle), at, first.data_ptr(), count, key.data_ptr(), value.data_ptr(), _DTYPE[dtype]))
        return key, value

    def fork(self, parents: torch.Tensor) -> None:
        """Sequence ``b`` becomes what sequence ``parents[b]`` (int32 ``[batch]``) was before the call.

        ``parents[b] = b`` keeps it, a negative one empties it, several may name the same parent.  Pages are
        shared, not copied; :meth:`extend` copies a shared last page when it has to.  ``parents[b] >= batch`` is
        refused: the sequence keeps its rows.  ``starts`` becomes ``lengths`` everywhere: rows added before are no
        longer the latest.
        """
        check_lengths(_OP, "parents", parents, self.batch, self.device, optional=False)
        _cabi.check(_cabi.lib().pk_cache_fork(C.byref(self.handle()), parents.data_ptr()))

    def truncate(self, lengths: torch.Tensor) -> None:
        """Every sequence keeps its first ``lengths[b]`` rows (int32 ``[batch]``; 0 or less: none; more than it
        has: all) and releases the pages behind them; ``starts`` becomes ``lengths``."""
        check_lengths(_OP, "lengths", lengths, self.batch, self.device, optional=False)
        _cabi.check(_cabi.lib().pk_cache_truncate(C.byref(self.handle()), lengths.data_ptr()))

    def compact(self, paths: torch.Tensor, counts: torch.Tensor) -> None:
        """Of the rows added by the last :meth:`extend` keeps ``paths[b, i]``, ``i < counts[b]``, in all layers.

        ``paths`` is int32 ``[batch, most]``, ``counts`` int32 ``[batch]``.  Row ``starts[b] + paths[b, i]`` moves to
        ``starts[b] + i``; the rest is released as by :meth:`truncate`.  A path has to rise strictly and stay within
        the added rows; a sequence whose path or count does not is refused and left as it was.
        """
        if paths.dtype is not torch.int32 or paths.ndim != 2 or paths.shape[0] != self.batch or paths.shape[1] == 0:
            raise ValueError(f"{_OP} paths must be int32 of shape [{self.batch}, most], got {paths.dtype} {tuple(paths.shape)}")
        if paths.device != self.device:
            raise ValueError(f"{_OP} paths must be on {self.device}, got {paths.device}")
        if paths.shape[1] > 1 and paths.stride(1) != 1:
            raise ValueError(f"{_OP} paths' last dimension must be contiguous")
        check_lengths(_OP, "counts", counts, self.batch, self.device, optional=False)
        _cabi.check(_cabi.lib().pk_cache_compact(C.byref(self.handle()), paths.data_ptr(), paths.stride(0), paths.shape[1], counts.data_ptr()))
