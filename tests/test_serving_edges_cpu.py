"""CPU tests of the serving operators' edges: the list model of shared last pages, refusals."""

import ctypes as C
import random

import pytest
import torch

import piper_kernels_b200 as pk
from _serving import ListCache
from _serving_edges import LongestKeeps, unequal_owners
from piper_kernels_b200 import _cabi


def test_longest_owner_keeps_a_shared_page():
    m = LongestKeeps(2, 1, 16, 1)
    m.extend([9, 0])
    m.fork([0, 0])
    m.truncate([5, 9])
    m.extend([1, 1])  # no page is free for a copy
    assert m.refused == [1, 0] and m.length == [5, 10] and not m.overwritten()
    m = LongestKeeps(2, 2, 16, 1)
    m.extend([9, 0])
    m.fork([0, 0])
    m.truncate([5, 9])
    m.extend([1, 1])
    assert m.refused == [0, 0] and m.own == [[1], [0]] and m.copied == [(0, 1, 5)] and not m.overwritten()


@pytest.mark.parametrize("seed", range(20))
def test_no_new_row_falls_on_a_row_that_another_sequence_holds(seed):
    rng = random.Random(seed)
    batch, page = rng.choice([2, 3, 5]), 16
    m = LongestKeeps(batch, batch + rng.randrange(3), page, 3)
    for what, argument in unequal_owners(rng, batch, page, 60):
        getattr(m, what)(argument)
        assert not m.overwritten()


def test_equal_owners_are_as_in_the_list_model():
    rng = random.Random(1)
    models = [LongestKeeps(6, 14, 16, 3), ListCache(6, 14, 16, 3)]
    for step in range(60):
        counts, keep = [rng.choice([1, 1, 7, 20])] * 6, rng.choice([3, 20, 10**6])
        for m in models:
            m.extend(counts)
            if step % 3 == 2:
                m.fork([step % 6] * 6)
            m.truncate([keep] * 6)
        a, b = models
        assert (a.own, a.length, a.start, a.refused) == (b.own, b.length, b.start, b.refused)


def test_tables_that_32_bits_cannot_count_are_refused():
    lib, n = _cabi.lib(), C.c_uint64()
    query = _cabi.PkCacheQuery(4, 1, 0, _cabi.PK_F16, 0, 0, 0.1, 256)

    def ask(batch, width):
        c = _cabi.PkCache(1, 10, 2, 16, 64, batch, width, _cabi.PK_F16)
        for name in ("keys", "values", "table", "lengths", "starts", "uses", "refused", "scratch"):
            setattr(c, name, 256)
        return lib.pk_cache_attention_workspace_bytes(C.byref(c), C.byref(query), C.byref(n))

    assert ask(4096, 2**19 - 1) == ask(1, 2**26 - 1) == ask(4095, 2**19) == _cabi.PK_OK
    assert ask(4096, 2**19) == ask(33, 2**26 - 1) == _cabi.PK_ERR_BAD_ARG
    assert b"table" in lib.pk_last_error()
    make = {n: torch.empty(s, dtype=d, device="meta") for n, s, d in (
        ("keys", (1, 4, 1, 16, 64), torch.float16), ("values", (1, 4, 1, 16, 64), torch.float16), ("lengths", 4096, torch.int32),
        ("starts", 4096, torch.int32), ("uses", 4, torch.int32))}
    with pytest.raises(ValueError, match="table must have fewer than"):
        pk.PageCache.from_tensors(table=torch.empty(4096, 2**19, dtype=torch.int32, device="meta"), **make)


def test_copy_maps_of_two_threads_are_one(monkeypatch):
    """A second thread asks for the maps while the first one's are being made: what either was given stays alive."""
    cache = pk.PageCache(1, 2, 16, 1, 64, dtype=torch.float16, device="cpu")
    given, inner = [], []

    class Library:
        def pk_cache_maps(self, c, at):
            given.append(at)
            if len(given) == 1:
                inner.append(cache.mapped_handle())
            return _cabi.PK_OK

    monkeypatch.setattr(cache, "handle", _cabi.PkCache)
    monkeypatch.setattr(_cabi, "lib", Library)
    outer = cache.mapped_handle()
    assert outer.maps == inner[0].maps == cache.mapped_handle().maps and outer.maps in given
    start = C.addressof(cache._maps[0])
    assert start <= outer.maps <= start + 64 and outer.maps % 64 == 0


def test_stalled_wait_drill_refuses_before_the_device():
    lib = _cabi.lib()
    p, c, q = _cabi.PkWindowProblem(), _cabi.PkCache(), _cabi.PkCacheQuery()
    for cycles, copy in ((0, 1), (-5, 1), (2 * 10**9, 1), (1000, -2)):
        assert lib.pk_debug_window_stall(C.byref(p), cycles, copy) == _cabi.PK_ERR_BAD_ARG and b"stall" in lib.pk_last_error()
        assert lib.pk_debug_cache_stall(C.byref(c), C.byref(q), cycles, copy) == _cabi.PK_ERR_BAD_ARG and b"stall" in lib.pk_last_error()
    assert lib.pk_debug_window_stall(C.byref(p), 1000, 1) == _cabi.PK_ERR_BAD_ARG and b"batch" in lib.pk_last_error()
