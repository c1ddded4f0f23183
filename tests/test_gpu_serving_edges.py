"""Serving operators on a B200 at the places where a result could be lost: single keys far above the rest,
values that are not finite side by side, values near the type's largest, shared pages when the pool runs
out, waits that run out."""

import ctypes as C
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import piper_kernels_b200 as pk
from _serving import attend, check, tree_visible, window_visible
from _serving_edges import LongestKeeps, unequal_owners
from piper_kernels_b200 import _cabi, _ops

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
ROOT = Path(__file__).resolve().parents[1]
LN2 = 0.6931471805599453


def normal(*shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache_of(k, v, tokens, page=16):
    """A cache whose sequences hold the rows of k and v, the last ``tokens`` of them added last."""
    batch, kv_heads, n, dim = k.shape
    cache = pk.PageCache(batch, batch * -(-n // page), page, kv_heads, dim, dtype=k.dtype, max_length=n)
    for count in (n - tokens, tokens):
        cache.extend(ints([count] * batch))
        at = slice(0, count) if count == n - tokens else slice(n - tokens, n)
        if count:
            cache.write(k[:, :, at].contiguous(), v[:, :, at].contiguous(), layer=0)
    return cache


def check_rows(got, q, k, v, *, window, scale, heads=None):
    group, visible = q.shape[1] // k.shape[1], window_visible(q.shape[2], k.shape[2], window, 0, k.shape[2]).cuda()
    for b in range(q.shape[0]):
        for h in range(q.shape[1]) if heads is None else heads:
            want, off = attend(q[b, h], k[b, h // group], v[b, h // group], visible, scale, q.dtype)
            check(got[b, h], want, off, f"batch {b} head {h}")


@pytest.mark.parametrize("gap", [13, 100, 128, 129, 140, 200, 255, 256, 261, 300, 400, 512, 520, 700])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("rows", ["all", "one"])
def test_single_key_far_above_the_rest(gap, dim, dtype, rows):
    """Head h's key at place h of the second 128-key tile scores ``gap`` (base 2) above all others, in every query
    row or in one of them; prompt rows (two row tiles, the second with few rows) and rows over a cache."""
    heads, n_q, n_k = 32, 140, 300
    q = torch.zeros(1, heads, n_q, dim, device="cuda")
    q[:, :, slice(None) if rows == "all" else 77] = 1
    k = torch.zeros(1, heads, n_k, dim, device="cuda")
    # the first rows of the chunk stand at 160: some rows of either kind do not see all of the tile
    k[0, torch.arange(heads), 128 + torch.arange(heads)] = gap * LN2 / dim
    q, k, v = q.to(dtype), k.to(dtype), normal(1, heads, n_k, dim, dtype=dtype, seed=gap)
    check_rows(pk.window_attention(q, k, v, window=400, scale=1.0), q, k, v, window=400, scale=1.0)
    check_rows(pk.cache_attention(q, cache_of(k, v, n_q), scale=1.0), q, k, v, window=400, scale=1.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("place", [14, 15, 30, 79])
def test_single_key_far_above_the_rest_in_shared_units(dtype, place):
    """The same in long rows whose key tiles several CTAs share, with random keys, for single rows of the last tile."""
    q, k = normal(1, 2, 700, 128, dtype=dtype, seed=1).abs(), 0.1 * normal(1, 2, 2500, 128, dtype=dtype, seed=2)
    v = normal(1, 2, 2500, 128, dtype=dtype, seed=3)
    k[0, 0, 1280 + place] += 14
    k[0, 1, 128 + place] += 20
    check_rows(pk.window_attention(q, k, v, window=3000), q, k, v, window=3000, scale=128**-0.5)


def test_single_key_far_above_the_rest_in_a_tree():
    """64 drafted tokens (128 rows of a key head), one of which scores far above the context in the rows below it."""
    q = torch.ones(1, 32, 64, 64, device="cuda", dtype=F16)
    k = torch.zeros(1, 16, 300, 64, device="cuda", dtype=F16)
    k[0, torch.arange(16), 236 + torch.arange(16)] = 150 * LN2 / 64  # draft tokens 0 to 15
    v = normal(1, 16, 300, 64, dtype=F16, seed=4)
    tree = [-1] + [(t - 1) // 2 for t in range(1, 64)]
    got = pk.cache_attention(q, cache_of(k, v, 64), scale=1.0, tree=ints(tree))
    visible = tree_visible(64, 236, 300, tree, None, 0).cuda()
    for h in range(32):
        want, off = attend(q[0, h], k[0, h // 2], v[0, h // 2], visible, 1.0, F16)
        check(got[0, h], want, off, f"head {h}")


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("n_q,n_k,window", [(300, 300, 400), (300, 300, 40), (300, 2600, 3000), (9, 300, 400)])
@pytest.mark.parametrize("apart", [1, 16, 64])
def test_two_nan_keys_make_every_row_that_sees_them_nan(dim, dtype, n_q, n_k, window, apart):
    """Head h: key rows at place h of a tile and ``apart`` behind it are NaN; whole units, units whose key tiles
    several CTAs share, few rows, and rows over a cache."""
    heads = 32
    q, k, v = (normal(1, heads, n, dim, dtype=dtype, seed=s) for n, s in ((n_q, 5), (n_k, 6), (n_k, 7)))
    h = torch.arange(heads, device="cuda")
    first = (128 if n_k == 300 else 2304) + h
    clean = k.clone()
    k[0, h, first] = k[0, h, first + apart] = float("nan")
    visible = window_visible(n_q, n_k, window, 0, n_k).cuda()
    calls = [pk.window_attention(q, k, v, window=window)]
    if n_k == 300:
        calls.append(pk.cache_attention(q, cache_of(k, v, n_q), window=window))
    for got in calls:
        for i in range(heads):
            lost = visible[:, first[i]] | visible[:, first[i] + apart]
            assert lost.any() and got[0, i][lost].isnan().all()
            want, off = attend(q[0, i], clean[0, i], v[0, i], visible, dim**-0.5, dtype)
            check(got[0, i][~lost], want[~lost], off[~lost], f"head {i}")


class TaggedCache:
    """A cache and its list model, whose rows hold numbers of their own; every row is compared after every call."""

    def __init__(self, batch, pages, page, width):
        self.cache = pk.PageCache(batch, pages, page, 1, 64, layers=2, dtype=F16, max_length=width * page)
        self.model = LongestKeeps(batch, pages, page, width)
        self.rows, self.tag = [[] for _ in range(batch)], 0

    def call(self, what, argument):
        m, c = self.model, self.cache
        getattr(m, what)(argument)
        getattr(c, what)(ints(argument))
        if what == "fork":
            self.rows = [list(self.rows[p]) for p in argument]
        self.rows = [rows[: m.start[b]] for b, rows in enumerate(self.rows)]
        if what == "extend":
            added = [m.length[b] - m.start[b] for b in range(m.batch)]
            data = torch.zeros(2, m.batch, 1, max(1, *added), 64, dtype=F16)
            for b, n in enumerate(added):
                for t in range(n):
                    self.tag = self.tag % 2047 + 1
                    self.rows[b].append(self.tag)
                    data[:, b, 0, t] = self.tag
            c.write(data.cuda(), -data.cuda())
        assert [c.table.tolist(), c.lengths.tolist(), c.starts.tolist(), c.uses.tolist(), c.refused.tolist()] == [
            m.table(), m.length, m.start, m.uses(), m.refused]
        longest = max(1, *m.length)
        want = torch.tensor([rows + [0] * (longest - len(rows)) for rows in self.rows], dtype=F16, device="cuda")
        k, v = c.read(ints([0] * m.batch), longest)
        want = want[None, :, None, :, None].expand_as(k)
        assert torch.equal(k, want) and torch.equal(v, -want)


def test_extend_leaves_the_rows_of_a_refused_owner():
    for pages in (1, 2):
        c = TaggedCache(2, pages, 16, 1)
        c.call("extend", [9, 0])
        c.call("fork", [0, 0])
        c.call("truncate", [5, 9])
        c.call("extend", [1, 1])
        assert c.cache.refused.tolist() == [2 - pages, 0]


@pytest.mark.parametrize("seed", range(4, 10))
def test_sequences_of_different_lengths_that_share_a_last_page(seed):
    rng = random.Random(seed)
    batch = rng.choice([2, 3, 5])
    c = TaggedCache(batch, batch + rng.randrange(3), 16, 3)
    for what, argument in unequal_owners(rng, batch, 16, 60):
        c.call(what, argument)


def test_extend_of_nearly_the_largest_batch():
    """In a process of its own: leave for more shared memory, once given, stays with the kernel."""
    code = """
import torch
import piper_kernels_b200 as pk
for batch in (3400, 4084, 4085, 4090, 4095, 4096):
    cache = pk.PageCache(batch, batch, 16, 1, 64, dtype=torch.float16, max_length=16)
    cache.extend(torch.ones(batch, dtype=torch.int32, device="cuda"))
    assert cache.table.flatten().tolist() == list(range(batch)) and int(cache.lengths.sum()) == batch, batch
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n_q,n_k", [(1, 200), (9, 300), (40, 1500), (140, 300), (300, 2600)])
def test_results_up_to_the_largest_number_of_float16(dim, n_q, n_k):
    """Every value is +-65504 and a later key's weight is up to 2^12 times the first ones': the result is finite, and as
    near 65504 as two roundings allow (probabilities, 2^-11 relative, and the result, 2^-11: ``attend``).  Single
    tokens, few rows, prompt rows and units that several CTAs share; also over a cache."""
    heads = 24
    q = torch.ones(1, heads, n_q, dim, device="cuda", dtype=F16)
    k = torch.zeros(1, heads, n_k, dim, device="cuda")
    h = torch.arange(heads, device="cuda")
    k[0, h, n_k - n_q - h] = (0.5 * h[:, None] + 0.3) * LN2 / dim
    v = torch.full((1, heads, n_k, dim), 65504.0, device="cuda")
    v[..., dim // 2:] *= -1
    k, v = k.to(F16), v.to(F16)
    calls = [pk.window_attention(q, k, v, window=n_k, scale=1.0)]
    if n_k <= 300:
        calls.append(pk.cache_attention(q, cache_of(k, v, n_q), scale=1.0))
    for got in calls:
        assert got.isfinite().all()
        check_rows(got, q, k, v, window=n_k, scale=1.0, heads=(0, 7, 23))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [5, 12, 40])
@pytest.mark.parametrize("n_q,n_k", [(1, 200), (9, 300), (40, 1500), (140, 300), (1000, 4000)])
def test_largest_number_of_float16_under_random_weights(dim, window, n_q, n_k):
    """The same with scores anywhere in [0, 12) (base 2) and few keys to a row, so that a rounded probability
    decides the quotient."""
    heads = 48
    gen = torch.Generator().manual_seed(n_q + window)
    q = torch.ones(1, heads, n_q, dim, device="cuda", dtype=F16)
    k = (12 * LN2 / dim * torch.rand(1, heads, n_k, 1, generator=gen).cuda()).expand(1, heads, n_k, dim).to(F16)
    v = torch.full((1, heads, n_k, dim), 65504.0, device="cuda", dtype=F16)
    v[..., dim // 2:] *= -1
    calls = [pk.window_attention(q, k, v, window=window, scale=1.0)]
    if n_k <= 300:
        calls.append(pk.cache_attention(q, cache_of(k, v, n_q), window=window, scale=1.0))
    for got in calls:
        assert got.isfinite().all()
        check_rows(got, q, k, v, window=window, scale=1.0, heads=(0, 11, 47))


@pytest.mark.parametrize("n_q,n_k", [(140, 300), (300, 2600)])
def test_largest_number_of_float16_in_prompt_rows(n_q, n_k):
    """The same with one key that outweighs all others together, by every factor that does not yet raise the
    reference of its tile."""
    heads = 256
    gen = torch.Generator().manual_seed(n_q)
    gaps = 10.5 + 1.45 * torch.rand(heads, generator=gen).cuda()
    q = torch.ones(1, heads, n_q, 64, device="cuda", dtype=F16)
    k = torch.full((1, heads, n_k, 64), -20 * LN2 / 64, device="cuda")
    k[:, :, :4] = 0
    k[0, torch.arange(heads), n_k - n_q - torch.arange(heads) % 30] = gaps[:, None] * LN2 / 64
    k = k.to(F16)
    v = torch.full((1, heads, n_k, 64), 65504.0, device="cuda", dtype=F16)
    for got in (pk.window_attention(q, k, v, window=n_k, scale=1.0), pk.cache_attention(q, cache_of(k, v, n_q), scale=1.0)):
        assert got.isfinite().all()
        check_rows(got, q, k, v, window=n_k, scale=1.0, heads=range(0, heads, 17))


SENTINEL = 777.0


def window_stall(q, k, v, window, cycles, copy):
    """pk_debug_window_stall into rows that hold a number of their own."""
    lib, n, out = _cabi.lib(), C.c_uint64(), torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    p = _cabi.PkWindowProblem(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], _ops._DTYPE[q.dtype], window, 0, q.shape[3] ** -0.5,
                              q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride()[:3], k.stride()[:3], v.stride()[:3], None, out.data_ptr(),
                              None, 0, 0, torch.cuda.current_stream().cuda_stream)
    _cabi.check(lib.pk_window_workspace_bytes(C.byref(p), C.byref(n)))
    ws = torch.full((n.value,), 255, dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = ws.data_ptr(), n.value
    _cabi.check(lib.pk_debug_window_stall(C.byref(p), cycles, copy))
    torch.cuda.synchronize()
    return out


def cache_stall(q, cache, cycles, copy, tree=None, scale=None):
    lib, n, out = _cabi.lib(), C.c_uint64(), torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    c = cache.mapped_handle()
    query = _cabi.PkCacheQuery(q.shape[1], q.shape[2], 0, _ops._DTYPE[q.dtype], 0, 0, q.shape[3] ** -0.5 if scale is None else scale, q.data_ptr(),
                               q.stride()[:3], None if tree is None else tree.data_ptr(), 0, out.data_ptr(), None, 0)
    _cabi.check(lib.pk_cache_attention_workspace_bytes(C.byref(c), C.byref(query), C.byref(n)))
    ws = torch.full((n.value,), 255, dtype=torch.uint8, device="cuda")
    query.workspace, query.workspace_bytes = ws.data_ptr(), n.value
    _cabi.check(lib.pk_debug_cache_stall(C.byref(c), C.byref(query), cycles, copy))
    torch.cuda.synchronize()
    return out


def check_stalled(stall, run, copies, site):
    """``stall(copy)`` leaves rows of NaN and rows as ``run`` makes them, nothing else; the wait is reported once, and
    the next call is as before."""
    want = run()
    lost = []
    for copy in copies:
        got = stall(copy)
        nan = got.isnan().all(-1)
        assert torch.equal(got[~nan], want[~nan]), copy
        lost.append(int(nan.sum()))
        if lost[-1]:
            with pytest.raises(_cabi.PiperB200Error, match=f"wait site ({site});"):
                run()
        assert torch.equal(run(), want)
    return lost


CYCLES = 2_000_000  # about a millisecond


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("batch,heads,n_q,n_k", [
    (1, 32, 1, 4000),   # a cluster for every key head
    (300, 2, 1, 300),   # units shared by all CTAs
    (3, 4, 32, 3000),   # the same, 64 rows
    (2, 8, 20, 40),     # a CTA for every key head
])
def test_stalled_wait_of_few_rows(dim, dtype, batch, heads, n_q, n_k):
    q = normal(batch, heads, n_q, dim, dtype=dtype, seed=8)
    k, v = (normal(batch, heads // 2, n_k, dim, dtype=dtype, seed=s) for s in (9, 10))
    lost = check_stalled(lambda copy: window_stall(q, k, v, n_k, CYCLES, copy), lambda: pk.window_attention(q, k, v, window=n_k), (0, 1, 4, -1, 10**6), "61|62")
    assert lost[0] == batch * q.shape[1] * n_q and lost[3:] == [0, 0]


@pytest.mark.parametrize("store", [F16, torch.int8])
@pytest.mark.parametrize("tokens,room", [(1, None), (16, None), (16, 40000), (64, 40000)])
def test_stalled_wait_over_a_cache(store, tokens, room):
    lengths, page, dim = [1500, 700, tokens], 32, 128
    cache = pk.PageCache(3, 90, page, 2, dim, dtype=store, max_length=room or 1504)
    for counts in ([n - tokens for n in lengths], [tokens] * 3):
        cache.extend(ints(counts))
        rows = normal(2, 3, 2, max(counts), dim, dtype=F16, seed=11)
        cache.write(rows[0], rows[1], layer=0)
    q, tree = normal(3, 8, tokens, dim, dtype=F16, seed=12), ints([-1] + [(t - 1) // 2 for t in range(1, tokens)])
    lost = check_stalled(lambda copy: cache_stall(q, cache, CYCLES, copy, tree), lambda: pk.cache_attention(q, cache, tree=tree), (0, 1, 3, -1), "61|62|7[0-9]|80")
    assert lost[0] == q[..., 0].numel() and lost[3] == 0


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("batch,heads,n_q,n_k", [
    (1, 8, 300, 300),      # units of few key tiles
    (1, 2, 1500, 3000),    # all units shared
    (10, 16, 100, 333),    # more units than SMs, the rest of them shared
    (40, 16, 80, 200),     # several rounds, none shared
])
def test_stalled_wait_of_prompt_rows(dim, dtype, batch, heads, n_q, n_k):
    q = normal(batch, heads, n_q, dim, dtype=dtype, seed=13)
    k, v = (normal(batch, heads, n_k, dim, dtype=dtype, seed=s) for s in (14, 15))
    lost = check_stalled(lambda copy: window_stall(q, k, v, n_k, CYCLES, copy), lambda: pk.window_attention(q, k, v, window=n_k), (0, 1, 2, 3, 7, 12, -1, 10**6), "7[0-9]|80")
    assert lost[0] == lost[1] == q[..., 0].numel() and lost[6:] == [0, 0]


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("batch,n_q,n_k", [
    (592, 16, 20000),  # few rows, two units for each of 296 CTAs
    (592, 100, 4000),  # prompt rows, four units for each of 148 CTAs
])
def test_waits_for_rows_that_are_evaluated_one_by_one(dim, dtype, batch, n_q, n_k):
    """A NaN in the last value row reaches the tiles of tokens that do not see it: these are evaluated one by one, which
    takes some hundred times as long as the other warps' waits may last here."""
    q = normal(1, 1, n_q, dim, dtype=dtype, seed=16).expand(batch, 1, n_q, dim)
    k, v = (normal(1, 1, n_k, dim, dtype=dtype, seed=s) for s in (17, 18))
    clean = v.clone()
    v[0, 0, -1] = float("nan")
    visible = window_visible(n_q, n_k, n_k, 0, n_k).cuda()
    want, off = attend(q[0, 0], k[0, 0], clean[0, 0], visible, dim**-0.5, dtype)
    got = window_stall(q, k.expand(batch, 1, n_k, dim), v.expand(batch, 1, n_k, dim), n_k, 1_000_000, -1)
    assert torch.equal(got[1:, :, :-1], got[:1, :, :-1].expand_as(got[1:, :, :-1])) and got[:, :, -1].isnan().all()
    check(got[0, 0, :-1], want[:-1], off[:-1])
    code = C.c_int32(0)
    _cabi.check(_cabi.lib().pk_poll_device_fault(0, C.byref(code)))
    assert code.value == 0


@pytest.mark.parametrize("dim,dtype,store", [(64, F16, F16), (128, BF16, BF16), (128, F16, torch.int8), (64, BF16, torch.int8)])
@pytest.mark.parametrize("tokens", [1, 16, 100])
def test_pages_of_256_rows(dim, dtype, store, tokens):
    """The largest pages: longer than a key tile."""
    n = 500 + tokens
    cache = pk.PageCache(2, 6, 256, 2, dim, dtype=store, max_length=n)
    rows = normal(2, 2, 2, n, dim, dtype=dtype, seed=19)
    cache.extend(ints([n, n]))
    cache.write(rows[0], rows[1], layer=0)
    cache.starts.fill_(500)
    q = normal(2, 4, tokens, dim, dtype=dtype, seed=20)
    k, v = cache.read(ints([0, 0]), n, layer=0)
    step = float(cache.value_scales.max()) * 127 if store is torch.int8 else 0.0
    for window, sinks in ((None, 0), (200, 5)):
        got = pk.cache_attention(q, cache, window=window, sinks=sinks)
        visible = window_visible(tokens, n, window or n, sinks, n).cuda()
        for b in range(2):
            for h in range(4):
                want, off = attend(q[b, h], k[b, h // 2], v[b, h // 2], visible, dim**-0.5, dtype, step)
                check(got[b, h], want, off, f"sequence {b} head {h}")
