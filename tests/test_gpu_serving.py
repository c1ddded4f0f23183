"""Sliding-window attention, attention over a paged cache and the cache's page work on a B200, against
plain evaluations in 64 bits (tests/_serving.py says how far off a result may be, and why)."""

import itertools
import random

import pytest
import torch

import piper_kernels_b200 as pk
from _serving import ListCache, attend, check, tree_visible, window_visible

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def normal(*shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def check_window(q, k, v, *, window, sinks=0, lengths=None, scale=None, got=None):
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if got is None:
        got = pk.window_attention(q, k, v, window=window, sinks=sinks, lengths=lens, scale=scale)
    group = q.shape[1] // k.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for b in range(q.shape[0]):
        n = k.shape[2] if lengths is None else min(max(lengths[b], 0), k.shape[2])
        visible = window_visible(q.shape[2], k.shape[2], window, sinks, n).cuda()
        for h in range(q.shape[1]):
            want, off = attend(q[b, h], torch.nan_to_num(k[b, h // group]) if lengths else k[b, h // group],
                               torch.nan_to_num(v[b, h // group]) if lengths else v[b, h // group], visible, scale, q.dtype)
            check(got[b, h], want, off, f"batch {b} head {h}")
            assert not got[b, h][~visible.any(-1)].any()
    return got


@pytest.mark.parametrize("dim,dtype", [(64, F16), (64, BF16), (128, F16), (128, BF16)])
@pytest.mark.parametrize("q_len,kv_len,window,sinks", [
    (1, 1, 1, 0), (1, 700, 64, 4), (3, 65, 7, 2), (64, 64, 64, 0), (65, 65, 1, 0), (129, 300, 128, 130), (257, 257, 1000, 3), (200, 17, 5, 1),
])
def test_window_sizes(dim, dtype, q_len, kv_len, window, sinks):
    q = normal(2, 4, q_len, dim, dtype=dtype, seed=1)
    k, v = (normal(2, 2, kv_len, dim, dtype=dtype, seed=s) for s in (2, 3))
    check_window(q, k, v, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,q_len", [(1, 1, 700), (8, 1, 300), (5, 1, 37), (6, 3, 2), (24, 8, 5), (40, 8, 13)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_window_head_groups(heads, kv_heads, q_len, dtype):
    q = normal(1, heads, q_len, 128, dtype=dtype, seed=4)
    k, v = (normal(1, kv_heads, 701, 128, dtype=dtype, seed=s) for s in (5, 6))
    check_window(q, k, v, window=130, sinks=5)


@pytest.mark.parametrize("q_len", [1, 40, 300])
def test_window_ragged_batch_ignores_what_is_behind_the_lengths(q_len):
    q = normal(5, 2, q_len, 64, dtype=BF16, seed=7)
    k, v = (normal(5, 2, 300, 64, dtype=BF16, seed=s) for s in (8, 9))
    lengths = [300, 0, 1, 299, 400]
    for b, n in enumerate(lengths):
        k[b, :, min(n, 300):] = float("nan")
        v[b, :, min(n, 300):] = float("inf")
    check_window(q, k, v, window=50, sinks=2, lengths=lengths)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q_len", [9, 300])
def test_window_values_that_are_not_finite_reach_only_the_rows_that_see_them(dtype, q_len):
    q = normal(1, 2, q_len, 128, dtype=dtype, seed=10)
    k, v = (normal(1, 2, 300, 128, dtype=dtype, seed=s) for s in (11, 12))
    k[0, 0, 150] = float("nan")
    v[0, 0, 200, 3] = float("inf")
    v[0, 1, 299] = float("nan")
    got = pk.window_attention(q, k, v, window=20)
    clean_k, clean_v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    clean = check_window(q, clean_k, clean_v, window=20)
    p = torch.arange(q_len, device="cuda") + 300 - q_len
    nan0 = (p >= 150) & (p < 170)
    inf0 = (p >= 200) & (p < 220)
    assert got[0, 0][nan0].isnan().all()
    assert (got[0, 0, inf0, 3] == float("inf")).all()
    assert got[0, 1, -1].isnan().all()
    fine = ~(nan0 | inf0)
    visible = window_visible(q_len, 300, 20, 0, 300).cuda()
    for h, rows in ((0, fine), (1, p < 299)):
        want, off = attend(q[0, h], clean_k[0, h], clean_v[0, h], visible, 128**-0.5, dtype)
        check(got[0, h][rows], want[rows], off[rows])
    cols = [c for c in range(128) if c != 3]
    want, off = attend(q[0, 0], clean_k[0, 0], clean_v[0, 0], visible, 128**-0.5, dtype)
    check(got[0, 0][inf0][:, cols], want[inf0][:, cols], off[inf0][:, cols])
    assert clean.isfinite().all()


def test_window_strides():
    """Interleaved, sliced, transposed, expanded and odd-offset views give what their copies give."""
    def same(q, k, v, **kw):
        a = pk.window_attention(q, k, v, window=33, sinks=2, **kw)
        b = pk.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), window=33, sinks=2, **kw)
        assert a.is_contiguous() and torch.equal(a, b)
        check_window(q, k, v, window=33, sinks=2, got=a)

    for n in (5, 200):
        kv = normal(2, 200, 2, 2, 64, dtype=F16, seed=13)  # [batch, key, k/v, head, dim]
        q = normal(2, n, 4, 64, dtype=F16, seed=14).transpose(1, 2)
        same(q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2))
        wide = normal(2, 2, 200, 200, dtype=F16, seed=15)
        same(q, wide[..., 8:72], wide[..., 120:184])
        same(q, wide[..., 1:65], wide[..., 3:67])  # not on 16 bytes
        odd = normal(2, 2, 200 * 67, dtype=F16, seed=16).view(2, 2, 200, 67)[..., :64]
        same(odd[:, :, :n], odd, odd)
        one = normal(1, 1, 200, 64, dtype=F16, seed=17)
        same(q, one.expand(2, 2, 200, 64), one.expand(2, 2, 200, 64))
        same(q, kv[:, :1, 0].transpose(1, 2).expand(2, 2, 200, 64), kv[:, :1, 1].transpose(1, 2).expand(2, 2, 200, 64))


def check_some(q, k, v, got, heads, **kw):
    """A few heads of a call with many."""
    group = q.shape[1] // k.shape[1]
    for b, h in heads:
        one = slice(b, b + 1)
        check_window(q[one, h:h + 1], k[one, h // group:h // group + 1], v[one, h // group:h // group + 1], got=got[one, h:h + 1], **kw)


@pytest.mark.parametrize("batch,heads,kv_heads,q_len,kv_len", [
    (10, 32, 16, 100, 333),   # more units of 256 rows than SMs: whole rounds, the rest shared
    (40, 32, 16, 80, 200),    # several rounds, none shared
    (1, 2, 2, 3000, 3000),    # few units with many keys: all shared
    (3, 7, 1, 333, 900),      # units that end inside a token's heads
])
@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, F16)])
def test_window_units_over_the_sms(batch, heads, kv_heads, q_len, kv_len, dim, dtype):
    q = normal(batch, heads, q_len, dim, dtype=dtype, seed=70)
    k, v = (normal(batch, kv_heads, kv_len, dim, dtype=dtype, seed=s) for s in (71, 72))
    some = [(0, 0), (batch - 1, heads - 1), (batch // 2, heads // 2), (batch // 3, 0)]
    for kw in ({"window": 150, "sinks": 4}, {"window": 5000}):
        check_some(q, k, v, pk.window_attention(q, k, v, **kw), some, **kw)


@pytest.mark.parametrize("q_len", [1, 20, 300])
@pytest.mark.parametrize("dim,dtype", [(128, F16), (64, BF16)])
@pytest.mark.parametrize("jump", [0.02, 0.4, 3.0])
def test_window_scores_that_keep_growing(q_len, dim, dtype, jump):
    """Later keys score higher and higher (or far higher at once), so that the reference exponent of the
    probabilities has to be raised again and again."""
    q = normal(1, 4, q_len, dim, dtype=dtype, seed=73).abs()
    k = (torch.linspace(0, 1, 700, device="cuda")[:, None] ** 2 * jump * 8 + 0.1 * normal(1, 2, 700, dim, dtype=torch.float32, seed=74)).to(dtype)
    k[:, :, 400] += jump * 4
    v = normal(1, 2, 700, dim, dtype=dtype, seed=75)
    check_window(q, k, v, window=1000)
    check_window(q, k.flip(2), v, window=300, sinks=70)


@pytest.mark.parametrize("q_len", [2, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_window_scores_far_below_zero(q_len, dtype):
    """Scores of some -300 and less, alone and beside others: 2^score is zero in 32 bits, the softmax is not."""
    q = normal(1, 2, q_len, 64, dtype=dtype, seed=79).abs() + 1
    k = -(normal(1, 2, 500, 64, dtype=dtype, seed=80).abs() + 1)
    v = normal(1, 2, 500, 64, dtype=dtype, seed=81)
    check_window(q, k, v, window=600, scale=2.0)
    k[:, :, 200:260] *= 0.1
    check_window(q, k, v, window=90, sinks=3, scale=2.0)


def test_calls_from_two_threads():
    from concurrent.futures import ThreadPoolExecutor

    q = normal(2, 4, 300, 64, dtype=F16, seed=76)
    k, v = (normal(2, 2, 300, 64, dtype=F16, seed=s) for s in (77, 78))
    cache = filled(2, 40, 16, 2, 64, F16, [300, 77], [1, 1], seed=30)
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            a = pk.window_attention(q, k, v, window=90)
            b = pk.cache_attention(q[:, :, :1], cache)
            torch.cuda.current_stream().synchronize()
        return a, b

    want = work(0)
    with ThreadPoolExecutor(2) as pool:
        for a, b in pool.map(work, range(20)):
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_window_scale_and_large_scores():
    q = 30 * normal(1, 2, 90, 64, dtype=BF16, seed=18)
    k, v = (normal(1, 2, 90, 64, dtype=BF16, seed=s) for s in (19, 20))
    for scale in (1e-3, 0.7, 4.0):
        check_window(q, 5 * k, v, window=40, scale=scale)


def test_window_head_result_does_not_depend_on_repetition_or_stream():
    q = normal(3, 8, 500, 128, dtype=BF16, seed=21)
    k, v = (normal(3, 2, 500, 128, dtype=BF16, seed=s) for s in (22, 23))
    want = pk.window_attention(q, k, v, window=100, sinks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [pk.window_attention(q, k, v, window=100, sinks=4) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_window_compiles_and_captures():
    q = normal(1, 4, 60, 64, dtype=F16, seed=24)
    k, v = (normal(1, 4, 60, 64, dtype=F16, seed=s) for s in (25, 26))
    want = pk.window_attention(q, k, v, window=9, sinks=1)
    f = torch.compile(lambda a, b, c: pk.window_attention(a, b, c, window=9, sinks=1), fullgraph=True, backend="eager")
    assert torch.equal(f(q, k, v), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pk.window_attention(q, k, v, window=9, sinks=1)
    q.copy_(q.flip(2))
    graph.replay()
    assert torch.equal(out, pk.window_attention(q, k, v, window=9, sinks=1))


# ---------------------------------------------------------------------------------------------------- cache
def filled(batch, pages, page, kv_heads, dim, dtype, lengths, tokens, *, layers=1, seed=0, max_length=None):
    """A cache whose sequences hold ``lengths`` rows, ``tokens[b]`` of them added last, on scattered pages."""
    cache = pk.PageCache(batch, pages, page, kv_heads, dim, layers=layers, dtype=dtype, max_length=max_length or max(lengths + [1]))
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=gen).tolist()
    for b, n in enumerate(lengths):
        for i in range(-(-n // page)):
            p = order.pop()
            cache.table[b, i] = p
            cache.uses[p] = 1
    cache.lengths.copy_(torch.tensor(lengths))
    cache.starts.copy_(torch.tensor([n - t for n, t in zip(lengths, tokens)]))
    shape = tuple(cache.keys.shape)
    if dtype is torch.int8:
        for t in (cache.keys, cache.values):
            t.copy_(torch.randint(-127, 128, shape, generator=gen))
        for t in (cache.key_scales, cache.value_scales):
            t.copy_((0.2 + torch.rand(shape[:-1], generator=gen)) * (3 / 127))
    else:
        for t in (cache.keys, cache.values):
            t.copy_(torch.randn(shape, generator=gen))
    return cache


def rows_of(cache, b, layer, head):
    """All rows of a sequence in 64 bits, from the tensors alone."""
    n = int(cache.lengths[b])
    at = [(int(cache.table[b, j // cache.page_size]), j % cache.page_size) for j in range(n)]
    pages, rows = [p for p, _ in at], [r for _, r in at]
    k, v = (t[layer, pages, head, rows].double() for t in (cache.keys, cache.values))
    if cache.dtype is torch.int8:
        k = k * cache.key_scales[layer, pages, head, rows].double()[:, None]
        v = v * cache.value_scales[layer, pages, head, rows].double()[:, None]
    return k, v


def check_cached(q, cache, *, layer=0, window=None, sinks=0, tree=None, scale=None):
    parents = None if tree is None else torch.tensor(tree, dtype=torch.int32, device="cuda")
    got = pk.cache_attention(q, cache, layer=layer, window=window, sinks=sinks, tree=parents, scale=scale)
    group = q.shape[1] // cache.kv_heads
    step = float(cache.value_scales.max()) * 127 if cache.dtype is torch.int8 else 0.0
    for b in range(cache.batch):
        start, n = int(cache.starts[b]), int(cache.lengths[b])
        up = None if tree is None else tree[b] if isinstance(tree[0], list) else tree
        visible = tree_visible(q.shape[2], start, max(n, start + q.shape[2]), up, window, sinks)[:, :n]
        visible[max(0, n - start):] = False
        visible = visible.cuda()
        for h in range(cache.kv_heads):
            if n == 0:
                assert not got[b].any()
                continue
            k, v = rows_of(cache, b, layer, h)
            for g in range(group):
                want, off = attend(q[b, h * group + g], k, v, visible, q.shape[-1] ** -0.5 if scale is None else scale, q.dtype, step)
                check(got[b, h * group + g], want, off, f"sequence {b} head {h * group + g}")
    return got


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (F16, torch.int8), (BF16, torch.int8)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_cached_single_tokens(dim, dtype, store, page):
    lengths = [1, 2, page, page + 1, 700, 0]
    cache = filled(6, 70, page, 2, dim, store, lengths, [1, 1, 1, 1, 1, 0], seed=page)
    check_cached(normal(6, 8, 1, dim, dtype=dtype, seed=30), cache)
    check_cached(normal(6, 2, 1, dim, dtype=dtype, seed=31), cache, window=65, sinks=3)


@pytest.mark.parametrize("dtype,store", [(F16, F16), (BF16, BF16), (F16, torch.int8), (BF16, torch.int8)])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(4, 4, 1), (7, 1, 3), (16, 1, 1), (32, 2, 1), (6, 2, 9), (8, 1, 64), (3, 3, 100), (2, 1, 200)])
def test_cached_chains(dtype, store, heads, kv_heads, tokens):
    lengths = [tokens, 500 + tokens, 333]
    cache = filled(3, 120, 16, kv_heads, 128, store, lengths, [tokens, tokens, 5], layers=2, seed=tokens)
    q = normal(3, heads, tokens, 128, dtype=dtype, seed=32)
    check_cached(q, cache, layer=1)
    check_cached(q, cache, layer=0, window=40, sinks=5)


def some_tree(tokens, rng):
    return [-1] + [rng.randrange(max(0, t - 6), t) for t in range(1, tokens)]


@pytest.mark.parametrize("dim,dtype,store", [(128, BF16, BF16), (64, F16, F16), (128, F16, torch.int8), (64, BF16, torch.int8)])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 2, 2), (2, 4, 2), (16, 4, 1), (33, 4, 2), (63, 8, 2), (64, 2, 1)])
def test_cached_trees(dim, dtype, store, tokens, heads, kv_heads):
    rng = random.Random(tokens)
    lengths = [tokens, 130 + tokens, 600, 64 + tokens // 2]
    cache = filled(4, 70, 32, kv_heads, dim, store, lengths, [tokens, tokens, tokens, tokens // 2], seed=tokens)
    q = normal(4, heads, tokens, dim, dtype=dtype, seed=33)
    trees = [some_tree(tokens, rng), [t - 1 for t in range(tokens)], [-1] * tokens, some_tree(tokens, rng)]
    check_cached(q, cache, tree=trees)
    check_cached(q, cache, tree=trees, window=5, sinks=2)
    check_cached(q, cache, tree=some_tree(tokens, rng), window=200)


def test_cached_large_trees_of_many_sequences():
    """64 tokens of 8 heads per key head (512 rows: two units), lengths from the tree alone to long contexts."""
    rng = random.Random(3)
    lengths = [64, 1500, 300, 64 + 128, 70]
    cache = filled(5, 160, 16, 2, 128, F16, lengths, [64, 64, 64, 64, 20], seed=32)
    q = normal(5, 16, 64, 128, dtype=F16, seed=59)
    trees = [some_tree(64, rng) for _ in range(5)]
    check_cached(q, cache, tree=trees)
    check_cached(q, cache, tree=trees, window=17, sinks=30)


def test_cached_tree_that_is_a_chain_is_the_chain():
    cache = filled(2, 40, 16, 2, 64, F16, [300, 77], [20, 20], seed=3)
    q = normal(2, 8, 20, 64, dtype=F16, seed=34)
    chain = torch.arange(-1, 19, dtype=torch.int32, device="cuda")
    for kw in ({}, {"window": 30, "sinks": 4}):
        assert torch.equal(pk.cache_attention(q, cache, **kw), pk.cache_attention(q, cache, tree=chain, **kw))


def test_cached_tree_parents_that_are_none():
    """Parents outside [-1, t) count as -1, cycles among them."""
    cache = filled(1, 10, 16, 1, 64, F16, [40], [4], seed=4)
    q = normal(1, 1, 4, 64, dtype=F16, seed=35)
    tree = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    want = pk.cache_attention(q, cache, tree=tree([-1, -1, 1, -1]))
    for bad in ([0, 1, 1, 3], [-7, 2, 1, 2**31 - 1], [3, -2**31, 1, 64]):
        assert torch.equal(pk.cache_attention(q, cache, tree=tree(bad)), want)


def test_cached_pages_that_are_not_there_are_not_seen():
    cache = filled(2, 40, 16, 2, 128, BF16, [200, 300], [3, 3], seed=5)
    eight = filled(2, 40, 16, 2, 128, torch.int8, [200, 300], [3, 3], seed=5)
    q = normal(2, 4, 3, 128, dtype=BF16, seed=36)
    for c in (cache, eight):
        kept = c.table.clone()
        c.table[0, 2], c.table[1, 7], c.table[1, 18] = -1, 40, 2**31 - 1
        seen = pk.cache_attention(q, c)
        holes = {0: list(range(32, 48)), 1: list(range(112, 128)) + list(range(288, 300))}
        c.table.copy_(kept)  # the oracle reads the rows, and leaves the holes out
        group = q.shape[1] // c.kv_heads
        for b in range(2):
            n, start = int(c.lengths[b]), int(c.starts[b])
            visible = tree_visible(3, start, n, None, None, 0)
            visible[:, holes[b]] = False
            for h in range(2):
                kk, vv = rows_of(c, b, 0, h)
                for g in range(group):
                    want, off = attend(q[b, h * group + g], kk, vv, visible.cuda(), 128**-0.5, BF16, 3.6)
                    check(seen[b, h * group + g], want, off)


def test_cached_rows_left_behind_by_others_are_not_seen():
    for store in (F16, torch.int8):
        cache = filled(2, 12, 32, 1, 64, store, [40, 33], [1, 1], seed=6)
        clean = check_cached(normal(2, 4, 1, 64, dtype=F16, seed=37), cache)
        owned = torch.zeros(12, 32, dtype=torch.bool, device="cuda")
        for b in range(2):
            for j in range(int(cache.lengths[b])):
                owned[cache.table[b, j // 32], j % 32] = True
        for t in (cache.keys, cache.values) if store is F16 else (cache.key_scales, cache.value_scales):
            t[0, :, 0][~owned] = float("nan")
        assert torch.equal(pk.cache_attention(normal(2, 4, 1, 64, dtype=F16, seed=37), cache), clean)


def test_cached_nan_in_one_branch_stays_in_it():
    cache = filled(1, 10, 16, 1, 128, BF16, [70], [6], seed=7)
    q = normal(1, 2, 6, 128, dtype=BF16, seed=38)
    tree = [-1, 0, 0, 1, 2, 3]
    want = check_cached(q, cache, tree=tree)
    j = 64 + 2
    cache.values[0, cache.table[0, j // 16], 0, j % 16] = float("nan")
    got = pk.cache_attention(q, cache, tree=torch.tensor(tree, dtype=torch.int32, device="cuda"))
    hit = torch.tensor([False, False, True, False, True, False], device="cuda")
    assert got[0, :, hit].isnan().all() and not got[0, :, ~hit].isnan().any()
    off = torch.finfo(BF16).eps * 2
    assert ((got - want)[0, :, ~hit].abs() <= off * want[0, :, ~hit].abs() + 1e-3).all()


def test_cached_zero_scale_rows_count_with_their_weight():
    cache = filled(1, 4, 16, 1, 64, torch.int8, [33], [1], seed=8)
    cache.value_scales[0, cache.table[0, 0], 0, 3] = 0.0
    cache.values[0, cache.table[0, 0], 0, 3] = 77
    cache.key_scales[0, cache.table[0, 1], 0, 5] = 0.0
    check_cached(normal(1, 2, 1, 64, dtype=F16, seed=39), cache)
    cache.value_scales.zero_()
    assert not pk.cache_attention(normal(1, 2, 1, 64, dtype=F16, seed=39), cache).any()


@pytest.mark.parametrize("least,most", [(1e-6, 1e2)])
def test_cached_scales_of_many_sizes(least, most):
    cache = filled(1, 20, 16, 1, 128, torch.int8, [300], [1], seed=9)
    gen = torch.Generator().manual_seed(1)
    spread = torch.exp(torch.rand(cache.value_scales.shape, generator=gen) * torch.log(torch.tensor(most / least))) * least
    cache.value_scales.copy_(spread)
    check_cached(normal(1, 4, 1, 128, dtype=BF16, seed=40), cache)


def test_cached_strided_queries():
    cache = filled(2, 20, 16, 2, 64, F16, [100, 90], [5, 5], seed=10)
    q = normal(2, 5, 4, 67, dtype=F16, seed=41)
    for view in (q[..., :64].transpose(1, 2), q[..., 3:].transpose(1, 2), q[:1, :, :, :64].transpose(1, 2).expand(2, 4, 5, 64)):
        assert torch.equal(pk.cache_attention(view, cache), pk.cache_attention(view.contiguous(), cache))
    check_cached(q[..., 3:].transpose(1, 2), cache)


def test_cached_one_long_sequence_beside_short_ones():
    cache = filled(5, 700, 64, 2, 128, BF16, [40000, 1, 64, 65, 300], [1] * 5, seed=11)
    q = normal(5, 8, 1, 128, dtype=BF16, seed=42)
    check_cached(q, cache)
    check_cached(q, cache, window=4096, sinks=4)


@pytest.mark.parametrize("dim,dtype,store", [(128, BF16, BF16), (64, F16, torch.int8)])
@pytest.mark.parametrize("batch,heads,kv_heads,tokens", [(3, 8, 2, 1), (3, 3, 3, 20), (3, 4, 2, 32), (40, 8, 8, 1), (60, 3, 3, 2)])
@pytest.mark.parametrize("room", [None, 40000])
def test_cached_units_of_one_cluster_and_shared_by_all(dim, dtype, store, batch, heads, kv_heads, tokens, room):
    """The same sequences where each could be long (tiles are shared by all CTAs) and where none is (clusters of
    16 to one CTAs, by the number of sequences), chains and trees."""
    rng = random.Random(batch + tokens)
    lengths = [(tokens, 1500, 700)[b % 3] if batch < 4 else tokens + rng.randrange(200) for b in range(batch)]
    cache = filled(batch, sum(-(-n // 16) for n in lengths), 16, kv_heads, dim, store, lengths, [tokens] * batch, seed=tokens, max_length=room)
    q = normal(batch, heads, tokens, dim, dtype=dtype, seed=83)
    check_cached(q, cache)
    check_cached(q, cache, window=130, sinks=9)
    check_cached(q, cache, tree=some_tree(tokens, rng))


@pytest.mark.parametrize("store", [F16, torch.int8])
@pytest.mark.parametrize("room", [None, 40000])
def test_cached_rows_that_are_not_finite_in_pieces(store, room):
    """A row that one token of a tree sees and others do not, in one of many pieces of a sequence."""
    cache = filled(2, 200, 16, 2, 64, store, [1400, 33], [3, 3], seed=5, max_length=room)
    q = normal(2, 6, 3, 64, dtype=F16, seed=84)
    tree = [-1, 0, 0]
    want = check_cached(q, cache, tree=tree)
    values = cache.value_scales if store is torch.int8 else cache.values
    values[0, cache.table[0, 1399 // 16], :, 1399 % 16] = float("nan")
    got = pk.cache_attention(q, cache, tree=torch.tensor(tree, dtype=torch.int32, device="cuda"))
    assert got[0, :, 2].isnan().all() and torch.equal(got[1], want[1]) and not got[0, :, :2].isnan().any()
    off = torch.finfo(F16).eps * 2
    assert ((got - want)[0, :, :2].abs() <= off * want[0, :, :2].abs() + 1e-3).all()


def test_cached_many_sequences():
    lengths = [1 + 7 * i % 90 for i in range(500)]
    cache = filled(500, 4000, 16, 1, 64, F16, lengths, [1] * 500, seed=12)
    q = normal(500, 2, 1, 64, dtype=F16, seed=43)
    got = pk.cache_attention(q, cache)
    for b in range(0, 500, 37):
        k, v = rows_of(cache, b, 0, 0)
        for h in range(2):
            want, off = attend(q[b, h], k, v, torch.ones(1, lengths[b], dtype=torch.bool, device="cuda"), 0.125, F16)
            check(got[b, h], want, off)


def test_cached_far_pages():
    """Offsets in the pool pass 2^32 elements."""
    pages = 2**32 // (64 * 8 * 64) + 40
    free, _ = torch.cuda.mem_get_info()
    if free < 2 * 2 * pages * 64 * 8 * 64 + 2**31:
        pytest.skip("not enough memory")
    keys, values = (torch.empty(1, pages, 8, 64, 64, dtype=F16, device="cuda") for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(pages - 3, pages, dtype=torch.int32, device="cuda").flip(0).view(1, 3).contiguous()
    cache = pk.PageCache.from_tensors(keys, values, table, ints(0), ints(0), torch.zeros(pages, dtype=torch.int32, device="cuda"))
    cache.lengths.fill_(150)
    rows = normal(2, 1, 8, 150, 64, dtype=F16, seed=44)
    cache.write(rows[0], rows[1], layer=0)
    cache.starts.fill_(149)
    check_cached(normal(1, 8, 1, 64, dtype=F16, seed=45), cache)
    k, v = cache.read(ints(0), 150, layer=0)
    assert torch.equal(k, rows[0]) and torch.equal(v, rows[1])


def test_cached_graph_replays_with_new_lengths():
    cache = filled(3, 60, 16, 2, 64, F16, [100, 60, 10], [1, 1, 1], seed=13, max_length=200)
    q = normal(3, 4, 1, 64, dtype=F16, seed=46)
    k, v = (normal(3, 2, 1, 64, dtype=F16, seed=s) for s in (47, 48))
    ones = torch.ones(3, dtype=torch.int32, device="cuda")
    pk.cache_attention(q, cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(ones)
        cache.write(k, v, layer=0)
        out = pk.cache_attention(q, cache)
    for _ in range(40):
        graph.replay()
    assert cache.lengths.tolist() == [140, 100, 50]
    assert torch.equal(out, check_cached(q, cache))


# ---------------------------------------------------------------------------------------------------- page work
def state(cache):
    return [cache.table.tolist(), cache.lengths.tolist(), cache.starts.tolist(), cache.uses.tolist(), cache.refused.tolist()]


def listed(model):
    return [model.table(), model.length, model.start, model.uses(), model.refused]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("batch,pages,page,width,seed", [(1, 5, 16, 5, 0), (4, 30, 16, 9, 1), (7, 40, 32, 6, 2), (33, 200, 16, 12, 3), (6, 9, 16, 20, 4)])
def test_page_work_follows_the_lists(batch, pages, page, width, seed):
    """Random runs of all operations against the list model: table, lengths, uses, refusals, and every row
    against a dictionary of what was written."""
    rng = random.Random(seed)
    layers, heads, dim = 2, 2, 64
    cache = pk.PageCache(batch, pages, page, heads, dim, layers=layers, dtype=F16, max_length=width * page)
    model = ListCache(batch, pages, page, width)
    rows = [[] for _ in range(batch)]  # token tags of each sequence
    tag = 0
    gen = torch.Generator(device="cuda").manual_seed(seed)
    memory = {}
    for step in range(40):
        what = rng.choice(["extend", "extend", "extend", "compact", "fork", "truncate"])
        if what in ("extend", "compact"):
            counts = [rng.choice([0, 0, 1, 1, 2, 5, page, 3 * page + 1, -3]) for _ in range(batch)]
            model.extend(counts)
            cache.extend(ints(counts))
            assert state(cache) == listed(model), f"step {step} extend"
            most = max(1, *(max(c, 0) for c in counts))
            data = torch.randn(2, layers, batch, heads, most, dim, generator=gen, device="cuda").to(F16)
            if step % 2:
                cache.write(data[0], data[1])
            else:
                for layer in range(layers):
                    cache.write(data[0, layer], data[1, layer], layer=layer)
            for b in range(batch):
                for t in range(model.length[b] - model.start[b]):
                    memory[tag] = (data, b, t)
                    rows[b].append(tag)
                    tag += 1
        if what == "compact":
            added = [model.length[b] - model.start[b] for b in range(batch)]
            keep = [rng.randrange(0, a + 1) for a in added]
            width_ = max(1, *added)
            paths = [sorted(rng.sample(range(a), n)) + [-9] * (width_ - n) for a, n in zip(added, keep)]
            if rng.random() < 0.3 and keep[0] > 1:
                paths[0][0], paths[0][1] = paths[0][1], paths[0][0]
            start = list(model.start)
            model.compact(paths, keep)
            cache.compact(ints(paths), ints(keep))
            for b in range(batch):
                if not model.refused[b]:
                    rows[b] = rows[b][: start[b]] + [rows[b][start[b] + i] for i in paths[b][: keep[b]]]
        elif what == "fork":
            parents = [rng.choice([b, b, rng.randrange(batch), -1, batch]) for b in range(batch)]
            model.fork(parents)
            cache.fork(ints(parents))
            rows = [list(rows[b if p >= batch else p]) if p >= 0 else [] for b, p in enumerate(parents)]
        elif what == "truncate":
            lengths = [rng.choice([0, -1, 3, page, model.length[b], model.length[b] + 4, model.length[b] // 2]) for b in range(batch)]
            model.truncate(lengths)
            cache.truncate(ints(lengths))
            rows = [r[: max(n, 0)] for r, n in zip(rows, lengths)]
        assert state(cache) == listed(model), f"step {step} {what}"
        longest = max(1, *model.length)
        k, v = cache.read(ints([0] * batch), longest)
        for b in range(batch):
            assert len(rows[b]) == model.length[b]
            for j in set(rows[b]) and [0, len(rows[b]) // 2, len(rows[b]) - 1]:
                data, sb, t = memory[rows[b][j]]
                assert torch.equal(k[:, b, :, j], data[0, :, sb, :, t]) and torch.equal(v[:, b, :, j], data[1, :, sb, :, t]), (step, b, j)
            assert not k[:, b, :, len(rows[b]):].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (64, 70), (128, 33), (128, 300)])
def test_eight_bit_rows(dtype, dim, tokens):
    cache = pk.PageCache(2, 60, 16, 3, dim, dtype=torch.int8, layers=2)
    counts = [tokens, max(0, tokens - 2)]
    cache.extend(ints(counts))
    key, value = (5 * normal(2, 2, 3, tokens, dim, dtype=dtype, seed=s) for s in (50, 51))
    key[0, 0, 0, 0] = 0
    cache.write(key, value)
    got = cache.read(ints([0, 0]), tokens + 1)
    for x, y, codes, scales in ((key, got[0], cache.keys, cache.key_scales), (value, got[1], cache.values, cache.value_scales)):
        x = x.float()
        scale = x.abs().amax(-1) / torch.full((), 127.0, device="cuda") + 1e-7
        want = (x / scale[..., None]).round()  # the same operations in the same order: equal bit for bit
        for b in range(2):
            for t in range(counts[b]):
                p, r = int(cache.table[b, t // 16]), t % 16
                assert torch.equal(codes[:, p, :, r].float(), want[:, b, :, t])
                assert torch.equal(scales[:, p, :, r], scale[:, b, :, t])
            assert torch.equal(y[:, b, :, : counts[b]], want[:, b, :, : counts[b]] * scale[:, b, :, : counts[b], None])
            assert not y[:, b, :, counts[b]:].any()
    for out in (F16, BF16):
        half = cache.read(ints([0, 0]), tokens + 1, layer=1, dtype=out)
        assert torch.equal(half[0], got[0][1].to(out)) and torch.equal(half[1], got[1][1].to(out))


def test_eight_bit_rows_that_are_not_finite():
    cache = pk.PageCache(1, 4, 16, 1, 64, dtype=torch.int8)
    cache.extend(ints([4]))
    rows = normal(1, 1, 1, 4, 64, dtype=BF16, seed=52)
    rows[..., 1, 5], rows[..., 2, 63] = float("nan"), float("-inf")
    cache.write(rows, rows)
    k, v = cache.read(ints([0]), 4)
    for x in (k, v):
        assert x[..., 1:3, :].isnan().all() and x[..., 0, :].isfinite().all() and x[..., 3, :].isfinite().all()


def test_write_takes_strided_rows_and_leaves_the_rest():
    for store in (BF16, torch.int8):
        cache = filled(2, 20, 16, 2, 64, store, [20, 31], [0, 0], layers=2, seed=14, max_length=100)
        cache.extend(ints([3, 0]))
        before = [t.clone() for t in (cache.keys, cache.values)]
        rows = normal(2, 5, 2, 67, dtype=BF16, seed=53)
        for view in (rows[..., :64].transpose(1, 2), rows[..., 3:].transpose(1, 2)):
            cache.write(view, view, layer=1)
            k, v = cache.read(cache.starts, 3, layer=1)
            other = cache.read(cache.starts, 3, layer=1)
            assert torch.equal(k, other[0])
            cache.write(view.contiguous(), view.contiguous(), layer=1)
            again = cache.read(cache.starts, 3, layer=1)
            assert torch.equal(k, again[0]) and torch.equal(v, again[1])
        changed = (cache.keys != before[0]).any(-1).any(2)  # [layers, pages, rows]
        allowed = torch.zeros_like(changed)
        for t in range(20, 23):
            allowed[1, cache.table[0, t // 16], t % 16] = True
        assert not (changed & ~allowed).any()


def test_write_with_fewer_rows_than_were_added_leaves_the_others():
    cache = pk.PageCache(2, 10, 16, 1, 64, dtype=F16)
    cache.keys.fill_(7)
    cache.extend(ints([20, 3]))
    rows = normal(2, 1, 5, 64, dtype=F16, seed=55)
    cache.write(rows, rows, layer=0)
    k, _ = cache.read(ints([0, 0]), 20, layer=0)
    assert torch.equal(k[0, :, :5], rows[0]) and (k[0, :, 5:] == 7).all()
    assert torch.equal(k[1, :, :3], rows[1, :, :3]) and not k[1, :, 3:].any()


def test_step_is_captured_and_replayed():
    """A whole speculative step in one graph: room, rows, attention of the tree, the accepted path."""
    cache = filled(2, 60, 16, 2, 64, BF16, [100, 33], [0, 0], seed=31, max_length=400)
    eager = pk.PageCache.from_tensors(*(getattr(cache, n).clone() for n in ("keys", "values", "table", "lengths", "starts", "uses")))
    q, k, v = (normal(2, h, 6, 64, dtype=BF16, seed=s) for h, s in ((4, 56), (2, 57), (2, 58)))
    tree, counts = ints([-1, 0, 0, 1, 1, 3]), ints([6, 4])
    paths, keep = ints([[0, 1, 3, 5], [0, 2, 0, 0]]), ints([4, 2])

    def step(c):
        c.extend(counts)
        c.write(k, v, layer=0)
        out = pk.cache_attention(q, c, tree=tree)
        c.compact(paths, keep)
        return out

    kept = [t.clone() for t in (cache.keys, cache.values, cache.table, cache.lengths, cache.starts, cache.uses)]
    step(cache)
    for t, old in zip((cache.keys, cache.values, cache.table, cache.lengths, cache.starts, cache.uses), kept):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for _ in range(5):
        k.add_(1)
        graph.replay()
        assert torch.equal(out, step(eager)) and state(cache) == state(eager)
        assert torch.equal(cache.keys, eager.keys) and torch.equal(cache.values, eager.values)


def test_read_outside_a_sequence_is_zero():
    cache = filled(2, 10, 16, 1, 64, F16, [20, 5], [0, 0], seed=15, max_length=40)
    k, v = cache.read(ints([-3, 2**31 - 2]), 30, layer=0)
    assert not k[0, :, :3].any() and k[0, :, 3:23].any() and not k[0, :, 23:].any() and not k[1].any() and not v[1].any()


def test_samples_of_one_prompt_grow_apart():
    """fork, extend, write, attend, drop: eight samples of a prompt, each with its own continuation."""
    cache = pk.PageCache(8, 40, 16, 2, 64, layers=1, dtype=BF16, max_length=100)
    cache.extend(ints([41] + [0] * 7))
    prompt = normal(2, 8, 2, 41, 64, dtype=BF16, seed=54)
    cache.write(prompt[0], prompt[1], layer=0)
    cache.fork(ints([0] * 8))
    assert int(cache.uses.sum()) == 24 and int((cache.uses > 0).sum()) == 3
    for step in range(20):
        cache.extend(ints([1] * 8))
        rows = normal(2, 8, 2, 1, 64, dtype=BF16, seed=100 + step)
        cache.write(rows[0], rows[1], layer=0)
        if step % 5 == 0:
            check_cached(normal(8, 4, 1, 64, dtype=BF16, seed=200 + step), cache)
    assert cache.lengths.tolist() == [61] * 8 and not cache.refused.any()
    k, _ = cache.read(ints([0] * 8), 41, layer=0)
    assert all(torch.equal(k[b], prompt[0, 0]) for b in range(8))
    cache.fork(ints([3, 3] + [-1] * 6))
    assert int((cache.uses > 0).sum()) == 4
    cache.truncate(ints([0] * 8))
    assert not cache.uses.any() and (cache.table == -1).all()


def test_prompt_then_drafts():
    """The operators together: a windowed prompt, its rows into the cache, then drafted trees of which a path
    is kept; each token's attention equals that of the whole sequence so far."""
    dim, heads, kv_heads, window, sinks = 128, 4, 2, 48, 3
    cache = pk.PageCache(1, 20, 16, kv_heads, dim, dtype=F16, max_length=256)
    n = 90
    q, k, v = normal(1, heads, 200, dim, dtype=F16, seed=60), normal(1, kv_heads, 200, dim, dtype=F16, seed=61), normal(1, kv_heads, 200, dim, dtype=F16, seed=62)
    pk.window_attention(q[:, :, :n], k[:, :, :n], v[:, :, :n], window=window, sinks=sinks)
    cache.extend(ints([n]))
    cache.write(k[:, :, :n], v[:, :, :n], layer=0)
    rng = random.Random(5)
    while n < 150:
        tokens = 12
        tree = some_tree(tokens, rng)
        path = [tokens - 1]
        while tree[path[-1]] >= 0:
            path.append(tree[path[-1]])
        path.reverse()
        # the path's tokens are the true continuation, the others noise
        rows_k, rows_v, rows_q = (normal(1, h, tokens, dim, dtype=F16, seed=70 + n + i) for i, h in enumerate((kv_heads, kv_heads, heads)))
        for i, t in enumerate(path):
            rows_k[:, :, t], rows_v[:, :, t], rows_q[:, :, t] = k[:, :, n + i], v[:, :, n + i], q[:, :, n + i]
        cache.extend(ints([tokens]))
        cache.write(rows_k, rows_v, layer=0)
        out = pk.cache_attention(rows_q, cache, window=window, sinks=sinks, tree=ints(tree))
        n += len(path)
        whole = window_visible(n, n, window, sinks, n).cuda()
        for h in range(heads):
            want, off = attend(q[0, h, :n], k[0, h // 2, :n], v[0, h // 2, :n], whole, dim**-0.5, F16)
            check(out[0, h, path], want[n - len(path):], off[n - len(path):])
        cache.compact(ints([path]), ints([len(path)]))
        assert cache.lengths.tolist() == [n] and not cache.refused.any()
    got = cache.read(ints([0]), n, layer=0)
    assert torch.equal(got[0][0], k[0, :, :n]) and torch.equal(got[1][0], v[0, :, :n])


def test_page_work_of_a_large_batch():
    batch = 4096
    cache = pk.PageCache(batch, 9000, 16, 1, 64, dtype=F16, max_length=64)
    model = ListCache(batch, 9000, 16, 4)
    rng = random.Random(9)
    for counts in ([rng.choice([0, 5, 16, 17]) for _ in range(batch)], [rng.choice([0, 1, 30]) for _ in range(batch)], [40] * batch):
        model.extend(counts)
        cache.extend(ints(counts))
        assert state(cache) == listed(model)
    parents = [b // 64 * 64 for b in range(batch)]
    model.fork(parents)
    cache.fork(ints(parents))
    assert state(cache) == listed(model)
    model.extend([1] * batch)
    cache.extend(ints([1] * batch))
    assert state(cache) == listed(model)


@pytest.mark.parametrize("store", [F16, torch.int8])
@pytest.mark.parametrize("tokens", [1, 9, 64])
def test_prepared_copy_maps_change_nothing(store, tokens):
    import ctypes as C

    from piper_kernels_b200 import _cabi

    cache = filled(2, 60, 32, 2, 128, store, [300, 64 + tokens], [tokens, tokens], layers=2, seed=33)
    q = normal(2, 8, tokens, 128, dtype=F16, seed=64)
    want = pk.cache_attention(q, cache, layer=1)
    out = torch.empty_like(want)
    c = cache.handle()  # without maps
    assert not c.maps and cache.mapped_handle().maps
    query = _cabi.PkCacheQuery(8, tokens, 1, _cabi.PK_F16, 0, 0, 128**-0.5, q.data_ptr(), q.stride()[:3], None, 0, out.data_ptr(), None, 0)
    n = C.c_uint64()
    _cabi.check(_cabi.lib().pk_cache_attention_workspace_bytes(C.byref(c), C.byref(query), C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    query.workspace, query.workspace_bytes = ws.data_ptr(), n.value
    _cabi.check(_cabi.lib().pk_cache_attention_fwd(C.byref(c), C.byref(query)))
    assert torch.equal(out, want)


def test_two_streams_on_two_caches():
    caches = [filled(4, 100, 16, 2, 64, F16, [300, 20, 100, 7], [1] * 4, seed=20 + i) for i in range(2)]
    q = normal(4, 4, 1, 64, dtype=F16, seed=63)
    want = [pk.cache_attention(q, c) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _, (i, s) in itertools.product(range(10), enumerate(streams)):
        with torch.cuda.stream(s):
            got[i].append(pk.cache_attention(q, caches[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
