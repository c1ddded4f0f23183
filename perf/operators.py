"""What the sliding-window and paged-cache attention operators are measured on.

Three kinds of case: ``window`` (prompt attention over a sliding window with sink tokens), ``cache`` (attention
of single tokens, chains and trees of drafted tokens over a paged cache) and the cache's own page work (``write``,
``step``, ``fork``).  ``run`` computes a case in elementary torch operations in 32 bits, or with the package's
operators where ``own`` is set.
"""

import math

import torch

own = False

HALF, BF16 = "float16", "bfloat16"


def listed():
    return [
        # One short prompt of a small model (8 heads of 64 features, 1024 tokens): latency counts.
        _window("window short prompt", batch=1, heads=8, kv_heads=8, q_len=1024, kv_len=1024, dim=64, dtype=HALF, window=256, sinks=4),
        # A batch of full prompts, four query heads to each key head.
        _window("window prompt batch", batch=4, heads=32, kv_heads=8, q_len=8192, kv_len=8192, dim=128, dtype=HALF, window=1024, sinks=4),
        # A right-padded batch of prompts of odd lengths, window and sinks off every tile border.
        _window("window ragged prompts", batch=2, heads=24, kv_heads=24, q_len=4001, kv_len=4001, dim=128, dtype=BF16, window=511, sinks=3, ragged=True),
        # The last chunk of a long prompt against all of its keys.
        _window("window chunk of a long prompt", batch=1, heads=40, kv_heads=8, q_len=2048, kv_len=32760, dim=128, dtype=BF16, window=4096, sinks=64),
        # One user, one token: nothing but latency.
        _cache("token alone", batch=1, heads=32, kv_heads=8, dim=128, dtype=BF16, length=1000, tokens=1, page=16),
        # A serving batch of single tokens, contexts from short to 8192.
        _cache("token batch", batch=64, heads=32, kv_heads=8, dim=128, dtype=BF16, length=8192, tokens=1, page=64),
        # The same kind of batch on an 8-bit cache with a sliding window and sinks, long contexts.
        _cache("token batch 8-bit window", batch=48, heads=40, kv_heads=8, dim=128, dtype=HALF, length=32760, tokens=1, page=64, eight_bit=True, window=4096, sinks=4),
        # A small draft tree of one user on an 8-bit cache.
        _cache("tree alone", batch=1, heads=24, kv_heads=8, dim=64, dtype=HALF, length=1500, tokens=16, page=16, eight_bit=True, tree=True),
        # Draft trees of a serving batch.
        _cache("tree batch", batch=8, heads=32, kv_heads=8, dim=128, dtype=BF16, length=8192, tokens=63, page=32, tree=True),
        # A batch of prompts is quantised into an 8-bit cache and read back (a hand-over between two workers).
        _pages("write", "write prompts", layers=1, batch=8, kv_heads=8, dim=128, dtype=BF16, length=0, tokens=2047, page=64, eight_bit=True),
        # What a speculative step does to the cache of all layers: drop the last draft, add one, keep the accepted path.
        _pages("step", "draft step", layers=16, batch=32, kv_heads=8, dim=128, dtype=BF16, length=500, tokens=16, page=16),
        # Samples of shared prompts: forked, then each gets room for one token (its own copy of the last page).
        _pages("fork", "fork samples", layers=16, batch=64, kv_heads=8, dim=128, dtype=BF16, length=1000, tokens=1, page=64),
    ]


def draw(rng):
    kind = rng.choice(["window", "window", "cache", "cache", "cache", "write", "step", "fork"])
    dim, dtype = rng.choice([64, 128]), rng.choice([HALF, BF16])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if kind == "window":
        group = rng.choice([1, 2, 4, 5, 8])
        kv_len = _log(rng, 1, 16384)
        q_len = kv_len if rng.random() < 0.6 else _log(rng, 1, kv_len)
        batch = max(1, min(rng.choice([1, 2, 3, 8]), 16384 // kv_len, 131072 // (q_len * kv_heads * group)))
        return _window(None, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, dim=dim, dtype=dtype,
                       window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 7, 64, 130]), ragged=rng.random() < 0.4)
    page, eight_bit = rng.choice([16, 32, 64, 128]), rng.random() < 0.4
    if kind == "cache":
        group = rng.choice([1, 2, 3, 4, 7, 8, 16])
        tokens = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        length = _log(rng, tokens, 32768)
        batch = min(_log(rng, 1, 64), max(1, 131072 // (length * max(1, tokens * group // 64))))
        windowed = rng.random() < 0.4
        return _cache(None, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, length=length, tokens=tokens,
                      page=page, eight_bit=eight_bit, tree=tokens > 1 and rng.random() < 0.7,
                      window=_log(rng, 1, 8192) if windowed else 0, sinks=rng.choice([0, 4, 33]) if windowed else 0)
    tokens = _log(rng, 1, 64) if kind != "write" else _log(rng, 1, 2048)
    return _pages(kind, None, layers=rng.choice([1, 2, 5]), batch=rng.choice([1, 2, 7, 16, 33]) if kind != "write" else rng.choice([1, 3, 8]),
                  kv_heads=kv_heads, dim=dim, dtype=dtype, length=_log(rng, 1, 1000), tokens=tokens, page=page, eight_bit=eight_bit)


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _named(name, case):
    return {"name": name, **case} if name else case


def _window(name, *, batch, heads, kv_heads, q_len, kv_len, dim, dtype, window, sinks, ragged=False):
    return _named(name, dict(kind="window", batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, dim=dim, dtype=dtype,
                             window=window, sinks=sinks, ragged=ragged))


def _cache(name, *, batch, heads, kv_heads, dim, dtype, length, tokens, page, eight_bit=False, tree=False, window=0, sinks=0):
    return _named(name, dict(kind="cache", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, length=length, tokens=tokens,
                             page=page, eight_bit=eight_bit, tree=tree, window=window, sinks=sinks, layers=1))


def _pages(kind, name, *, layers, batch, kv_heads, dim, dtype, length, tokens, page, eight_bit=False):
    return _named(name, dict(kind=kind, layers=layers, batch=batch, kv_heads=kv_heads, dim=dim, dtype=dtype, length=length, tokens=tokens,
                             page=page, eight_bit=eight_bit))


def _spread(most, least, count):
    """``count`` lengths between ``least`` and ``most``, evenly spread, the longest first."""
    return [most - (most - least) * i // count for i in range(count)]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def shuffled(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")[torch.randperm(len(values), generator=gen, device="cuda")]

    c = case
    if c["kind"] == "window":
        s = {"query": normal(c["batch"], c["heads"], c["q_len"], c["dim"]), "key": normal(c["batch"], c["kv_heads"], c["kv_len"], c["dim"]),
             "value": normal(c["batch"], c["kv_heads"], c["kv_len"], c["dim"]), "lengths": None}
        s["key"] += 0.5 * normal(1, c["kv_heads"], 1, c["dim"])  # a channel bias, as the keys of real models have
        if c["ragged"]:
            s["lengths"] = shuffled(_spread(c["kv_len"], (c["kv_len"] + 1) // 2, c["batch"]))
        return {**c, **s}
    batch, page, tokens = c["batch"], c["page"], c["tokens"]
    # `length` counts a context (and, for a cache case, its new tokens); page work leaves room for `tokens` more
    room = c["length"] if c["kind"] == "cache" else c["length"] + tokens
    width = -(-room // page)
    count = batch * width + (batch if c["kind"] == "fork" else 0)
    s = {"table": torch.full((batch, width), -1, dtype=torch.int32, device="cuda"), "uses": torch.zeros(count, dtype=torch.int32, device="cuda")}
    shape = (c["layers"], count, c["kv_heads"], page, c["dim"])
    if c["eight_bit"]:
        s["keys"], s["values"] = (torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8) for _ in range(2))
        s["key_scales"], s["value_scales"] = ((0.5 + torch.rand(shape[:-1], generator=gen, device="cuda")) * (3.0 / 127.0) for _ in range(2))
    else:
        s["keys"], s["values"], s["key_scales"], s["value_scales"] = normal(*shape), normal(*shape), None, None
    if c["kind"] == "cache":
        s["lengths"] = shuffled(_spread(c["length"], min(c["length"], tokens + c["length"] // 8), batch))
        s["starts"] = s["lengths"] - tokens
        s["query"] = normal(batch, c["heads"], tokens, c["dim"])
        s["tree"] = None
        if c["tree"]:  # node 0 is the last token that is certain; each other node hangs under one of the eight before it
            at = torch.arange(tokens, device="cuda").expand(batch, tokens)
            back = torch.randint(1, 9, (batch, tokens), generator=gen, device="cuda")
            s["tree"] = torch.where(at == 0, -1, (at - back).clamp(min=0)).to(torch.int32)
    else:
        s["lengths"] = shuffled(_spread(c["length"], c["length"] // 2, batch))
        s["starts"] = s["lengths"].clone()
        s["base"] = s["lengths"].clone()
        s["counts"] = shuffled(_spread(tokens, (tokens + 1) // 2, batch))
        s["key"], s["value"] = (3.0 * normal(c["layers"], batch, c["kv_heads"], tokens, c["dim"]) for _ in range(2))
        keep = [max(1, n // 3) for n in _spread(tokens, (tokens + 1) // 2, batch)]
        s["keep"] = torch.minimum(shuffled(keep), s["counts"])
        # an accepted path: ascending places in the draft
        order = torch.rand(batch, tokens, generator=gen, device="cuda")
        order = torch.where(torch.arange(tokens, device="cuda") < s["counts"][:, None], order, 2.0).argsort(1)
        chosen = torch.where(torch.arange(tokens, device="cuda") < s["keep"][:, None], order, tokens).sort(1).values
        s["paths"] = chosen.to(torch.int32)
        group = torch.arange(batch, device="cuda", dtype=torch.int32) // 8 * 8  # eight samples to a prompt
        s["parents"] = group
        s["ones"] = torch.ones(batch, dtype=torch.int32, device="cuda")
    # the contexts' pages, scattered over the pool as in a server that has run for a while
    pages = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)[: batch * width].view(batch, width)
    held = torch.arange(width, device="cuda") < -(-s["lengths"] // page)[:, None]
    s["table"] = torch.where(held, pages, -1).to(torch.int32).contiguous()
    s["uses"][pages[held].long()] = 1
    if own:
        from piper_kernels_b200 import PageCache

        names = ("keys", "values", "table", "lengths", "starts", "uses", "key_scales", "value_scales")
        s["cache"] = PageCache.from_tensors(**{n: s[n] for n in names})
    return {**c, **s}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from piper_kernels_b200 import cache_attention, window_attention

    if s["kind"] == "window":
        return window_attention(s["query"], s["key"], s["value"], window=s["window"], sinks=s["sinks"], lengths=s["lengths"])
    cache = s["cache"]
    if s["kind"] == "cache":
        return cache_attention(s["query"], cache, window=s["window"] or None, sinks=s["sinks"], tree=s["tree"])
    cache.truncate(s["base"])
    if s["kind"] == "fork":
        cache.fork(s["parents"])
        cache.extend(s["ones"])
    else:
        cache.extend(s["counts"])
        cache.write(s["key"], s["value"])
    if s["kind"] == "step":
        cache.compact(s["paths"], s["keep"])
    out = {"table": cache.table, "lengths": cache.lengths, "uses": cache.uses}
    if s["kind"] == "write" or cache.key_scales is not None:
        out["keys"], out["values"] = cache.read(*_touched(s), dtype=torch.float32)
    else:
        out["keys"], out["values"] = cache.keys, cache.values
    return out


def _run_plain(s):
    if s["kind"] == "window":
        return _plain_window(s)
    if s["kind"] == "cache":
        return _plain_cache(s)
    _truncate(s, s["base"])
    if s["kind"] == "fork":
        _fork(s)
        _extend(s, s["ones"])
    else:
        _extend(s, s["counts"])
        _write(s)
    if s["kind"] == "step":
        _compact(s)
    out = {n: s[n] for n in ("table", "lengths", "uses")}
    if s["kind"] == "write" or s["key_scales"] is not None:
        out["keys"], out["values"] = _read(s, "keys"), _read(s, "values")
    else:
        out["keys"], out["values"] = s["keys"], s["values"]
    return out


def _touched(s):
    """The first row and the number of rows, in each slot, that a pass of page work may have changed."""
    if s["kind"] == "fork":
        return s["starts"] // s["page"] * s["page"], s["page"]
    return s["base"], s["tokens"]


def _softmax_product(scores, visible, value):
    """Rows of softmax(scores over what is visible) times value; a row that sees nothing is zero."""
    scores = scores.masked_fill_(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    return (weights @ value) / weights.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_window(s):
    """Blocks of query rows against the band of keys that any of them sees, the sinks in front."""
    q, k, v, window, sinks = s["query"], s["key"].float(), s["value"].float(), min(s["window"], s["kv_len"]), min(s["sinks"], s["kv_len"])
    b, h, n_q, d = q.shape
    h_kv, n_k = k.shape[1], k.shape[2]
    block = min(n_q, max(64, 1 << (window - 1).bit_length() - 1))
    blocks = -(-n_q // block)
    rows = torch.arange(blocks * block, device=q.device).view(blocks, block)  # [blocks, block]
    band = (n_k - n_q) + torch.arange(blocks, device=q.device)[:, None] * block + torch.arange(1 - window, block, device=q.device)
    at = torch.cat([torch.arange(sinks, device=q.device).expand(blocks, sinks), band], 1)  # key of each column, [blocks, columns]
    position = rows + (n_k - n_q)
    limit = torch.full((b,), n_k, device=q.device) if s["lengths"] is None else s["lengths"].clamp(0, n_k)
    once = (torch.arange(at.shape[1], device=q.device) < sinks) | (at >= sinks)  # a sink inside the band counts as a sink only
    far = position[:, :, None] - at[:, None, :]
    visible = (far >= 0) & ((far < window) | (at < sinks)[:, None, :]) & (once & (at >= 0))[:, None, :]
    inside = (at[:, None, :] < limit[:, None, None, None]) & (position[:, :, None] < limit[:, None, None, None])
    visible = (visible & inside)[:, None, None]  # [b, 1, 1, blocks, block, columns]
    columns = at.clamp(0, n_k - 1).reshape(-1)
    kb, vb = (t[:, :, columns].view(b, h_kv, 1, blocks, -1, d) for t in (k, v))
    qb = torch.nn.functional.pad(q.float() * d**-0.5, (0, 0, 0, blocks * block - n_q)).view(b, h_kv, h // h_kv, blocks, block, d)
    out = _softmax_product(qb @ kb.transpose(-1, -2), visible, vb)
    return out.reshape(b, h, blocks * block, d)[:, :, :n_q].to(q.dtype)


def _rows_of(s, name):
    """All rows that the table leads to, [batch, kv_heads, width * page, dim] in 32 bits."""
    rows = s[name][0][s["table"].clamp_min(0).long()].float()
    if s[name[:-1] + "_scales"] is not None:
        rows = rows * s[name[:-1] + "_scales"][0][s["table"].clamp_min(0).long()][..., None]
    return rows.transpose(1, 2).flatten(2, 3)


def _plain_cache(s):
    q, tokens, starts, lengths = s["query"], s["tokens"], s["starts"].long(), s["lengths"].long()
    b, h, _, d = q.shape
    k, v = _rows_of(s, "keys"), _rows_of(s, "values")
    h_kv, n = k.shape[1], k.shape[2]
    at, t = torch.arange(n, device=q.device), torch.arange(tokens, device=q.device)
    draft = at - starts[:, None]  # place of each key in the draft, [b, n]
    if s["tree"] is None:
        kin = (t[:, None] >= t).expand(b, tokens, tokens)
    else:
        kin = torch.eye(tokens, device=q.device) + torch.nn.functional.one_hot(s["tree"].long() + 1, tokens + 1)[..., 1:].float()
        kin = torch.linalg.matrix_power(kin, tokens) > 0  # [b, token, itself and those above it]
    depth = kin.sum(-1) - 1
    inside = (draft >= 0) & (draft < tokens)
    place = draft.clamp(0, tokens - 1)
    position = torch.where(inside, starts[:, None] + depth.gather(1, place), at)  # of each key
    visible = torch.where(inside[:, None, :], kin.gather(2, place[:, None, :].expand(b, tokens, n)), (draft < 0)[:, None, :])
    if s["window"]:
        visible &= ((starts[:, None] + depth)[:, :, None] - position[:, None, :] < s["window"]) | (position < s["sinks"])[:, None, :]
    visible &= (at < lengths[:, None])[:, None, :] & (t < (lengths - starts)[:, None])[:, :, None]
    qg = (q.float() * d**-0.5).view(b, h_kv, h // h_kv, tokens, d)
    out = _softmax_product(qg @ k[:, :, None].transpose(-1, -2), visible[:, None, None], torch.where(at[:, None] < lengths[:, None, None, None], v, 0.0)[:, :, None])
    return out.reshape(b, h, tokens, d).to(q.dtype)


def _truncate(s, lengths):
    s["lengths"].copy_(torch.minimum(s["lengths"], lengths.clamp_min(0)))
    s["starts"].copy_(s["lengths"])
    page, table = s["page"], s["table"]
    gone = (torch.arange(table.shape[1], device=table.device) >= -(-s["lengths"] // page)[:, None]) & (table >= 0)
    s["uses"].index_add_(0, table.clamp_min(0).flatten(), -gone.to(torch.int32).flatten())
    table.masked_fill_(gone, -1)


def _extend(s, counts):
    """Room for ``counts`` more tokens: a last page shared with others is copied, but for the first of its owners
    where all of them are extended; new pages are the lowest free ones, slot by slot."""
    table, uses, page, lengths = s["table"], s["uses"], s["page"], s["lengths"]
    old, new = lengths.long(), (lengths + counts).long()
    s["starts"].copy_(lengths)
    lengths.copy_(new)
    b, width = table.shape
    slots = torch.arange(b, device=table.device)
    last = (old // page).clamp(max=width - 1)
    tail = table[slots, last]
    grows = (old % page != 0) & (counts > 0)
    same = (tail[:, None] == tail) & grows
    everyone = same.sum(1) >= uses[tail.clamp_min(0).long()]
    first = same.int().argmax(1) == slots
    copies = grows & (uses[tail.clamp_min(0).long()] > 1) & ~(everyone & first)
    held, wanted = -(-old // page), -(-new // page)
    need = wanted - held + copies
    before = need.cumsum(0) - need
    free = torch.sort((uses != 0).to(torch.int32), stable=True).indices.to(torch.int32)
    columns = torch.arange(width, device=table.device)
    fresh = ((columns >= held[:, None]) & (columns < wanted[:, None])) | (copies[:, None] & (columns == last[:, None]))
    rank = (before[:, None] + fresh.cumsum(1) - 1).clamp(0, uses.numel() - 1)
    uses.index_add_(0, tail.clamp_min(0), -copies.to(torch.int32))
    table.copy_(torch.where(fresh, free[rank], table))
    uses.index_add_(0, table.clamp_min(0).flatten(), fresh.to(torch.int32).flatten())
    source, target, rows = (x[copies].long() for x in (tail, table[slots, last], old % page))
    kept = torch.arange(page, device=table.device) < rows[:, None]  # [copies, page]
    for name in ("keys", "values", "key_scales", "value_scales"):
        if s[name] is not None:
            mask = kept[None, :, None, :, None] if s[name].dim() == 5 else kept[None, :, None, :]
            s[name][:, target] = torch.where(mask, s[name][:, source], s[name][:, target])


def _fork(s):
    table, uses = s["table"], s["uses"]
    parents = s["parents"].long()
    new = table[parents]
    uses.index_add_(0, table.clamp_min(0).flatten(), -(table >= 0).to(torch.int32).flatten())
    uses.index_add_(0, new.clamp_min(0).flatten(), (new >= 0).to(torch.int32).flatten())
    table.copy_(new)
    s["lengths"].copy_(s["lengths"][parents])
    s["starts"].copy_(s["lengths"])


def _places(s, index):
    """Page and row of each token index of each slot."""
    return s["table"].gather(1, (index // s["page"]).clamp(max=s["table"].shape[1] - 1)).long(), index % s["page"]


def _quantise(x):
    scale = x.float().abs().amax(-1) / torch.full((), 127.0, device=x.device) + 1e-7
    return (x.float() / scale[..., None]).round().clamp(-127, 127).to(torch.int8), scale


def _write(s):
    t = torch.arange(s["tokens"], device="cuda")
    valid = t < (s["lengths"] - s["starts"])[:, None]
    page, row = _places(s, (s["starts"][:, None] + t).long())
    page, row = page[valid], row[valid]
    for name in ("key", "value"):
        rows = s[name].transpose(2, 3)[:, valid].transpose(0, 1)  # [rows, layers, heads, dim]
        if s["key_scales"] is not None:
            rows, scales = _quantise(rows)
            s[name + "_scales"][:, page, :, row] = scales
        s[name + "s"][:, page, :, row] = rows


def _read(s, name):
    first, count = _touched(s)
    index = (first[:, None] + torch.arange(count, device="cuda")).long()
    page, row = _places(s, index)
    rows = s[name][:, page.clamp_min(0), :, row].float()  # [batch, rows, layers, heads, dim]
    if s["key_scales"] is not None:
        rows = rows * s[name[:-1] + "_scales"][:, page.clamp_min(0), :, row][..., None]
    return torch.where((index < s["lengths"][:, None])[:, :, None, None, None], rows, 0.0).permute(2, 0, 3, 1, 4).contiguous()


def _compact(s):
    t = torch.arange(s["tokens"], device="cuda")
    valid = t < s["keep"][:, None]
    from_page, from_row = (x[valid] for x in _places(s, (s["starts"][:, None] + s["paths"]).long()))
    to_page, to_row = (x[valid] for x in _places(s, (s["starts"][:, None] + t).long()))
    for name in ("keys", "values", "key_scales", "value_scales"):
        if s[name] is not None:
            s[name][:, to_page, :, to_row] = s[name][:, from_page, :, from_row]
    _truncate(s, s["starts"] + s["keep"])


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _seen(position, window, sinks):
    """Keys that a token at ``position`` (counted from 0) sees."""
    near = min(position + 1, window) if window else position + 1
    return near + max(0, min(sinks, position + 1 - near))


def work(case):
    c = case
    if c["kind"] == "window":
        off = c["kv_len"] - c["q_len"]
        lengths = _spread(c["kv_len"], (c["kv_len"] + 1) // 2, c["batch"]) if c["ragged"] else [c["kv_len"]] * c["batch"]
        pairs = sum(_seen(p, c["window"], c["sinks"]) for n in lengths for p in range(off, n))
        keys = sum(min(n, max(0, n - max(0, off - c["window"] + 1)) + min(c["sinks"], max(0, off - c["window"] + 1))) for n in lengths if n > off)
        rows = c["batch"] * c["q_len"] + sum(max(0, n - off) for n in lengths)  # every output row, the query rows that count
        return {"bytes": 2 * c["dim"] * (rows * c["heads"] + 2 * keys * c["kv_heads"]), "flops": 4 * c["dim"] * c["heads"] * pairs}
    size = 1 if c["eight_bit"] else 2
    row = 2 * c["kv_heads"] * (c["dim"] * size + (4 if c["eight_bit"] else 0))  # one token's key and value in a layer of the cache
    if c["kind"] == "cache":
        lengths = _spread(c["length"], min(c["length"], c["tokens"] + c["length"] // 8), c["batch"])
        pairs = keys = 0
        for n in lengths:
            start = n - c["tokens"]
            # a chain's counts; a tree's nodes see fewer of each other
            pairs += sum(_seen(start + t, c["window"], c["sinks"]) for t in range(c["tokens"]))
            low = max(0, start - c["window"] + 1) if c["window"] else 0
            keys += n - low + min(c["sinks"], low)
        tensors = 2 * 2 * c["batch"] * c["heads"] * c["tokens"] * c["dim"]
        return {"bytes": keys * row + tensors + 4 * (keys // c["page"] + 2 * c["batch"]), "flops": 4 * c["dim"] * c["heads"] * pairs}
    counts, lengths = _spread(c["tokens"], (c["tokens"] + 1) // 2, c["batch"]), _spread(c["length"], c["length"] // 2, c["batch"])
    source = 2 * c["kv_heads"] * c["dim"] * 2  # one token's key and value as they come
    if c["kind"] == "write":  # taken, stored, read back and given in 32 bits (zeros behind a short one)
        total = sum(counts) * (source + 2 * row) + c["batch"] * c["tokens"] * 2 * source
    elif c["kind"] == "step":  # taken and stored; the accepted rows read and stored
        total = sum(counts) * (source + row) + sum(max(1, n // 3) for n in counts) * 2 * row
    else:  # seven of eight samples copy what their prompt's last page holds
        total = sum(n % c["page"] for n in lengths) * 7 // 8 * 2 * row
    return {"bytes": c["layers"] * total + 4 * 2 * c["batch"], "flops": 0}


# ------------------------------------------------------------------------------------------------ the same from the definition, in 64 bits
def exact(case, seed):
    def attend(q, k, v, visible, scale):
        """One head group in 64 bits: q [g, m, d], k and v [n, d], visible [m, n]."""
        p = torch.where(visible, q @ k.T * scale, -math.inf)
        return torch.nan_to_num(torch.softmax(p, -1)) @ v

    def window(s):
        b, h, n_q, d = s["query"].shape
        group, n_k = h // s["kv_heads"], s["kv_len"]
        if b * h * n_q * (min(s["window"], n_k) + 2048) * d > 4e13:
            return None
        out = torch.zeros(b, h, n_q, d, dtype=torch.float64, device="cuda")
        for i in range(b):
            n = n_k if s["lengths"] is None else int(s["lengths"][i])
            for head in range(s["kv_heads"]):
                heads = slice(head * group, head * group + group)
                for low in range(0, n_q, 1024):
                    p = torch.arange(low, min(low + 1024, n_q), device="cuda")[:, None] + (n_k - n_q)
                    begin = max(0, low + (n_k - n_q) - s["window"] + 1)
                    keys = [j for j in range(min(s["sinks"], begin, n))] + list(range(begin, min(n, int(p[-1]) + 1)))
                    if not keys:
                        continue
                    j = torch.tensor(keys, device="cuda")
                    seen = (j <= p) & ((p - j < s["window"]) | (j < s["sinks"])) & (p < n)
                    out[i, heads, low:low + 1024] = attend(s["query"][i, heads, low:low + 1024].double(), s["key"][i, head, j].double(),
                                                            s["value"][i, head, j].double(), seen, 1 / math.sqrt(d))
        return out

    def cache(s):
        b, h, tokens, d = s["query"].shape
        group = h // s["kv_heads"]
        out = torch.zeros(b, h, tokens, d, dtype=torch.float64, device="cuda")
        for i in range(b):
            start, n, parents = int(s["starts"][i]), int(s["lengths"][i]), None if s["tree"] is None else s["tree"][i].tolist()
            above = [[t] for t in range(tokens)]  # each token and those above it, itself first
            for t in range(tokens):
                up = t - 1 if parents is None else parents[t]
                above[t] += above[up] if up >= 0 else []
            position = torch.tensor(list(range(start)) + [start + len(a) - 1 for a in above], device="cuda")
            seen = torch.zeros(tokens, n, dtype=torch.bool, device="cuda")
            seen[:, :start] = True
            for t in range(tokens):
                seen[t, torch.tensor(above[t], device="cuda") + start] = True
            if s["window"]:
                seen &= (position[start:, None] - position < s["window"]) | (position < s["sinks"])
            pages = s["table"][i, : -(-n // s["page"])].long()
            for head in range(s["kv_heads"]):
                k, v = (s[name][0, pages, head].double() for name in ("keys", "values"))
                if s["key_scales"] is not None:
                    k, v = k * s["key_scales"][0, pages, head].double()[..., None], v * s["value_scales"][0, pages, head].double()[..., None]
                heads = slice(head * group, head * group + group)
                out[i, heads] = attend(s["query"][i, heads].double(), k.flatten(0, 1)[:n], v.flatten(0, 1)[:n], seen, 1 / math.sqrt(d))
        return out

    def pages_work(s):
        """What the rows that are read back hold."""
        if s["kind"] == "fork" or s["key_scales"] is None and s["kind"] == "step":
            return None  # copies
        batch, out = range(s["batch"]), {"table": None, "lengths": None, "uses": None}
        count = (s["keep"] if s["kind"] == "step" else s["counts"]).tolist()
        for name in ("key", "value"):
            x = s[name].double()
            if s["key_scales"] is not None:
                scale = x.abs().amax(-1, keepdim=True) / 127 + 1e-7
                x = (x / scale).round() * scale
            out[name + "s"] = torch.zeros_like(x)
            for i in batch:
                rows = s["paths"][i, : count[i]].long() if s["kind"] == "step" else slice(0, count[i])
                out[name + "s"][:, i, :, : count[i]] = x[:, i, :, rows]
        return out

    s = prepare(case, seed)
    return {"window": window, "cache": cache}.get(case["kind"], pages_work)(s)
