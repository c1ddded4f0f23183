"""Oracles of the serving operators: attention from its definition in 64 bits, and the paged cache's
bookkeeping as plain Python lists, one sequence at a time."""

from __future__ import annotations

import torch


def window_visible(q_len, kv_len, window, sinks, length):
    """[q_len, kv_len] truth values, one comparison after the other."""
    p = torch.arange(q_len)[:, None] + kv_len - q_len
    j = torch.arange(kv_len)[None, :]
    return (j <= p) & ((p - j < window) | (j < sinks)) & (j < length) & (p < length) & (p >= 0)


def tree_visible(tokens, start, length, parents, window, sinks):
    """[tokens, length] for tokens at rows start + t; parents None: a chain."""
    seen = torch.zeros(tokens, length, dtype=torch.bool)
    above = []
    for t in range(tokens):
        up = t - 1 if parents is None else parents[t]
        above.append([t] + (above[up] if 0 <= up < t else []))
    position = list(range(start)) + [start + len(a) - 1 for a in above]
    for t in range(tokens):
        if start + t >= length:
            continue
        for j in list(range(start)) + [start + a for a in above[t]]:
            seen[t, j] = window is None or position[start + t] - position[j] < window or position[j] < sinks
    return seen


def attend(q, k, v, visible, scale, dtype, value_step=0.0):
    """One head in 64 bits: rows [m, d], keys [n, d].  Returns the result and how far a kernel that rounds
    its probabilities and its result to ``dtype`` may be off:

    - the result: half a step, h = eps / 2 relative;
    - each probability: h relative, and where a float16 is subnormal 2^-25 absolute (relative to the largest
      probability of the row, which is held at 1 or more): h * sum w|v| + n * 2^-25 * max|v|;
    - a score: a sum of d products in 32 bits, (d + 4) * 2^-24 * scale * sum|q k|, and the exponential,
      2^-18 (the exponential unit is within 2^-21; a polynomial that takes a part of the work has a largest
      relative error of 2.9e-6 = 2^-18.4): as a relative change of every weight, twice (the quotient).
    ``value_step``: the largest 8-bit row maximum; codes up to it share one reference exponent.
    """
    q, k, v = q.double(), k.double(), v.double()
    s = torch.where(visible, q @ k.T * scale, -torch.inf)
    w = torch.nan_to_num(torch.softmax(s, -1))
    size = v.abs()
    h = torch.finfo(dtype).eps / 2
    weight = (q.shape[1] + 4) * 2.0**-24 * torch.where(visible, scale * (q.abs() @ k.abs().T), 0).amax(-1, keepdim=True) + 2.0**-18
    out = w @ v
    n = visible.sum(-1, keepdim=True)
    tiny = n * 2.0**-25 * max(float(size.max()), value_step) if dtype is torch.float16 else 0
    return out, h * out.abs() + (h + 2 * weight) * (w @ size) + tiny


def check(got, want, off, where=""):
    got = got.double().cpu()
    want, off = want.cpu(), off.cpu()
    bad = ~((got - want).abs() <= off)
    assert not bad.any(), f"{where}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / off.clamp_min(1e-300)).max():.2f} of the bound"


class ListCache:
    """The bookkeeping of a PageCache: each sequence is a list of pages and a length."""

    def __init__(self, batch, pages, page, width):
        self.batch, self.pages, self.page, self.width = batch, pages, page, width
        self.own = [[] for _ in range(batch)]
        self.length, self.start = [0] * batch, [0] * batch
        self.refused, self.copied = [0] * batch, []

    def uses(self):
        n = [0] * self.pages
        for pages in self.own:
            for p in pages:
                n[p] += 1
        return n

    def table(self):
        return [pages + [-1] * (self.width - len(pages)) for pages in self.own]

    def extend(self, counts):
        uses, page = self.uses(), self.page
        free = [p for p in range(self.pages) if uses[p] == 0]
        counts = [max(c, 0) for c in counts]
        fits = [self.length[b] + counts[b] <= self.width * page for b in range(self.batch)]
        grows = [b for b in range(self.batch) if fits[b] and counts[b] and self.length[b] % page]
        copies = set()
        for b in grows:
            owners = [o for o in grows if self.own[o][-1] == self.own[b][-1]]
            if uses[self.own[b][-1]] > 1 and (len(owners) < uses[self.own[b][-1]] or owners[0] != b):
                copies.add(b)
        taken, self.copied = 0, []
        for b in range(self.batch):
            need = -(-(self.length[b] + counts[b]) // page) - len(self.own[b]) + (b in copies) if fits[b] else 0
            self.start[b] = self.length[b]
            self.refused[b] = int(not fits[b] or (need > 0 and taken + need > len(free)))
            mine, taken = free[taken:taken + need], taken + need
            if self.refused[b]:
                continue
            if b in copies:
                self.copied.append((self.own[b][-1], mine[0], self.length[b] % page))
                self.own[b][-1] = mine.pop(0)
            self.own[b] += mine
            self.length[b] += counts[b]

    def fork(self, parents):
        self.refused = [int(p >= self.batch) for p in parents]
        parents = [b if p >= self.batch else p for b, p in enumerate(parents)]
        own, length = self.own, self.length
        self.own = [list(own[p]) if p >= 0 else [] for p in parents]
        self.length = [length[p] if p >= 0 else 0 for p in parents]
        self.start = list(self.length)

    def truncate(self, lengths):
        for b in range(self.batch):
            self._cut(b, min(self.length[b], max(lengths[b], 0)))

    def _cut(self, b, keep):
        self.length[b] = self.start[b] = keep
        self.own[b] = self.own[b][: -(-keep // self.page)]

    def compact(self, paths, counts):
        for b in range(self.batch):
            added, path = self.length[b] - self.start[b], paths[b][: max(counts[b], 0)]
            good = 0 <= counts[b] <= min(added, len(paths[b])) and all(0 <= x < added for x in path) and all(x < y for x, y in zip(path, path[1:]))
            self.refused[b] = int(not good)
            if good:
                self._cut(b, self.start[b] + counts[b])
