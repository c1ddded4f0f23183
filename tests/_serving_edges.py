"""The paged cache's bookkeeping as lists, where sequences of different lengths share a last page."""

from __future__ import annotations

from _serving import ListCache


class LongestKeeps(ListCache):
    """Of the owners of a shared last page that all grow, the longest (the first of these) keeps it.

    ``ListCache`` lets the first of them keep it, whatever its length: where the copy of a longer owner is then
    refused, the first one's new rows fall on rows that the refused one still holds.
    """

    def extend(self, counts):
        uses, page = self.uses(), self.page
        free = [p for p in range(self.pages) if uses[p] == 0]
        counts = [max(c, 0) for c in counts]
        fits = [self.length[b] + counts[b] <= self.width * page for b in range(self.batch)]
        grows = [b for b in range(self.batch) if fits[b] and counts[b] and self.length[b] % page]
        last = {b: self.own[b][-1] for b in grows}
        keeper = {}
        for b in grows:
            owners = [o for o in grows if last[o] == last[b]]
            if len(owners) == uses[last[b]]:
                keeper[last[b]] = max(owners, key=lambda o: (self.length[o], -o))
        self.start, self.refused, self.copied = list(self.length), [0] * self.batch, []
        taken = 0
        for b in range(self.batch):
            copy = b in last and uses[last[b]] > 1 and keeper.get(last[b]) != b
            need = -(-(self.length[b] + counts[b]) // page) - len(self.own[b]) + copy if fits[b] else 0
            mine, taken = free[taken:taken + need], taken + need
            if not fits[b] or len(mine) < need:
                self.refused[b] = 1
                continue
            if copy:
                self.copied.append((last[b], mine[0], self.length[b] % page))
                self.own[b][-1] = mine.pop(0)
            self.own[b] += mine
            self.length[b] += counts[b]

    def places(self, b, first=0):
        """(page, row) of the sequence's rows from ``first`` on."""
        return [(self.own[b][j // self.page], j % self.page) for j in range(first, self.length[b])]

    def overwritten(self):
        """Places of rows added last that another sequence holds too."""
        added = [(b, at) for b in range(self.batch) for at in self.places(b, self.start[b])]
        return [(b, o, at) for b, at in added for o in range(self.batch) if o != b and at in self.places(o)]


def unequal_owners(rng, batch, page, steps):
    """A run of calls in which sequences of different lengths share last pages: (method, arguments) each."""
    for _ in range(steps // 3):
        parent = rng.randrange(batch)
        yield "fork", [parent if rng.random() < 0.7 else b for b in range(batch)]
        yield "truncate", [rng.choice([10**6, 10**6, page + 3, page - 5, page // 2]) for _ in range(batch)]
        few = rng.random() < 0.6  # all owners grow
        yield "extend", [1 + rng.randrange(page // 2) if few else rng.choice([0, 1, page // 2, page]) for _ in range(batch)]
