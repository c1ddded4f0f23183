"""CPU tests of the serving operators' edges: the list model of shared last pages."""

import random

import pytest

from _serving import ListCache
from _serving_edges import LongestKeeps, unequal_owners


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
