"""A step of PagedCache whose copy or whose upload fails leaves the book as it was: no sequence is longer than what was stored, no page
counts as copied that was not, and the step can be tried again."""
import copy

import pytest
import torch

from flame_amd import capi
from tests.test_paged_cache_book import cache, consistent, cpu_copies, read, write  # noqa: F401 (cpu_copies: a fixture)


def book(c):
    return copy.deepcopy((c._pages, c._len, c._users, sorted(c._free), c._next))


def fail(*a, **k):
    raise RuntimeError("no room")


def started(c):
    """A sequence of 20 tokens (a whole page and part of one), three that share it, and one of its own."""
    a, lone = c.new(), c.new()
    b = c.extend([a, lone], [20, 16])
    write(c, [a, lone], b, [list(range(1, 21)), list(range(41, 57))])
    return a, [c.fork(a) for _ in range(3)], lone


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("what", ["copy", "upload"])
def test_a_failed_step_changes_nothing(cpu_copies, monkeypatch, what, share):  # noqa: F811
    c = cache()
    a, forks, lone = started(c)
    seqs, counts = [a, forks[0], lone, forks[1]], [1, 30, 1, 2]
    with monkeypatch.context() as m:
        if what == "copy":
            m.setattr(capi, "kv_copy_pages", fail)
        else:
            m.setattr(torch, "tensor", fail)
        before = book(c)
        for _ in range(2):
            with pytest.raises(RuntimeError, match="no room"):
                c.extend(seqs, counts, share_prefix=share)
            assert book(c) == before
            consistent(c)
    batch = c.extend(seqs, counts, share_prefix=share)
    consistent(c)
    tokens = [[100 + i] * n for i, n in enumerate(counts)]
    write(c, seqs, batch, tokens)
    for s, t in zip(seqs, tokens):
        had = list(range(41, 57)) if s == lone else list(range(1, 21))
        assert read(c, s, len(had) + len(t)) == had + t and c.length(s) == len(had) + len(t)
    assert read(c, forks[2], 20) == list(range(1, 21)) and c.length(forks[2]) == 20


def test_a_failed_step_takes_the_same_pages_afterwards(cpu_copies, monkeypatch):  # noqa: F811
    """The lowest free pages first, whether or not a step failed before."""
    made = []
    for failing in (False, True):
        c = cache()
        a, forks, lone = started(c)
        if failing:
            with monkeypatch.context() as m:
                m.setattr(torch, "tensor", fail)
                with pytest.raises(RuntimeError):
                    c.extend([lone, a], [40, 40])
        c.extend([a, *forks], [3, 20, 1, 1])
        made.append([c.pages(s) for s in (a, *forks, lone)])
    assert made[0] == made[1]


def test_compaction_that_fails_moves_nothing(cpu_copies, monkeypatch):  # noqa: F811
    c = cache()
    a, forks, lone = started(c)
    c.free([a, *forks])
    before = book(c)
    with monkeypatch.context() as m:
        m.setattr(capi, "kv_copy_pages", fail)
        with pytest.raises(RuntimeError):
            c.compact()
    assert book(c) == before and c.compact() == 1 and read(c, lone, 16) == list(range(41, 57))
