"""What a batch of PagedCache says of itself, and what attend_rows takes: on the host, before anything reaches a device."""
import dataclasses

import pytest
import torch

from flame_amd.paged_cache import PagedBatch, PagedCache


def test_fields_by_position():
    """Callers with tables of their own name the first seven by their places; a number too many is an error, not another field."""
    c = PagedCache(1, 20, 16, 1, 16, device="cpu")
    seqs = [c.new(), c.new()]
    c.extend(seqs, [20, 3])
    batch = c.extend(seqs, [1, 30])
    names = [f.name for f in dataclasses.fields(PagedBatch) if not f.kw_only]
    assert names == ["page_table", "kv_len", "start", "cu", "prefix_table", "prefix_len", "counts"]
    again = PagedBatch(*(getattr(batch, n) for n in names))
    for n in names:
        assert getattr(again, n) is getattr(batch, n)
    assert batch.past.tolist() == [20, 3] and batch.start.tolist() == [20, 3] and batch.kv_len.tolist() == [21, 33]
    with pytest.raises(TypeError):
        PagedBatch(*(getattr(batch, n) for n in names), batch.past)


@pytest.fixture
def calls(monkeypatch):
    """attend_rows as far as the device's calls: reads the tables' numbers of keys."""
    from flame_amd import capi, functional
    made = []
    monkeypatch.setattr(capi, "kv_load", lambda kc, vc, table, cu, start, rows, *scales: (torch.zeros((rows, 1, 16)),) * 2)
    monkeypatch.setattr(capi, "kv_copy_pages", lambda *a: None)
    monkeypatch.setattr(functional, "sdpa_packed", lambda q, k, v, cu, cu_k, **more: made.append((cu.tolist(), cu_k.tolist())) or torch.zeros_like(q))
    return made


def cache_of(lens):
    c = PagedCache(1, 40, 16, 1, 16, device="cpu")
    seqs = [c.new() for _ in lens]
    c.extend(seqs, lens)
    return c, seqs


def q_of(batch):
    return torch.zeros((sum(batch.counts), 2, 16))


def test_rows_attend_to_all_that_is_held(calls):
    c, seqs = cache_of([20, 5, 0])
    for counts in ([3, 0, 16], [1, 1, 1], [0, 40, 0]):
        batch = c.extend(seqs, counts)
        held = c.held(seqs)
        other = c.new()                        # what happens to others does not matter
        c.extend([other], [30])
        c.attend_rows(0, q_of(batch), batch, held)
        assert calls[-1] == (batch.cu.tolist(), held.cu.tolist()) and held.counts == [c.length(s) for s in seqs]
        c.free([other])
    batch = c.extend(seqs, [0, 0, 2])
    mine = PagedBatch(batch.page_table, batch.kv_len, batch.start, batch.cu, None, None, batch.counts)       # tables of one's own
    c.attend_rows(0, q_of(mine), mine, c.held(seqs))


def test_stale_or_foreign_held_is_refused(calls):
    """Before the batch's tokens were counted, keys end too early and the causal line is shifted; everything else that changed in between is as bad."""
    c, seqs = cache_of([20, 5, 7])
    before = c.held(seqs)
    batch = c.extend(seqs, [1, 0, 3])
    with pytest.raises(ValueError, match="made after the batch"):
        c.attend_rows(0, q_of(batch), batch, before)
    with pytest.raises(ValueError, match="made after the batch"):
        c.attend_rows(0, q_of(batch), batch, c.held(seqs[::-1]))
    with pytest.raises(ValueError, match="other sequences"):
        c.attend_rows(0, q_of(batch), batch, c.held(seqs[:2]))
    held = c.held(seqs)
    c.cut(seqs[2], 7)
    again = c.extend(seqs, [1, 0, 3])          # as many tokens as before
    for b, h in ((again, held), (batch, c.held(seqs))):
        with pytest.raises(ValueError, match="made after the batch"):
            c.attend_rows(0, q_of(b), b, h)
    c.attend_rows(0, q_of(again), again, c.held(seqs))
    c.cut(seqs[0], c.length(seqs[0]))          # forgets nothing
    c.attend_rows(0, q_of(again), again, c.held(seqs))


def test_compaction_ends_a_held(calls):
    c, seqs = cache_of([20, 5, 7])
    batch = c.extend(seqs, [1, 1, 1])
    held = c.held(seqs[1:])
    some = c.extend(seqs[1:], [1, 1])
    c.free(seqs[:1])
    held = c.held(seqs[1:])
    c.attend_rows(0, q_of(some), some, held)
    assert c.compact() > 0
    with pytest.raises(ValueError, match="made after the batch"):
        c.attend_rows(0, q_of(some), some, c.held(seqs[1:]))
    assert len(calls) == 1 and batch.state[0][0] == seqs[0]
