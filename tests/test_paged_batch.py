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
