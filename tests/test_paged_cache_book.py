"""The book of pages of PagedCache on the host: the copies it asks for are made on CPU tensors by a stand-in, and what every
sequence reads back through its tables is compared with a plain list per sequence."""
import random

import pytest
import torch

from flame_amd import capi, paged_cache
from flame_amd.paged_cache import PagedCache


@pytest.fixture
def cpu_copies(monkeypatch):
    made = []

    def copy(k, v, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)        # what the call refuses
        made.append((list(src), list(dst)))
        for c in (k, v):
            c[:, dst] = c[:, src].clone()
    monkeypatch.setattr(capi, "kv_copy_pages", copy)
    return made


def cache(pages=40, page=16):
    return PagedCache(2, pages, page, 1, 8, device="cpu")


def write(c, seqs, batch, tokens):
    """Stores tokens[seq] (numbers) as keys through the batch's tables, as the kernel does."""
    held = int(batch.prefix_len[0]) if batch.prefix_len is not None else 0
    for i, s in enumerate(seqs):
        for j, t in enumerate(tokens[i]):
            pos = int(batch.start[i]) + j
            assert c.length(s) - len(tokens[i]) + j == held + pos
            page = int(batch.page_table[i, pos // c.page])
            assert c._users[page] == 1, "a shared page is written"
            c.k[:, page, :, pos % c.page] = t
            c.v[:, page, :, pos % c.page] = -t


def read(c, seq, n):
    return [int(c.k[1, c.pages(seq)[p // c.page], 0, p % c.page, 0]) for p in range(n)]


def consistent(c):
    held = [0] * len(c._users)
    for pages in c._pages.values():
        for p in pages:
            held[p] += 1
    assert held == c._users and sorted(c._free) == [p for p, n in enumerate(held) if n == 0]


def test_random_life(cpu_copies):
    rng = random.Random(3)
    c, said, number = cache(120), {}, 1
    for step in range(400):
        what = rng.random()
        if what < 0.15 or not said:
            said[c.new()] = []
        elif what < 0.3:
            s = rng.choice(list(said))
            said[c.fork(s)] = list(said[s])
        elif what < 0.4:
            gone = rng.sample(list(said), min(len(said), rng.randint(1, 3)))
            c.free(gone)
            for s in gone:
                del said[s]
        elif what < 0.5:
            s = rng.choice(list(said))
            n = rng.randint(0, len(said[s]))
            c.cut(s, n)
            said[s] = said[s][:n]
        elif what < 0.55:
            c.compact()
            used = len(c._users) - c.free_pages
            assert all(p < used for s in said for p in c.pages(s))
        else:
            seqs = rng.sample(list(said), min(len(said), rng.randint(1, 5)))
            counts = [rng.choice([0, 1, 1, 3, 20, 40]) for _ in seqs]
            tokens = [[number + i for i in range(n)] for n in counts]
            before = {s: c.pages(s) for s in said}, list(c._users), sorted(c._free)
            try:
                b = c.extend(seqs, counts, share_prefix=rng.random() < 0.7)
            except MemoryError:
                assert before == ({s: c.pages(s) for s in said}, list(c._users), sorted(c._free))
                continue
            write(c, seqs, b, tokens)
            for s, t in zip(seqs, tokens):
                said[s] = said[s] + t
            number = (number + 41) % 200 + 1        # whole numbers that bf16 holds
        consistent(c)
        for s, t in said.items():
            assert c.length(s) == len(t) and read(c, s, len(t)) == t
    assert len(cpu_copies) > 20


def test_prefix_of_forks(cpu_copies):
    c = cache()
    a = c.new()
    c.extend([a], [50])                             # three whole pages and two tokens
    forks = [a] + [c.fork(a) for _ in range(3)]
    b = c.extend(forks, [1] * 4)
    assert cpu_copies and len(cpu_copies[-1][0]) == 3 and len(set(cpu_copies[-1][0])) == 1       # the last holder writes to its own page
    assert b.prefix_table.tolist() == c.pages(a)[:3] and b.prefix_len.tolist() == [48]
    assert b.kv_len.tolist() == [3] * 4 and b.start.tolist() == [2] * 4 and b.cu.tolist() == [0, 1, 2, 3, 4]
    assert [row[0] for row in b.page_table.tolist()] == [c.pages(s)[3] for s in forks] and len({c.pages(s)[3] for s in forks}) == 4
    lone = c.new()
    b = c.extend(forks + [lone], [1, 1, 1, 1, 2])
    assert b.prefix_table is None and b.prefix_len is None and b.kv_len.tolist() == [52, 52, 52, 52, 2]
    # a prefix ends before every new token
    d, e = c.new(), None
    c.extend([d], [32])
    e = c.fork(d)
    assert c.extend([d, e], [0, 0]).prefix_len.tolist() == [32]
    c.cut(e, 20)
    assert c.extend([d, e], [0, 4]).prefix_len.tolist() == [16]


def test_refusals(cpu_copies):
    for bad in (dict(page=24), dict(page=8), dict(head_dim=60), dict(head_dim=136), dict(layers=0), dict(pages=0)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=1, pages=4, page=16, kv_heads=1, head_dim=64, device="cpu"), **bad})
    c = cache(4)
    a = c.new()
    for seqs, counts in (([], []), ([a], [1, 2]), ([a], [-1]), ([a, a], [1, 1])):
        with pytest.raises(ValueError):
            c.extend(seqs, counts)
    with pytest.raises(KeyError):
        c.extend([99], [1])
    with pytest.raises(MemoryError):
        c.extend([a], [65])
    c.extend([a], [64])
    assert c.free_pages == 0
    for seqs, err in (([a, a], ValueError), ([a, 99], KeyError)):
        with pytest.raises(err):
            c.free(seqs)
    with pytest.raises(ValueError):
        c.cut(a, 65)
    c.free([a])
    assert c.free_pages == 4
    b = PagedCache(1, 4, 16, 1, 8, device="cpu")
    s = b.new()
    batch = b.extend([s], [3])
    with pytest.raises(ValueError):
        b.store(0, torch.zeros(2, 1, 8), torch.zeros(2, 1, 8), batch)
    with pytest.raises(ValueError):
        b.attend(0, torch.zeros(1, 1, 1, 8), batch)


def test_documented_example_names_what_exists():
    for name in ("new", "fork", "free", "cut", "extend", "store", "attend", "compact"):
        assert callable(getattr(paged_cache.PagedCache, name))
