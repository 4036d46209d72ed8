"""A paged cache of keys and values for incremental inference: the tensors, and the host's book of pages.

    cache = PagedCache(layers=24, pages=4096, page=64, kv_heads=8, head_dim=128)
    seq = cache.new()
    batch = cache.extend([seq], [len(prompt)])        # pages for the prompt; tables and lengths on the device
    for layer in ...:                                 # the prompt itself: functional.sdpa_packed
        cache.store(layer, k, v, batch)
    answers = [seq] + [cache.fork(seq) for _ in range(7)]
    while ...:
        batch = cache.extend(answers, [1] * 8)        # one token each; the prompt's pages become a prefix, read once
        for layer in ...:
            cache.store(layer, k, v, batch)           # [8, kv_heads, D]
            o = cache.attend(layer, q, batch)         # q [8, H, 1, D]
    cache.free(answers)

The book is plain integers on the host: a page that several sequences share is counted and never written; what goes to the
device is one small upload per `extend`.  Keys and values move in capi.kv_store and capi.kv_copy_pages, attention is
functional.sdpa_paged; nothing here computes on the GPU by itself.  Not thread-safe; calls are ordered by the stream that is
current when they are made.  A batch is of use until one of its sequences is extended, cut or freed or the cache is compacted: after
that its places may belong to others.  Inference only: `store` and `attend` are for torch.no_grad() or tensors that require no gradient.
"""
from __future__ import annotations

import heapq
from dataclasses import dataclass

import torch

from . import capi, functional


@dataclass
class PagedBatch:
    """What `extend` puts on the device for a list of sequences: int32 tensors, as the calls take them."""
    page_table: torch.Tensor            # [B, pages] of the sequences' own keys
    kv_len: torch.Tensor                # [B] own keys, the new ones among them
    start: torch.Tensor                 # [B] place of the first new token among the own ones
    cu: torch.Tensor                    # [B + 1] bounds of the new tokens' rows
    prefix_table: torch.Tensor | None   # [pages] that all sequences share in front of their own
    prefix_len: torch.Tensor | None     # [1]
    counts: list[int]                   # new tokens per sequence


class PagedCache:
    """k, v: bf16 [layers, pages, kv_heads, page, head_dim]."""

    def __init__(self, layers, pages, page, kv_heads, head_dim, device="cuda"):
        if min(layers, pages, kv_heads, head_dim) < 1:
            raise ValueError("layers, pages, kv_heads and head_dim are positive")
        if page < 16 or page > 65536 or page & (page - 1):
            raise ValueError("a page holds a power of two tokens from 16 to 65536")
        if head_dim % 8 or head_dim > 128:
            raise ValueError("head_dim is a multiple of 8 up to 128")
        self.page = page
        self.k = torch.empty((layers, pages, kv_heads, page, head_dim), dtype=torch.bfloat16, device=device)
        self.v = torch.empty_like(self.k)
        self._users = [0] * pages               # sequences that hold the page
        self._free = list(range(pages))         # a heap: the lowest page first
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    # ------------------------------------------------------------------------------------------------- sequences
    def new(self) -> int:
        """An empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def fork(self, seq) -> int:
        """A sequence with the same tokens.  Its pages are shared; a partly filled last one is copied when either is extended."""
        pages = self._pages[seq]
        other = self.new()
        for p in pages:
            self._users[p] += 1
        self._pages[other], self._len[other] = list(pages), self._len[seq]
        return other

    def free(self, seqs) -> None:
        """Ends the sequences; pages that nobody else holds are free again."""
        seqs = list(seqs)
        if len(set(seqs)) < len(seqs):
            raise ValueError("a sequence is listed twice")
        for seq in seqs:
            self._pages[seq]                    # an unknown one: KeyError before anything changes
        for seq in seqs:
            self._drop(self._pages.pop(seq))
            del self._len[seq]

    def cut(self, seq, length) -> None:
        """Forgets the tokens from `length` on (drafted ones that were refused)."""
        if not 0 <= length <= self._len[seq]:
            raise ValueError("a sequence can be cut to at most its length")
        keep = -(-length // self.page)
        self._drop(self._pages[seq][keep:])
        del self._pages[seq][keep:]
        self._len[seq] = length

    def length(self, seq) -> int:
        return self._len[seq]

    def pages(self, seq) -> list[int]:
        return list(self._pages[seq])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _drop(self, pages):
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                heapq.heappush(self._free, p)

    # ---------------------------------------------------------------------------------------------------- a step
    def extend(self, seqs, counts, share_prefix=True) -> PagedBatch:
        """Room for counts[i] new tokens of sequence seqs[i], and the tables of the batch.

        A last page that is partly filled and shared is copied first (all copies of the call in one launch per 400).  With
        share_prefix, whole pages that all sequences have in common at their beginning, before every new token, are listed
        once as the batch's prefix.  Without enough free pages: MemoryError.  Where this or anything else is raised, the book is
        as it was."""
        seqs, counts = list(seqs), [int(n) for n in counts]
        if not seqs or len(seqs) != len(counts) or min(counts) < 0 or len(set(seqs)) < len(seqs):
            raise ValueError("different sequences, each with a number of new tokens")
        page, need, shared = self.page, [], []
        own = {}                                # of a shared last page: users that have not left it in this call
        for seq, n in zip(seqs, counts):
            pages, old = self._pages[seq], self._len[seq]
            need.append(-(-(old + n) // page) - len(pages))
            copy = False
            if n and old % page:
                last = pages[-1]
                users = own.setdefault(last, self._users[last])
                copy = users > 1                # the last one that holds a page may write to it
                if copy:
                    own[last] = users - 1
            shared.append(copy)
        if sum(need) + sum(shared) > len(self._free):
            raise MemoryError(f"the cache has {len(self._free)} free pages and needs {sum(need) + sum(shared)}")
        taken, src, dst, lists = [], [], [], []
        try:
            for seq, more, copy in zip(seqs, need, shared):
                pages, new = self._pages[seq], []
                for _ in range(copy + more):
                    taken.append(heapq.heappop(self._free))
                    new.append(taken[-1])
                if copy:
                    src.append(pages[-1])
                    dst.append(new[0])
                    pages = pages[:-1]
                lists.append(pages + new if new else pages)
            if src:
                capi.kv_copy_pages(self.k, self.v, src, dst)
            batch = self._batch(lists, [self._len[s] + n for s, n in zip(seqs, counts)], counts, share_prefix)
        except BaseException:
            for p in taken:
                heapq.heappush(self._free, p)
            raise
        # the copies and the upload were accepted: the book follows
        for p in src:
            self._users[p] -= 1
        for p in taken:
            self._users[p] = 1
        for seq, n, pages in zip(seqs, counts, lists):
            self._pages[seq] = pages
            self._len[seq] += n
        return batch

    def _batch(self, lists, lens, counts, share_prefix) -> PagedBatch:
        """Tables of sequences with these pages and lengths, the last counts[i] tokens of which are new."""
        common = 0
        if share_prefix and len(lists) > 1:
            most = min(m - n for m, n in zip(lens, counts)) // self.page
            first = lists[0]
            common = next((i for i in range(most) if any(x[i] != first[i] for x in lists)), most)
        B, width, held = len(lists), max(1, max(len(x) for x in lists) - common), common * self.page
        data = lists[0][:common] + [held]
        for x in lists:
            row = x[common:]
            data += row + [0] * (width - len(row))
        data += [m - held for m in lens] + [m - n - held for m, n in zip(lens, counts)]
        at = [0]
        for n in counts:
            at.append(at[-1] + n)
        up = torch.tensor(data + at, dtype=torch.int32).to(self.k.device)
        prefix, length, table, kv_len, start, cu = up.split([common, 1, B * width, B, B, B + 1])
        return PagedBatch(table.view(B, width), kv_len, start, cu, prefix if common else None, length if common else None, counts)

    def store(self, layer, k, v, batch) -> None:
        """Rows k, v [new tokens of the batch, kv_heads, head_dim], sequence after sequence, to their places.  Inference only, as `attend`: rows
        that require a gradient are refused unless torch.no_grad() is on."""
        if k.shape[0] != sum(batch.counts):
            raise ValueError("as many rows as the batch has new tokens")
        if not k.shape[0]:
            return
        capi.kv_store(k, v, self.k[layer], self.v[layer], batch.page_table, batch.cu, batch.start)

    def attend(self, layer, q, batch, scale=None):
        """functional.sdpa_paged of q [B, H, N, head_dim], the batch's N new tokens of each sequence (stored before)."""
        if any(n != q.shape[2] for n in batch.counts):
            raise ValueError("q holds the batch's new tokens, the same number of every sequence")
        return functional.sdpa_paged(q, self.k[layer], self.v[layer], batch.page_table, batch.kv_len, batch.prefix_table, batch.prefix_len, scale)

    # ------------------------------------------------------------------------------------------------ compaction
    def compact(self) -> int:
        """Moves the held pages to the lowest places of the cache and returns how many moved (the pages behind them are
        free then, in one piece).  Batches made before are of no use afterwards."""
        held = len(self._users) - len(self._free)
        src = [p for p in range(held, len(self._users)) if self._users[p]]
        dst = [p for p in range(held) if not self._users[p]]
        if src:
            capi.kv_copy_pages(self.k, self.v, src, dst)
            to = dict(zip(src, dst))
            for p, q in to.items():
                self._users[q], self._users[p] = self._users[p], 0
            for seq, pages in self._pages.items():
                self._pages[seq] = [to.get(p, p) for p in pages]
            self._free = list(range(held, len(self._users)))
        return len(src)
