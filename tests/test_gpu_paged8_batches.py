"""Batches of many sequences and many rows through stores into 8 bits and read-backs: more sequences than a wavefront has lanes, and so many
blocks and heads that a group of threads takes several.  A row is stored and read alike in any company: the large calls are compared bit for bit with
calls of few sequences, which other tests compare with 64-bit arithmetic, and the smaller ones with that arithmetic itself."""
import pytest
import torch

from flame_amd import capi
from tests import paged8_reference as ref
from tests.test_gpu_paged8_store import CODES, Cache, bounds, ints

pytestmark = pytest.mark.gpu


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int32)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page,block", [(16, 1), (16, 4), (32, 32)])
@pytest.mark.parametrize("seqs", [64, 65, 150])
def test_store_of_many_sequences(code, page, block, seqs):
    """Prompts, single tokens and sequences without any, in no order; rows behind the last one stay out."""
    c = Cache(seqs + block, code, seqs, 2, 1, page, 16, block)
    lens = [(7 * i) % (page + 3) if i % 3 == 0 else i % 2 for i in range(seqs)]
    start = [(5 * i) % (page - 2) for i in range(seqs)]
    lens[-1] = 5
    x = c.rows(sum(lens) + 3)
    print(f"[store] {code=} {page=} {block=} {seqs=}", flush=True)
    c.store(x, lens, start)
    c.check()


@pytest.mark.parametrize("code", CODES + ["bf16"])
@pytest.mark.parametrize("Hkv,D", [(1, 16), (8, 128)])
@pytest.mark.parametrize("seqs", [64, 65, 1000])
def test_load_of_many_sequences(code, Hkv, D, seqs):
    """Rows of one head of 16 numbers go many to a wavefront, those of eight heads one."""
    g = torch.Generator().manual_seed(seqs + D)
    page, block, width = 16, 8, 2
    lens = [(11 * i) % 23 if i % 4 else 0 for i in range(seqs)]
    start = [(3 * i) % 9 for i in range(seqs)]
    n = seqs * width
    table = torch.randperm(n, generator=g).view(seqs, width)
    at = torch.tensor(bounds(lens))
    rows = int(at[-1]) + 5
    b = torch.repeat_interleave(torch.arange(seqs), torch.tensor(lens))
    pos = torch.tensor(start)[b] + torch.arange(int(at[-1])) - at[b]
    caches, scales, want = [], [], []
    for _ in range(2):
        if code == "bf16":
            x = torch.randn((n, Hkv, page, D), generator=g).to(torch.bfloat16)
            caches.append(x.cuda())
        else:
            codes, s = ref.random_cache(g, n, Hkv, page, D, block, code)
            c, s32 = ref.to_device(codes, s, code)
            caches.append(c)
            scales.append(s32)
            x = ref.numbers(codes, s).float().to(torch.bfloat16)
        want.append(x[table[b, pos // page], :, pos % page])
    print(f"[load] {code=} {Hkv=} {D=} {seqs=}", flush=True)
    got = capi.kv_load(*caches, ints(table.tolist()), ints(at.tolist()), ints(start), rows, *(scales or (None, None)))
    for x, w in zip(got, want):
        assert torch.equal(x[:len(w)].cpu(), w)
        assert (x[len(w):] == 0).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("Hkv,D,block,seqs,rows", [
    (3, 128, 16, 1, 40000), (5, 64, 1, 3, 30000), (8, 128, 1, 70, 9000), (8, 128, 4, 5, 30000), (2, 128, 128, 2, 200000), (9, 80, 8, 90, 12000), (3, 16, 64, 4, 150000)])
def test_many_blocks_and_heads(code, Hkv, D, block, seqs, rows):
    """From 2^19 threads on a group takes several blocks' heads, as many as divide their number and fewer."""
    page = max(block, 64)
    lens = [rows // seqs + (i % 3 - 1) * min(i, 5) for i in range(seqs)]
    start = [(13 * i) % (2 * block + 1) for i in range(seqs)]
    width = -(-(max(lens) + 2 * block + 1) // page)
    g = torch.Generator(device="cuda").manual_seed(D + block)
    table = torch.randperm(seqs * width, device="cuda", generator=g).view(seqs, width).to(torch.int32)
    shape = (seqs * width, Hkv, page, D)
    dtype = ref.DTYPES[code]
    codes = torch.randint(0, 60, shape, dtype=torch.int8, device="cuda", generator=g).view(dtype)
    scales = torch.exp2(torch.randint(-8, 0, (*shape[:2], page // block), device="cuda", generator=g).float())
    many, few = ([codes.clone(), codes.flip(2).contiguous() if dtype == torch.int8 else codes.view(torch.int8).flip(2).contiguous().view(dtype), scales.clone(), scales.flip(1).contiguous()]
                 for _ in range(2))
    k, v = (torch.randn((sum(lens), Hkv, D), device="cuda", generator=g).mul_(torch.rand((sum(lens), Hkv, 1), device="cuda", generator=g) * 9).to(torch.bfloat16) for _ in range(2))
    at = bounds(lens)
    print(f"[many] {code=} {Hkv=} {D=} {block=} {seqs=} {rows=}", flush=True)
    capi.kv_store(k, v, many[0], many[1], table, ints(at), ints(start), many[2], many[3])
    piece = max(block, 1024 // block * block)              # whole blocks, so that every block's rows come in one call
    for i in range(seqs):
        first = 0
        while first < lens[i]:
            n = min(piece - (start[i] + first) % block, lens[i] - first)
            a = at[i] + first
            capi.kv_store(k[a:a + n], v[a:a + n], few[0], few[1], table[i:i + 1], ints([0, n]), ints([start[i] + first]), few[2], few[3])
            first += n
    for a, b in zip(many, few):
        assert torch.equal(raw(a), raw(b))
    got = capi.kv_load(many[0], many[1], table, ints(at), ints(start), sum(lens), many[2], many[3])
    one = [capi.kv_load(many[0], many[1], table[i:i + 1], ints([0, lens[i]]), ints([start[i]]), lens[i], many[2], many[3]) for i in range(seqs)]
    for which in range(2):
        assert torch.equal(got[which], torch.cat([x[which] for x in one]))
