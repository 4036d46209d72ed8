"""Stores into a cache in 8 bits, page copies and read-backs.  The codes and scales are defined to the last bit (the scales have four significant
bits, so that the rounding is the same in 32 and 64 bits): they are compared with the plain 64-bit arithmetic of paged8_reference for equality,
everything that a store leaves alone included."""
import math

import pytest
import torch

from flame_amd import capi
from tests import paged8_reference as ref

pytestmark = pytest.mark.gpu
CODES = ["int8", "e4m3"]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bounds(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


class Cache:
    """K and V on the device and in 64 bits; sequence i has `width` pages of its own in no order."""

    def __init__(self, seed, code, seqs, width, Hkv, page, D, block, fresh=False):
        self.g = torch.Generator().manual_seed(seed)
        self.code, self.block, self.Hkv, self.D, self.page = code, block, Hkv, D, page
        n = seqs * width + 2
        order = torch.randperm(n, generator=self.g).tolist()
        self.table = [order[i * width:(i + 1) * width] for i in range(seqs)]
        self.want, self.c, self.s = [], [], []
        for _ in range(2):
            codes, scales = ref.random_cache(self.g, n, Hkv, page, D, block, code)
            self.want.append([codes, scales])
            c, s = ref.to_device(codes, scales, code)
            self.c.append(c)
            self.s.append(s)

    def rows(self, n, size=None):
        x = torch.randn((2, n, self.Hkv, self.D), generator=self.g)
        x = x * (torch.exp(1.5 * torch.randn((2, n, self.Hkv, 1), generator=self.g)) if size is None else size)
        return x.to(torch.bfloat16)

    def store(self, x, lens, start, table=None):
        table = self.table if table is None else table
        cu = bounds(lens)
        k, v = x.cuda()
        capi.kv_store(k, v, *self.c, ints(table), ints(cu), ints(start), *self.s)
        for i in range(2):
            ref.store(*self.want[i], x[i], table, cu, start, self.block, self.code)

    def check(self):
        torch.cuda.synchronize()
        for c, s, (codes, scales) in zip(self.c, self.s, self.want):
            assert torch.equal(torch.nan_to_num(s.cpu().double(), nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
            assert torch.equal(ref.from_device(c), codes)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page,block", [(16, 1), (16, 2), (16, 16), (32, 8), (64, 32), (64, 64), (128, 128), (256, 128)])
@pytest.mark.parametrize("D", [16, 64, 80, 128])
def test_store(code, page, block, D):
    """Sequences that begin, continue, end inside blocks; none at all; rows behind the last one stay out."""
    c = Cache(page + block + D, code, 7, 3, 2, page, D, block)
    start = [0, 1, page - 1, block, max(block - 1, 0), 2 * page - 3, 5]
    lens = [2 * page + 1, 1, 2, block, block + 1, 0, 3]
    x = c.rows(sum(lens) + 4)
    print(f"[store] {code=} {page=} {block=} {D=}", flush=True)
    c.store(x, lens, start)
    c.check()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("Hkv", [1, 3, 8])
def test_token_by_token(code, Hkv):
    """A block's scale only grows until its first token is stored again, and no number is off by more than its last step (int8; e4m3: by more than
    a sixteenth of itself or half of its smallest step, the older ones twice)."""
    page = block = 16
    c = Cache(Hkv, code, 3, 2, Hkv, page, 64, block)
    held = [[], [], []]
    for step in range(20):
        x = c.rows(3)
        c.store(x, [1, 1, 1], [step] * 3)
        for b in range(3):
            held[b].append(x[:, b])
    c.check()
    for which in range(2):
        now = ref.numbers(*c.want[which])
        for b in range(3):
            for t, x in enumerate(held[b]):
                p, at = c.table[b][t // page], t % page
                s = c.want[which][1][p, :, at // block][:, None]
                off = (now[p, :, at] - x[which].double()).abs()
                if code == "int8":
                    assert (off <= s).all()
                else:
                    assert (off <= x[which].double().abs() / 8 + s * 2.0 ** -9).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-30, 2.0 ** -100, 1e-20, 1.0, 1e30, 1e38])
def test_magnitudes(code, size):
    c = Cache(3, code, 2, 2, 2, 16, 64, 16)
    x = c.rows(20, size=0.25 * size)
    c.store(x, [17, 3], [0, 16])
    c.check()
    c.store(x.flip(1)[:, :2] * 3, [1, 1], [17, 19])          # behind older tokens
    c.check()


@pytest.mark.parametrize("code", CODES)
def test_borders(code):
    """Halves, quarters and small whole parts of the largest number: quotients on and next to the borders of the codes."""
    c = Cache(4, code, 1, 4, 1, 16, 128, 16)
    Q = int(ref.LARGEST[code])
    x = torch.zeros((2, 64, 1, 128))
    for t in range(64):
        top = (128 + t) / 64.0                             # of the block of t
        x[:, t] = top * torch.tensor([i / 128.0 for i in range(128)])
    whole = torch.arange(128) + 0.5
    x[:, 16:32] = (whole * (Q / 128.0)).to(torch.bfloat16).float()
    x[:, 16, 0, 0] = float(Q)                              # scale 1 exactly: halves are borders
    x[1] = -x[1]
    c.store(x.to(torch.bfloat16), [64], [0])
    c.check()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite(code, bad):
    """The block's scale becomes NaN, the others' do not, and stays until the first token is stored again."""
    c = Cache(5, code, 2, 2, 2, 16, 64, 8)
    x = c.rows(30)
    x[0, 3, 1, 5] = bad
    x[1, 20, 0, 0] = bad
    c.store(x, [15, 15], [0, 3])
    c.check()
    assert torch.isnan(c.want[0][1]).sum() == 1 and torch.isnan(c.want[1][1]).sum() == 1
    c.store(c.rows(2), [1, 1], [5, 7])
    c.check()
    assert torch.isnan(c.s[0]).any()
    c.store(c.rows(16), [16, 0], [0, 0])
    c.check()
    assert not torch.isnan(c.s[0]).any()


def test_blocks_whose_beginning_was_never_stored():
    c = Cache(6, "int8", 3, 1, 1, 16, 64, 16)
    for i, s in enumerate((0.0, -1.0, math.inf)):
        for which in range(2):
            c.s[which][c.table[i][0]] = s
            c.want[which][1][c.table[i][0]] = s
    c.store(c.rows(6), [2, 2, 2], [3, 4, 5])
    c.check()
    assert all(torch.isnan(c.s[0][t[0]]).all() for t in c.table)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block", [1, 16])
def test_places_outside_the_cache(code, block):
    """Pages that do not exist, lengths past the table, places in front of it."""
    c = Cache(7, code, 5, 2, 2, 16, 64, block)
    table = [list(t) for t in c.table]
    table[1][0], table[2][1], table[3][0] = -1, 10 ** 9, 12
    c.store(c.rows(100), [20, 20, 20, 20, 20], [20, 3, 3, 0, -5], table)
    c.check()


def test_strided_tensors():
    """Rows out of a wider tensor, caches with the tokens outside of the heads, scales out of a wider tensor."""
    c = Cache(8, "int8", 2, 2, 2, 16, 64, 4)
    x = c.rows(30)
    wide = torch.zeros((30, 5, 2, 96), dtype=torch.bfloat16, device="cuda")
    wide[:, 1, :, 16:80] = x[0].cuda()
    wide[:, 3, :, 16:80] = x[1].cuda()
    apart = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in c.c]
    pairs = torch.zeros((*c.s[0].shape, 2), device="cuda")
    for i in range(2):
        pairs[..., i] = c.s[i]
    cu, start = bounds([13, 15]), [3, 0]
    capi.kv_store(wide[:, 1, :, 16:80], wide[:, 3, :, 16:80], *apart, ints(c.table), ints(cu), ints(start), pairs[..., 0], pairs[..., 1])
    for i in range(2):
        ref.store(*c.want[i], x[i], c.table, cu, start, 4, "int8")
        c.c[i], c.s[i] = apart[i], pairs[..., i]
    c.check()
    k, v = capi.kv_load(*apart, ints(c.table), ints(bounds([20, 3])), ints([1, 0]), 23, pairs[..., 0], pairs[..., 1])
    assert torch.equal(k, capi.kv_load(*(t.contiguous() for t in apart), ints(c.table), ints(bounds([20, 3])), ints([1, 0]), 23, *(s.contiguous() for s in c.s))[0])


@pytest.mark.parametrize("code", CODES + ["bf16"])
@pytest.mark.parametrize("Hkv,D", [(1, 16), (2, 64), (8, 128), (3, 80), (12, 128)])
@pytest.mark.parametrize("page,block", [(16, 1), (64, 16), (128, 128)])
def test_load(code, Hkv, D, page, block):
    """Every row of ragged sequences, the rows behind them (zeros) and those without a place (NaN)."""
    g = torch.Generator().manual_seed(D + page)
    lens, start, width = [5, 0, 2 * page, 1, page + 3], [0, 3, page - 1, 3 * page - 1, 1], 3
    cu = bounds(lens)
    rows, n = cu[-1] + 3, 5 * width + 1
    order = torch.randperm(n, generator=g).tolist()
    table = [order[i * width:(i + 1) * width] for i in range(5)]
    table[4][1] = n                                        # outside
    caches, scales, want = [], [], []
    for _ in range(2):
        if code == "bf16":
            x = torch.randn((n, Hkv, page, D), generator=g).to(torch.bfloat16)
            caches.append(x.cuda())
            want.append(x)
        else:
            codes, s = ref.random_cache(g, n, Hkv, page, D, block, code)
            c, s32 = ref.to_device(codes, s, code)
            caches.append(c)
            scales.append(s32)
            want.append(ref.numbers(codes, s).float().to(torch.bfloat16))          # (eleven bits at most: exact in fp32)
    print(f"[load] {code=} {Hkv=} {D=} {page=} {block=}", flush=True)
    out = [torch.full((rows, Hkv, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    got = capi.kv_load(*caches, ints(table), ints(cu), ints(start), rows, *(scales or (None, None)), out=out)
    assert got[0].data_ptr() == out[0].data_ptr()
    fresh = capi.kv_load(*caches, ints(table), ints(cu), ints(start), rows, *(scales or (None, None)))
    for x, y, w in zip(got, fresh, want):
        x = x.cpu()
        assert torch.equal(torch.nan_to_num(x, nan=99.0), torch.nan_to_num(y.cpu(), nan=99.0))
        for b in range(5):
            for i in range(lens[b]):
                pos = start[b] + i
                r = x[cu[b] + i]
                if pos // page < width and table[b][pos // page] < n:
                    assert torch.equal(r, w[table[b][pos // page], :, pos % page])
                else:
                    assert torch.isnan(r).all()
        assert (x[cu[-1]:] == 0).all()


@pytest.mark.parametrize("code", CODES)
def test_page_copies(code):
    for layers, block, D, Hkv in ((1, 16, 64, 1), (3, 1, 128, 2), (2, 4, 16, 3)):
        g = torch.Generator().manual_seed(layers)
        codes, s = ref.random_cache(g, layers * 9, Hkv, 16, D, block, code)
        kc, ks = ref.to_device(codes, s, code)
        kc, ks = kc.view(layers, 9, Hkv, 16, D), ks.view(layers, 9, Hkv, 16 // block)
        vc, vs = kc.view(torch.uint8).flip(1).contiguous().view(kc.dtype), ks.flip(1).contiguous()
        before = [t.view(torch.uint8).clone() if t.element_size() == 1 else t.clone() for t in (kc, vc, ks, vs)]
        src, dst = [0, 0, 4, 8], [1, 2, 7, 3]
        capi.kv_copy_pages(kc, vc, src, dst, ks, vs)
        for t, b in zip((kc, vc, ks, vs), before):
            b[:, dst] = b[:, src]
            assert torch.equal(t.view(torch.uint8) if t.element_size() == 1 else t, b)
    one = [t[0].clone() if t.element_size() > 1 else t.view(torch.uint8)[0].clone().view(t.dtype) for t in (kc, vc, ks, vs)]
    capi.kv_copy_pages(*one[:2], [1], [0], *one[2:])
    assert torch.equal(one[2][0], one[2][1])


def test_autograd_is_told():
    c = Cache(9, "int8", 1, 1, 1, 16, 64, 16)
    versions = [t._version for t in c.c + c.s]
    c.store(c.rows(3), [3], [0])
    assert all(t._version > v for t, v in zip(c.c + c.s, versions))
    version = c.c[0]._version
    capi.kv_load(*c.c, ints(c.table), ints([0, 3]), ints([0]), 3, *c.s)
    assert c.c[0]._version == version
