"""Attention of new tokens over a paged cache (with a prefix that the batch shares and without), stores into the pages and
page copies, against plain 64-bit arithmetic on the CPU.

Tolerance of O: the weights meet V rounded to bf16 (half a step: 2^-8 of each) and O is rounded to bf16 once, so it is off by
at most 2^-8 sum_j P_ij |v_j| + 2^-8 |O| <= 2^-7 sum_j P_ij |v_j|; everything else is fp32.  Stores and copies move bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8


def rand(g, *shape):
    return torch.randn(shape, generator=g).to(torch.bfloat16)


def make(seed, lens, H, Hkv, N, D, page, prefix=0, spare=5, wide=0):
    """A cache whose unused places hold NaN, and its tables (entries behind a sequence's last page are wild)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in [prefix] + lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    kc, vc = (torch.full((n_pages, Hkv, page, D), float("nan"), dtype=torch.bfloat16) for _ in range(2))
    tables, keys, at = [], [], 0
    for n, m in zip([prefix] + lens, need):
        mine = order[at:at + m]
        at += m
        k, v = rand(g, Hkv, m * page, D), rand(g, Hkv, m * page, D)
        for j, pg in enumerate(mine):
            held = min(page, n - j * page)
            kc[pg, :, :held] = k[:, j * page:j * page + held]
            vc[pg, :, :held] = v[:, j * page:j * page + held]
        tables.append(mine)
        keys.append((k[:, :n], v[:, :n]))
    width = max(1, max(need[1:])) + wide
    table = torch.tensor([t + [2 ** 31 - 1] * (width - len(t)) for t in tables[1:]], dtype=torch.int32)
    pre = torch.tensor(tables[0] + [-7] * 2, dtype=torch.int32) if prefix else None
    return rand(g, len(lens), H, N, D), kc, vc, table, torch.tensor(lens, dtype=torch.int32), pre, keys


def reference(q, keys, scale):
    B, H, N, D = q.shape
    o, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((B, H, N), -math.inf, dtype=torch.float64)
    pk, pv = keys[0]
    for b in range(B):
        k, v = keys[1 + b]
        n, m = k.shape[1], pk.shape[1]
        keep = torch.ones((N, m + n), dtype=torch.bool)
        keep[:, m:] = torch.arange(n)[None] <= torch.arange(N)[:, None] + n - N
        for h in range(H):
            c = h // (H // len(pk))
            kk, vv = torch.cat([pk[c], k[c]]).double(), torch.cat([pv[c], v[c]]).double()
            if m + n == 0:
                continue
            s = (q[b, h].double() @ kk.T * scale).masked_fill(~keep, -math.inf)
            l = torch.logsumexp(s, 1)
            lse[b, h] = l
            p = torch.exp(s - torch.where(l == -math.inf, 0.0, l)[:, None])
            o[b, h] = p @ vv
            bound[b, h] = 2 * HALF * (p @ vv.abs())
    return o, bound, lse


def check(got, lse, want):
    o, bound, l = want
    off = (got.cpu().double() - o).abs()
    assert not torch.isnan(off).any()
    assert (off <= bound + 1e-30).all(), (float(off.max()), float((off / (bound + 1e-30)).max()))
    lse = lse.cpu().double().view(l.shape)
    assert torch.equal(torch.isinf(lse), torch.isinf(l))
    fine = ~torch.isinf(l)
    assert ((lse - l)[fine].abs() <= 1e-5 * (1 + l[fine].abs())).all()


def run(seed, lens, H, Hkv, N, D, page, prefix=0, **kw):
    from flame_amd import capi
    print(f"[paged] {lens=} {H=} {Hkv=} {N=} {D=} {page=} {prefix=}", flush=True)
    q, kc, vc, table, kv_len, pre, keys = make(seed, lens, H, Hkv, N, D, page, prefix, **kw)
    extra = (pre.cuda(), torch.tensor([prefix], dtype=torch.int32, device="cuda")) if prefix else (None, None)
    out = torch.full_like(q, float("nan")).cuda()
    args = [t.cuda() for t in (q, kc, vc, table, kv_len)]
    o, lse = capi.attn_paged_fwd(*args, D ** -0.5, *extra, want_lse=True, out=out)
    torch.cuda.synchronize()
    want = reference(q, keys, D ** -0.5)
    check(o, lse, want)
    if not prefix and page * table.shape[1] <= 2048:           # short tables go to kernels of their own; a wider one goes the long way
        wider = torch.cat([table, torch.full((len(lens), 2048 // page + 1), -1, dtype=torch.int32)], 1).cuda()
        o2, l2 = capi.attn_paged_fwd(*args[:3], wider, args[4], D ** -0.5, want_lse=True)
        check(o2, l2, want)
    return args, extra, o, lse


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_one_token(page, D):
    run(page + D, [1, 16, 17, 33, 300, 129, 128, 0], 8, 2, 1, D, page)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (5, 5), (8, 1), (24, 8), (32, 4), (64, 1), (6, 3)])
def test_heads(H, Hkv):
    run(H, [70, 5, 200], H, Hkv, 1, 64, 16)
    run(H, [70, 5, 200], H, Hkv, 1, 64, 16, prefix=100)


@pytest.mark.parametrize("N", [2, 3, 8, 40])
def test_several_new_tokens(N):
    """Sequences shorter than the new tokens leave queries without a key."""
    run(N, [N, 1, 100, 65, 0, N + 1], 4, 2, N, 64, 16)
    run(N, [N, 1, 100, 65, 0, N + 1], 8, 2, N, 128, 32, prefix=50)


@pytest.mark.parametrize("D", [8, 40, 72, 80, 120])
def test_head_dims_between(D):
    run(D, [140, 65], 4, 2, 1, D, 16)
    run(D, [140, 65], 4, 2, 2, D, 16, prefix=33)


@pytest.mark.parametrize("prefix", [1, 16, 100, 1024, 5000])
@pytest.mark.parametrize("B", [1, 2, 9, 17, 40])
def test_shared_prefix(prefix, B):
    """Up to 64 rows of a key head the wavefronts take the keys apart, above the rows."""
    run(prefix + B, [(37 * i) % 90 for i in range(B)], 8, 2, 1, 64, 16, prefix=prefix)
    run(prefix + B, [(37 * i) % 90 for i in range(B)], 8, 2, 2, 128 if B % 2 else 96, 32, prefix=prefix)


def test_many_sequences_with_short_tables():
    """Grids of workgroups of eight and of four wavefronts."""
    for B in (7, 300):
        for D in (64, 128):
            run(B + D, [(53 * i) % 97 for i in range(B)], 4, 2, 1, D, 16)


def test_shared_prefix_of_many_sequences():
    """More sequences than the threads of a workgroup."""
    run(1, [(13 * i) % 40 for i in range(600)], 2, 1, 1, 64, 16, prefix=64)
    run(1, [(13 * i) % 40 for i in range(600)], 2, 1, 1, 64, 16)


def test_long_sequences():
    run(2, [9000, 3, 4097], 8, 2, 1, 128, 64, wide=40)
    run(3, [20001], 4, 4, 2, 64, 16)


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("longest", [2000, 2049, 4500, 9000])
def test_many_walks(longest, prefix):
    """256 heads and sequences and more: tables that one workgroup walks, and long walks in even pieces among short ones."""
    lens = [longest] + [(997 * i) % longest for i in range(17)]
    run(longest, lens, 16, 16, 1, 64, 16, prefix=prefix)
    run(longest + 1, lens[:10], 30, 30, 1, 40, 32, prefix=prefix)


def test_more_pages_than_a_wavefront_holds():
    """Units so long that a wavefront walks more than 64 pages."""
    from flame_amd import capi
    g = torch.Generator(device="cuda").manual_seed(3)
    n, Hkv, D, page = 200000, 64, 8, 16
    kc, vc = (torch.randn((n // page, Hkv, page, D), device="cuda", generator=g, dtype=torch.float32).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(n // page, device="cuda", generator=g).to(torch.int32)[None]
    q = torch.randn((1, Hkv, 1, D), device="cuda", generator=g).to(torch.bfloat16)
    o, lse = capi.attn_paged_fwd(q, kc, vc, table, torch.tensor([n - 3], dtype=torch.int32, device="cuda"), D ** -0.5, want_lse=True)
    k, v = (c[table[0].long()].transpose(1, 2).reshape(-1, Hkv, D)[:n - 3].transpose(0, 1).double() for c in (kc, vc))
    s = (k @ q[0, :, 0, :, None].double())[..., 0] * D ** -0.5
    p = torch.softmax(s, 1)[:, None]
    want, bound = (p @ v)[:, 0].cpu(), (p @ v.abs())[:, 0].cpu() * 2 * HALF
    assert ((o[0, :, 0].cpu().double() - want).abs() <= bound).all()
    assert ((lse[:, 0].double() - torch.logsumexp(s, 1)).abs() <= 1e-4).all()


def test_the_largest_pages():
    """65536 tokens in a page: one page, a page and a bit, part of one."""
    run(12, [65536, 65537, 300], 2, 1, 1, 8, 65536, spare=1)
    run(13, [1000, 1], 2, 1, 3, 8, 65536, prefix=65000, spare=1)


def test_offsets_past_32_bits():
    """Pages whose first element lies more than 2^32 elements into the cache."""
    from flame_amd import capi
    Hkv, page, D, n_pages = 8, 256, 128, 17000
    assert n_pages * Hkv * page * D > 2 ** 32
    kc = torch.empty((n_pages, Hkv, page, D), dtype=torch.bfloat16, device="cuda")
    mine = [n_pages - 1, 3, n_pages - 2]
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn((600, Hkv, D), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    table, cu, start = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([mine], [0, 600], [0]))
    vc = torch.empty_like(kc)
    capi.kv_store(k, v, kc, vc, table, cu, start)
    for j, pg in enumerate(mine):
        held = min(page, 600 - j * page)
        assert torch.equal(kc[pg, :, :held], k[j * page:j * page + held].transpose(0, 1)) and torch.equal(vc[pg, :, :held], v[j * page:j * page + held].transpose(0, 1))
    q = torch.randn((1, Hkv, 1, D), device="cuda", generator=g).to(torch.bfloat16)
    o, lse = capi.attn_paged_fwd(q, kc, vc, table, torch.tensor([600], dtype=torch.int32, device="cuda"), D ** -0.5, want_lse=True)
    none = (torch.zeros((Hkv, 0, D)), torch.zeros((Hkv, 0, D)))
    check(o, lse, reference(q.cpu(), [none, (k.transpose(0, 1).cpu(), v.transpose(0, 1).cpu())], D ** -0.5))
    kc[5], vc[5] = 1.0, 2.0
    capi.kv_copy_pages(kc, vc, [mine[0], 5], [7, n_pages - 3])
    assert torch.equal(kc[7], kc[mine[0]]) and torch.equal(vc[7], vc[mine[0]]) and bool((kc[n_pages - 3] == 1).all()) and bool((vc[n_pages - 3] == 2).all())


def test_strided_caches_and_outputs():
    """Caches [pages, page, Hkv, D] in memory, as views in the order of the call, K and V interleaved; q and O as [B, N, H, D]."""
    from flame_amd import capi
    q, kc, vc, table, kv_len, pre, keys = make(9, [100, 31, 7], 6, 2, 3, 64, 16, 40)
    both = torch.stack([kc.transpose(1, 2), vc.transpose(1, 2)], 1).contiguous().cuda()       # [pages, 2, page, Hkv, D]
    sk, sv = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    sq = q.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    out = torch.full_like(q.transpose(1, 2), 7.0).contiguous().cuda().transpose(1, 2)
    wide = torch.full((3, table.shape[1] + 3), -1, dtype=torch.int32)
    wide[:, 1:1 + table.shape[1]] = table
    o, lse = capi.attn_paged_fwd(sq, sk, sv, wide.cuda()[:, 1:1 + table.shape[1]], kv_len.cuda(), 0.125, pre.cuda(), torch.tensor([40], dtype=torch.int32).cuda(),
                                 want_lse=True, out=out)
    check(o, lse, reference(q, keys, 0.125))


def test_bad_pages_and_lengths():
    """Numbers that the host cannot see: the rows that would read there are NaN, the others are as they were."""
    from flame_amd import capi
    q, kc, vc, table, kv_len, pre, keys = make(4, [100, 50, 64, 20], 4, 2, 1, 64, 16)
    want = reference(q, keys, 0.125)
    table[0, 2], table[2, 0], kv_len[3] = kc.shape[0], -1, 16 * table.shape[1] + 1
    o, lse = capi.attn_paged_fwd(*(t.cuda() for t in (q, kc, vc, table, kv_len)), 0.125, want_lse=True)
    lse = lse.view(4, 4, 1)
    assert torch.isnan(o[[0, 2, 3]]).all() and torch.isnan(lse[[0, 2, 3]]).all()
    check(o[1:2], lse[1:2], tuple(t[1:2] for t in want))
    q, kc, vc, table, kv_len, pre, keys = make(4, [100, 50], 4, 2, 1, 64, 16, 33)
    pre[1] = kc.shape[0]
    o, _ = capi.attn_paged_fwd(*(t.cuda() for t in (q, kc, vc, table, kv_len)), 0.125, pre.cuda(), torch.tensor([33], dtype=torch.int32).cuda())
    assert torch.isnan(o).all()
    kv_len[:] = -5
    o, lse = capi.attn_paged_fwd(*(t.cuda() for t in (q, kc, vc, table, kv_len)), 0.125, want_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


def test_nan_among_the_keys():
    """A NaN that is attended to comes out, in its own sequence and head only."""
    from flame_amd import capi
    q, kc, vc, table, kv_len, pre, keys = make(6, [100, 200], 4, 2, 1, 64, 16)
    want = reference(q, keys, 0.125)
    kc[table[1, 7], 1, 3, 5] = float("nan")
    o, lse = capi.attn_paged_fwd(*(t.cuda() for t in (q, kc, vc, table, kv_len)), 0.125, want_lse=True)
    assert torch.isnan(o[1, 2:]).all()
    lse = lse.view(2, 4, 1)
    check(o[:1], lse[:1], tuple(t[:1] for t in want))
    check(o[1:, :2], lse[1:, :2], tuple(t[1:, :2] for t in want))


def test_same_result_every_time():
    args, extra, o, lse = run(8, [3000, 41, 700], 8, 2, 1, 128, 16, prefix=2000)
    from flame_amd import capi
    for _ in range(3):
        o2, l2 = capi.attn_paged_fwd(*args, 128 ** -0.5, *extra, want_lse=True)
        assert torch.equal(o, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("lens,start,page", [([5, 0, 40, 1], [0, 3, 7, 15], 16), ([1] * 9, [31, 0, 5, 64, 63, 1, 2, 3, 32], 32), ([700], [9], 64)])
@pytest.mark.parametrize("D,Hkv", [(128, 8), (64, 1), (40, 3), (256, 2)])
def test_store(lens, start, page, D, Hkv):
    from flame_amd import capi
    print(f"[store] {lens=} {start=} {page=} {D=} {Hkv=}", flush=True)
    g = torch.Generator().manual_seed(len(lens) + D)
    need = [-(-(a + b) // page) for a, b in zip(lens, start)]
    n_pages = sum(need) + 3
    order, width = torch.randperm(n_pages, generator=g).tolist(), max(need)
    k, v = rand(g, sum(lens) + 6, Hkv, D), rand(g, sum(lens) + 6, Hkv, D)          # six rows behind the last sequence
    kc, vc = rand(g, n_pages, Hkv, page, D), rand(g, n_pages, Hkv, page, D)
    dk, dv = kc.clone().cuda(), vc.clone().cuda()
    table, at, row = torch.full((len(lens), width), -1, dtype=torch.int32), 0, 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = torch.tensor(order[at:at + need[b]])
        at += need[b]
        for pos in range(start[b], start[b] + n):
            kc[table[b, pos // page], :, pos % page], vc[table[b, pos // page], :, pos % page] = k[row], v[row]
            row += 1
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    capi.kv_store(k.cuda(), v.cuda(), dk, dv, table.cuda(), cu.cuda(), torch.tensor(start, dtype=torch.int32).cuda())
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)


def test_store_leaves_out_what_has_no_place():
    from flame_amd import capi
    g = torch.Generator().manual_seed(1)
    k, v = rand(g, 30, 2, 64), rand(g, 30, 2, 64)
    kc, vc = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    dk, dv = kc.cuda(), vc.cuda()
    table = torch.tensor([[2, 9], [-1, 1], [3, 0]], dtype=torch.int32)             # pages 9 and -1 do not exist
    start = torch.tensor([14, 14, 30], dtype=torch.int32)                          # the third runs past its pages
    capi.kv_store(k.cuda(), v.cuda(), dk, dv, table.cuda(), torch.tensor([0, 10, 20, 30], dtype=torch.int32).cuda(), start.cuda())
    for row, (page, off) in {0: (2, 14), 1: (2, 15), 20: (0, 14), 21: (0, 15), **{12 + i: (1, i) for i in range(8)}}.items():
        kc[page, :, off], vc[page, :, off] = k[row], v[row]
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)


@pytest.mark.parametrize("layers,n_pages,Hkv,page,D,n", [(1, 8, 2, 16, 64, 3), (3, 900, 1, 16, 8, 430), (2, 20, 8, 64, 128, 7), (5, 9, 3, 5, 40, 4)])
@pytest.mark.parametrize("swapped", [False, True])
def test_copies(layers, n_pages, Hkv, page, D, n, swapped):
    from flame_amd import capi
    print(f"[pages] {layers=} {n_pages=} {Hkv=} {page=} {D=} {n=}", flush=True)
    g = torch.Generator().manual_seed(n)
    kc, vc = rand(g, layers, n_pages, Hkv, page, D), rand(g, layers, n_pages, Hkv, page, D)
    order = torch.randperm(n_pages, generator=g).tolist()
    src, dst = order[:n], order[n:2 * n]
    src[-1] = src[0]                                                               # one page to two places
    dk, dv = kc.cuda(), vc.cuda()
    if swapped:                                                                    # [.., page, Hkv, D] in memory
        dk, dv = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (dk, dv))
    capi.kv_copy_pages(dk, dv, src, dst)
    for c in (kc, vc):
        c[:, dst] = c[:, src].clone()
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
    capi.kv_copy_pages(dk[0], dv[0], dst[:1], order[-1:])
    capi.kv_copy_pages(dk, dv, [], [])
    kc[0, order[-1]], vc[0, order[-1]] = kc[0, dst[0]], vc[0, dst[0]]
    assert torch.equal(dk.cpu(), kc) and torch.equal(dv.cpu(), vc)
