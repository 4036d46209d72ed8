"""Attention of new tokens over a paged cache in 8 bits, against plain 64-bit arithmetic on the CPU on the numbers that the codes stand for.

Tolerance of O, as with a bf16 cache: the weights (times the scale of their value) meet the codes rounded to bf16 and O is rounded to bf16 once,
half a step of 2^-8 each: off by at most 2^-7 sum_j P_ij |v_j|; the rest is fp32."""
import math

import pytest
import torch

from tests import paged8_reference as ref
from tests.test_gpu_paged import check, reference

pytestmark = pytest.mark.gpu


def make(seed, code, lens, H, Hkv, N, D, page, block, prefix=0, spare=5, wide=0):
    """Unused places hold the largest codes (e4m3: NaN) and scales of NaN where no held token shares them; entries behind a sequence's last
    page are wild."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in [prefix] + lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    caches = []
    for _ in range(2):
        s = (8 + torch.randint(0, 8, (n_pages, Hkv, page // block), generator=g)) / 8.0 * torch.exp2(torch.randint(-9, -4, (n_pages, Hkv, page // block), generator=g).double())
        top = ref.LARGEST[code]
        c = ref.nearest((torch.randn((n_pages, Hkv, page, D), generator=g).double() * top / 4).clamp(-top, top), code)
        caches.append([c, s.double()])
    tables, keys, at = [], [], 0
    used = torch.zeros((n_pages, page), dtype=torch.bool)
    for n, m in zip([prefix] + lens, need):
        mine = order[at:at + m]
        at += m
        for j, pg in enumerate(mine):
            used[pg, :min(page, n - j * page)] = True
        keys.append(tuple(ref.numbers(c, s)[mine].transpose(0, 1).reshape(Hkv, -1, D)[:, :n] for c, s in caches))
        tables.append(mine)
    device = []
    for c, s in caches:
        c = torch.where(used[:, None, :, None], c, math.nan if code == "e4m3" else 127.0)
        s = torch.where(used.view(n_pages, 1, -1, block).any(-1), s, math.nan)
        device.append(ref.to_device(c, s, code))
    width = max(1, max(need[1:])) + wide
    table = torch.tensor([t + [2 ** 31 - 1] * (width - len(t)) for t in tables[1:]], dtype=torch.int32)
    pre = torch.tensor(tables[0] + [-7] * 2, dtype=torch.int32) if prefix else None
    q = torch.randn((len(lens), H, N, D), generator=g).to(torch.bfloat16)
    return q, device, table, torch.tensor(lens, dtype=torch.int32), pre, keys


def run(seed, code, lens, H, Hkv, N, D, page, block, prefix=0, **kw):
    from flame_amd import capi
    print(f"[paged8] {code=} {lens=} {H=} {Hkv=} {N=} {D=} {page=} {block=} {prefix=}", flush=True)
    q, ((kc, ks), (vc, vs)), table, kv_len, pre, keys = make(seed, code, lens, H, Hkv, N, D, page, block, prefix, **kw)
    extra = (pre.cuda(), torch.tensor([prefix], dtype=torch.int32, device="cuda")) if prefix else (None, None)
    out = torch.full_like(q, float("nan")).cuda()
    args = [q.cuda(), kc, vc, table.cuda(), kv_len.cuda()]
    o, lse = capi.attn_paged_fwd(*args, D ** -0.5, *extra, want_lse=True, out=out, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    want = reference(q, keys, D ** -0.5)
    check(o, lse, want)
    if not prefix and page * table.shape[1] <= 2048:           # short tables go to kernels of their own; a wider one goes the long way
        wider = torch.cat([table, torch.full((len(lens), 2048 // page + 1), -1, dtype=torch.int32)], 1).cuda()
        o2, l2 = capi.attn_paged_fwd(*args[:3], wider, args[4], D ** -0.5, want_lse=True, k_scale=ks, v_scale=vs)
        check(o2, l2, want)
    return args, (ks, vs), extra, o, lse


CODES = ["int8", "e4m3"]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("page,block", [(16, 1), (16, 16), (32, 2), (64, 32), (256, 128)])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_one_token(code, page, block, D):
    run(page + D, code, [1, 16, 17, 33, 300, 129, 128, 0], 8, 2, 1, D, page, block)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("H,Hkv", [(1, 1), (5, 5), (8, 1), (24, 8), (64, 1), (6, 3)])
def test_heads(code, H, Hkv):
    run(H, code, [70, 5, 200], H, Hkv, 1, 64, 16, 4)
    run(H, code, [70, 5, 200], H, Hkv, 1, 128, 16, 8, prefix=100)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("N", [2, 3, 8, 40])
def test_several_new_tokens(code, N):
    """Sequences shorter than the new tokens leave queries without a key."""
    run(N, code, [N, 1, 100, 65, 0, N + 1], 4, 2, N, 64, 16, 16)
    run(N, code, [N, 1, 100, 65, 0, N + 1], 8, 2, N, 128, 32, 4, prefix=50)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D", [16, 32, 48, 80, 112])
def test_head_dims_between(code, D):
    run(D, code, [140, 65], 4, 2, 1, D, 16, 8)
    run(D, code, [140, 65], 4, 2, 2, D, 16, 1, prefix=33)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("prefix", [1, 16, 100, 1024, 5000])
@pytest.mark.parametrize("B", [1, 2, 9, 17, 40])
def test_shared_prefix(code, prefix, B):
    """Up to 64 rows of a key head the wavefronts take the keys apart, above the rows."""
    run(prefix + B, code, [(37 * i) % 90 for i in range(B)], 8, 2, 1, 64, 16, 16, prefix=prefix)
    run(prefix + B, code, [(37 * i) % 90 for i in range(B)], 8, 2, 2, 128 if B % 2 else 96, 32, 1, prefix=prefix)


@pytest.mark.parametrize("code", CODES)
def test_many_sequences(code):
    """Grids of workgroups of eight and of four wavefronts; more sequences than the threads of a workgroup."""
    for B in (7, 300):
        for D in (64, 128):
            run(B + D, code, [(53 * i) % 97 for i in range(B)], 4, 2, 1, D, 16, 16)
    run(1, code, [(13 * i) % 40 for i in range(600)], 2, 1, 1, 64, 16, 2, prefix=64)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("D", [64, 128])
def test_long_sequences(code, D):
    """Walks of many units, pages found again and again, the last tile of one key."""
    run(D, code, [9001, 3, 4097], 4, 1, 1, D, 16, 16)
    run(D, code, [20033, 12000], 4, 2, 4, D, 64, 32)
    run(D, code, [2500] * 40, 8, 4, 1, D, 128, 64)


@pytest.mark.parametrize("code", CODES)
def test_pages_outside_the_cache(code):
    """Rows that would read there are NaN, the others are right."""
    from flame_amd import capi
    for prefix, lens in ((0, [40, 40, 40, 40]), (64, [40, 40, 40, 40]), (0, [3000, 2500, 3000, 40])):
        q, ((kc, ks), (vc, vs)), table, kv_len, pre, keys = make(3, code, lens, 4, 2, 1, 64, 16, 8, prefix)
        table[1, 1], table[2, 0] = kc.shape[0], -1
        kv_len[3] = 16 * table.shape[1] + 1
        extra = (pre.cuda(), torch.tensor([prefix], dtype=torch.int32, device="cuda")) if prefix else (None, None)
        o, lse = capi.attn_paged_fwd(q.cuda(), kc, vc, table.cuda(), kv_len.cuda(), 0.125, *extra, want_lse=True, k_scale=ks, v_scale=vs)
        assert torch.isnan(o[1:]).all() and torch.isnan(lse.view(4, 4)[1:]).all()
        o64, bound, _ = reference(q[:1], keys[:2], 0.125)
        assert ((o[:1].cpu().double() - o64).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("code", CODES)
def test_scales_of_nan_stay_with_their_sequence(code):
    """A block whose scale is NaN makes every answer that attends to it NaN, in K and in V, and no other."""
    from flame_amd import capi
    q, ((kc, ks), (vc, vs)), table, kv_len, _, keys = make(4, code, [50, 50, 50, 50], 4, 2, 1, 64, 16, 8)
    ks[table[1, 1], 0, 0] = math.nan
    vs[table[2, 2], 1, 1] = math.nan
    o, _ = capi.attn_paged_fwd(q.cuda(), kc, vc, table.cuda(), kv_len.cuda(), 0.125, k_scale=ks, v_scale=vs)
    bad = torch.isnan(o.cpu()).all(-1)[:, :, 0]
    want = torch.zeros((4, 4), dtype=torch.bool)
    want[1, :2] = want[2, 2:] = True
    assert torch.equal(bad, want) and torch.equal(torch.isnan(o.cpu()).any(-1)[:, :, 0], want)


def test_far_offsets():
    """Caches of more than 2^32 bytes: pages, and scales, whose offsets 32 bits do not hold."""
    from flame_amd import capi
    D, page, Hkv = 128, 64, 8
    n = 2 ** 32 // (Hkv * page * D) + 40
    g = torch.Generator().manual_seed(5)
    kc = torch.zeros((n, Hkv, page, D), dtype=torch.int8, device="cuda")
    vc = torch.zeros_like(kc)
    ks, vs = (torch.ones((n, Hkv, page), device="cuda") for _ in range(2))
    last = list(range(n - 4, n))
    c, s = zip(*[ref.random_cache(g, 4, Hkv, page, D, 1, "int8") for _ in range(2)])
    for cache, scale, codes, sc in ((kc, ks, c[0], s[0] / 1000), (vc, vs, c[1], s[1] / 1000)):
        cache[last] = codes.to(torch.int8).cuda()
        scale[last] = sc.float().cuda()
    q = torch.randn((1, 8, 1, D), generator=g).to(torch.bfloat16)
    table = torch.tensor([last], dtype=torch.int32, device="cuda")
    o, lse = capi.attn_paged_fwd(q.cuda(), kc, vc, table, torch.tensor([250], dtype=torch.int32, device="cuda"), 0.1, want_lse=True, k_scale=ks, v_scale=vs)
    both = [ref.numbers(x, (y / 1000).float().double()).transpose(0, 1).reshape(Hkv, -1, D)[:, :250] for x, y in zip(c, s)]
    empty = (torch.zeros((Hkv, 0, D)), torch.zeros((Hkv, 0, D)))
    check(o, lse, reference(q, [empty, tuple(both)], 0.1))


@pytest.mark.parametrize("code", CODES)
def test_captured_and_on_another_stream(code):
    """A graph of store and attention, replayed with new rows, lengths and tables, with eager work between; a late side stream."""
    from flame_amd import capi, functional
    q, ((kc, ks), (vc, vs)), table, kv_len, _, _ = make(6, code, [300, 77, 2000], 8, 2, 1, 128, 16, 16)
    q, table, kv_len = q.cuda(), table.cuda(), kv_len.cuda()
    k, v = (torch.randn((3, 2, 128), device="cuda").to(torch.bfloat16) for _ in range(2))
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    start = kv_len - 1

    def step(caches):
        capi.kv_store(k, v, caches[0], caches[1], table, cu, start, caches[2], caches[3])
        return functional.sdpa_paged(q, caches[0], caches[1], table, kv_len, k_scale=caches[2], v_scale=caches[3])

    copy = lambda t: t.view(torch.uint8).clone().view(t.dtype) if t.element_size() == 1 else t.clone()
    live = [copy(t) for t in (kc, vc, ks, vs)]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step([copy(t) for t in live])
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(live)
    for i in range(4):
        k.normal_()
        v.normal_()
        q.normal_()
        eager_caches = [copy(t) for t in live]
        want = step(eager_caches)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(live, eager_caches):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))       # (bits: unused scales are NaN)
        kv_len -= 3
        start -= 3
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q2 = q * 1.0
        late = functional.sdpa_paged(q2, live[0], live[1], table, kv_len, k_scale=live[2], v_scale=live[3])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(late, functional.sdpa_paged(q, live[0], live[1], table, kv_len, k_scale=live[2], v_scale=live[3]))
