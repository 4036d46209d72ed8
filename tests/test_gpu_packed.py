"""Attention of packed sequences (grouped heads, sequences of different lengths one behind the other), forward and
backward, against plain 64-bit arithmetic on the CPU.

Tolerances.  O is rounded to bf16 once (half a step is 2^-8 of the value) and is a mean of V with weights that are rounded
to bf16, each off by at most 2^-8 of itself, so |O - O_exact| <= 2^-8 sum_j P_ij |v_j| + 2^-8 |O|, plus fp32 rounding of
sums of up to a few thousand terms, far below; 2^-7 sum_j P_ij |v_j| covers both.  The gradients take P and dS rounded to
bf16, the bf16 O in delta, and one rounding at the end: with A = P (|dO| |V|^T + sum_d |dO| |O| (1 + 2^-8)) the magnitude that dS is
formed of, each of dQ = scale dS K and dK = scale dS^T Q is off by at most (2^-8 for dS, 2^-8 for delta's O, 2^-8 at the
end) times scale A |K| or scale A^T |Q|, and dV by 2 * 2^-8 P^T |dO|: 4 * 2^-8 covers the products of the roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8


def make(seed, lq, lk, H, Hkv, D, behind=0, behind_k=0):
    g = torch.Generator().manual_seed(seed)

    def rand(n, h):
        return torch.randn((n, h, D), generator=g).to(torch.bfloat16)

    def bounds(lens):
        return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)

    return (rand(sum(lq) + behind, H), rand(sum(lk) + behind_k, Hkv), rand(sum(lk) + behind_k, Hkv), rand(sum(lq) + behind, H), bounds(lq), bounds(lk))


def reference(q, k, v, do, cq, ck, scale, causal):
    """(value, bound) of O, LSE, dQ, dK, dV; rows that no sequence has are 0 (LSE: -inf)."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    H, Hkv = q.shape[1], k.shape[1]
    z = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("O", q), ("dQ", q), ("dK", k), ("dV", v))}
    lse = torch.full((H, len(q)), -math.inf, dtype=torch.float64)
    for i in range(len(cq) - 1):
        Q, K = slice(int(cq[i]), int(cq[i + 1])), slice(int(ck[i]), int(ck[i + 1]))
        m, n = Q.stop - Q.start, K.stop - K.start
        if m == 0 or n == 0:
            continue
        keep = torch.ones((m, n), dtype=torch.bool).tril(n - m) if causal else torch.ones((m, n), dtype=torch.bool)
        for h in range(H):
            c = h // (H // Hkv)
            s = (q[Q, h] @ k[K, c].T * scale).masked_fill(~keep, -math.inf)
            l = torch.logsumexp(s, 1)
            lse[h, Q] = l
            p = torch.exp(s - torch.where(l == -math.inf, 0.0, l)[:, None])
            o = p @ v[K, c]
            z["O"][0][Q, h] = o
            z["O"][1][Q, h] = 2 * HALF * (p @ v[K, c].abs())
            delta = (do[Q, h] * o).sum(1, keepdim=True)
            ds = p * (do[Q, h] @ v[K, c].T - delta) * scale
            a = p * (do[Q, h].abs() @ v[K, c].abs().T + (do[Q, h] * o).abs().sum(1, keepdim=True)) * scale
            for name, at, got, off in (("dQ", (Q, h), ds @ k[K, c], a @ k[K, c].abs()), ("dK", (K, c), ds.T @ q[Q, h], a.T @ q[Q, h].abs())):
                z[name][0][at] += got
                z[name][1][at] += 4 * HALF * off
            z["dV"][0][K, c] += p.T @ do[Q, h]
            z["dV"][1][K, c] += 4 * HALF * (p.T @ do[Q, h].abs())
    return z, lse


def check(name, got, want, bound):
    off = (got.double() - want).abs()
    assert not torch.isnan(off).any(), name
    assert (off <= bound + 1e-30).all(), (name, float(off.max()), float((off / (bound + 1e-30)).max()))


def run(seed, lq, lk, H, Hkv, D, causal, behind=0, behind_k=0, poison=False):
    from flame_amd import capi
    print(f"[packed] {lq=} {lk=} {H=} {Hkv=} {D=} {causal=} {behind=}", flush=True)
    q, k, v, do, cq, ck = make(seed, lq, lk, H, Hkv, D, behind, behind_k)
    if poison:          # what lies behind the last sequence is never used
        for t, n in ((q, sum(lq)), (k, sum(lk)), (v, sum(lk)), (do, sum(lq))):
            t[n:] = float("nan")
    sc = 1.0 / math.sqrt(D)
    z, lse = reference(q, k, v, do, cq, ck, sc, causal)
    dev = [t.cuda() for t in (q, k, v, do, cq, ck)]
    dq, dk, dv, ddo, dcq, dck = dev
    nan = float("nan")
    out, lse_out = torch.full_like(dq, nan), torch.full((H, len(q)), nan, device="cuda")
    o, l = capi.attn_packed_fwd(dq, dk, dv, dcq, dck, sc, causal=causal, out=out, lse_out=lse_out)
    grads = tuple(torch.full_like(t, nan) for t in (dq, dk, dv))
    g = capi.attn_packed_bwd(dq, dk, dv, o, ddo, l, dcq, dck, sc, causal=causal, grads=grads)
    torch.cuda.synchronize()
    check("O", o.cpu(), *z["O"])
    l = l.cpu().double()
    assert torch.equal(torch.isinf(l), torch.isinf(lse)) and not torch.isnan(l).any()
    fine = ~torch.isinf(lse)
    assert ((l - lse)[fine].abs() <= 1e-5 * (1 + lse[fine].abs())).all()
    for name, t in zip(("dQ", "dK", "dV"), g):
        check(name, t.cpu(), *z[name])
    return dev, o, l, g


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("lens", [[1], [64], [65, 1, 127, 128, 129], [300, 7, 513], [0, 33, 0, 0, 200, 0]])
@pytest.mark.parametrize("H,behind", [(4, 0), (20, 0), (8, 2200)])
def test_self_attention(lens, D, causal, H, behind):
    """Few rows, whose keys the wavefronts of a workgroup share; room for many, which have 128 to a workgroup."""
    run(len(lens) * D, lens, lens, H, 2, D, causal, behind)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 72, 96, 128])
@pytest.mark.parametrize("lens,H", [([700, 1, 400], 10), ([1100, 900], 2), ([3000], 4), ([1, 2, 3] * 10 + [50], 5), ([31] * 70 + [700], 2)])
def test_shared_keys(lens, H, D, causal):
    """Grids of the kernels whose wavefronts share the keys, eight and four of them, more than 64 sequences, rows behind."""
    run(H, lens, lens, H, H // 2 if H % 2 == 0 else 1, D, causal, 40, 9)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (8, 8), (6, 3), (16, 8), (24, 8), (8, 1), (5, 5)])
def test_heads(H, Hkv):
    run(H, [70, 200, 3], [70, 200, 3], H, Hkv, 64, True)


@pytest.mark.parametrize("D", [8, 40, 72, 80, 120])
def test_head_dims_between(D):
    run(D, [140, 65], [140, 65], 4, 2, D, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([1, 5, 100], [300, 129, 100]), ([64, 200], [640, 257]), ([200, 129, 1], [100, 1, 1]), ([300], [40]),
                                   ([130, 0, 7], [0, 50, 9])])
def test_other_key_lengths(lq, lk, causal):
    """More keys than queries (earlier keys), fewer (queries without a key), and none of either."""
    run(len(lq), lq, lk, 6, 2, 64, causal)
    run(len(lq), lq, lk, 2, 2, 128, causal)
    run(len(lq), lq, lk, 10, 2, 96, causal, 1700)


@pytest.mark.parametrize("behind", [1, 127, 128, 500])
def test_rows_behind_the_last_sequence(behind):
    run(behind, [100, 29], [100, 129], 8, 4, 64, True, behind, 700 - behind, poison=True)


@pytest.mark.parametrize("n", [63, 64, 65, 300, 4200])
def test_many_sequences(n):
    """The search for a workgroup's sequence: one, two and three rounds of 64."""
    lens = [(7 * i) % 5 for i in range(n)]
    run(n, lens, lens, 2, 1, 64, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens,H,Hkv", [([100, 70, 130], 4, 2), ([1500, 40, 1700], 2, 1), ([3] * 40 + [20, 33] + [5] * 40, 4, 4)])
def test_neighbours_stay_apart(lens, H, Hkv, value, causal):
    """Infinities and NaN all over one sequence leave the others' results, to the bit, as they are without them."""
    from flame_amd import capi
    mid = len(lens) // 2
    lo, hi = sum(lens[:mid]), sum(lens[:mid + 1])
    q, k, v, do, cq, _ = (t.cuda() for t in make(5, lens, lens, H, Hkv, 128))
    got = []
    for _ in range(2):
        o, lse = capi.attn_packed_fwd(q, k, v, cq, cq, 0.1, causal=causal)
        grads = capi.attn_packed_bwd(q, k, v, o, do, lse, cq, cq, 0.1, causal=causal)
        got.append([torch.cat([t[:lo], t[hi:]]) for t in (o, lse.t(), *grads)])
        for t in (q, k, v, do):
            t[lo:hi] = value
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_long_sequence():
    run(77, [2500, 40], [2500, 40], 8, 2, 128, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("lq,lk", [([100, 5, 129], [5000, 1300, 129]), ([4200], [4200]), ([1, 0, 1], [5000, 700, 0]), ([2500, 40, 1700], [2500, 40, 1600])])
def test_walks_in_parts(lq, lk, D, causal):
    """Few tiles and long walks: the parts' sums are joined by a second launch.  Without room for them the walks stay whole."""
    from flame_amd import capi
    dev, o, l, g = run(sum(lq) + D, lq, lk, 4, 2, D, causal, behind=30, behind_k=200)
    q, k, v, do, cq, ck = dev
    assert capi.packed_fwd_workspace_bytes(len(lq), len(q), len(k), 4, D) > 0
    none = torch.empty(16, dtype=torch.uint8, device="cuda")
    o2, l2 = capi.attn_packed_fwd(q, k, v, cq, ck, D ** -0.5, causal=causal, workspace=none)
    z, lse = reference(*(t.cpu() for t in dev), D ** -0.5, causal)
    check("O", o2.cpu(), *z["O"])
    fine = ~torch.isinf(lse)
    assert torch.equal(torch.isinf(l2.cpu()), ~fine) and ((l2.cpu().double() - lse)[fine].abs() <= 1e-5 * (1 + lse[fine].abs())).all()
    least = torch.empty(-(-4 * len(q) * 4 // 256) * 512, dtype=torch.uint8, device="cuda")
    for name, t in zip(("dQ", "dK", "dV"), capi.attn_packed_bwd(q, k, v, o2, do, l2, cq, ck, D ** -0.5, causal=causal, workspace=least)):
        check(name, t.cpu(), *z[name])


def test_strided_views():
    """One projection's output [rows, (H + 2 Hkv) D] seen as q, k, v; outputs into a wider tensor."""
    from flame_amd import capi
    lens, H, Hkv, D = [90, 131], 4, 2, 64
    q, k, v, do, cq, ck = make(3, lens, lens, H, Hkv, D)
    both = torch.cat([q, k, v], 1).cuda()
    sq, sk, sv = both[:, :H], both[:, H:H + Hkv], both[:, H + Hkv:]
    z, _ = reference(q, k, v, do, cq, ck, 0.125, True)
    wide = torch.full((len(q), H + 2 * Hkv, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = torch.full((H, len(q), D), 7.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    o, lse = capi.attn_packed_fwd(sq, sk, sv, cq.cuda(), ck.cuda(), 0.125, out=out)
    g = capi.attn_packed_bwd(sq, sk, sv, o, do.cuda(), lse, cq.cuda(), ck.cuda(), 0.125, grads=(wide[:, :H], wide[:, H:H + Hkv], wide[:, H + Hkv:]))
    check("O", o.cpu(), *z["O"])
    for name, t in zip(("dQ", "dK", "dV"), g):
        check(name, t.cpu(), *z[name])


def test_rows_far_apart():
    """Row strides just below their limit, elements past 2^32: the results of the same rows close together, to the bit."""
    from flame_amd import capi
    lens, H, Hkv, D, far = [1, 170, 129], 4, 2, 64, (1 << 24) - 8
    q, k, v, do, cq, ck = (t.cuda() for t in make(8, lens, lens, H, Hkv, D))
    o, lse = capi.attn_packed_fwd(q, k, v, cq, ck, 0.125)
    near = (o, *capi.attn_packed_bwd(q, k, v, o, do, lse, cq, ck, 0.125))
    memory = torch.empty(len(q) * far, dtype=torch.bfloat16, device="cuda")
    assert memory.numel() > 2 ** 32
    at, views = 0, []
    for t in (q, k, v, do, o, q, k, v):
        views.append(memory.as_strided(t.shape, (far, D, 1), at))
        at += t.shape[1] * D
    for view, t in zip(views, (q, k, v, do)):
        view.copy_(t)
    fq, fk, fv, fdo, fo, *grads = views
    _, far_lse = capi.attn_packed_fwd(fq, fk, fv, cq, ck, 0.125, out=fo)
    capi.attn_packed_bwd(fq, fk, fv, fo, fdo, far_lse, cq, ck, 0.125, grads=tuple(grads))
    assert torch.equal(lse, far_lse)
    for a, b in zip(near, (fo, *grads)):
        assert torch.equal(a, b)


def test_same_result_every_time():
    dev, o, l, g = run(5, [700, 300, 64], [700, 300, 64], 8, 2, 128, True)
    for _ in range(3):
        _, o2, l2, g2 = run(5, [700, 300, 64], [700, 300, 64], 8, 2, 128, True)
        assert torch.equal(o, o2) and torch.equal(l, l2) and all(torch.equal(a, b) for a, b in zip(g, g2))
