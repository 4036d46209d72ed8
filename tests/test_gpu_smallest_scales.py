"""Scales so small that every score is zero: each query's weights are one over the number of its keys, LSE its logarithm.

Tolerances: O is a mean of V with weights rounded to bf16 (half a step: 2^-8 of each), rounded once more; dV = P^T dO with the same
roundings, all sums in fp32; dQ and dK are scale times sums of some hundred terms of a few hundred at most, nothing that bf16 keeps above 1e-30."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8
# the smallest normal number, one below which 8 / (scale log2 e) has no finite value, one well above, a subnormal one
SCALES = [1.1754944e-38, 1.6e-38, 1e-30, 1e-40]


def rand(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def near(name, got, want, bound):
    off = (got.cpu().double() - want).abs()
    assert not torch.isnan(off).any() and bool((off <= bound + 1e-30).all()), (name, float(off.max()))


def of_head(q, k, v, do, causal):
    """(O, bound), LSE, (dV, bound) of one head, [n, D] and [m, D]."""
    keep = torch.ones((len(q), len(k)), dtype=torch.float64)
    if causal:
        keep = keep.tril(len(k) - len(q))
    n = keep.sum(1, keepdim=True)
    p = keep / n.clamp(min=1)
    v, do = v.double(), do.double()
    return (p @ v, 2 * HALF * (p @ v.abs())), n[:, 0].log(), (p.T @ do, 2 * HALF * (p.T @ do.abs()))


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,H,behind,D", [([70, 200, 33], 2, 0, 64), ([70, 200, 33], 4, 0, 128), ([300, 64, 129], 20, 2200, 64), ([300, 64, 129], 20, 2200, 96),
                                             ([300, 64, 129], 20, 2200, 128), ([4200], 4, 0, 128)])
def test_packed(lens, H, behind, D, causal, scale):
    """Workgroups of 32 and of 128 queries, walks in parts."""
    from flame_amd import capi
    print(f"[scale] packed {lens=} {H=} {behind=} {D=} {causal=} {scale=}", flush=True)
    T = sum(lens) + behind
    q, k, v, do = rand(1, T, H, D), rand(2, T, H // 2, D), rand(3, T, H // 2, D), rand(4, T, H, D)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    dq, dk, dv, ddo, dcu = (t.cuda() for t in (q, k, v, do, cu))
    o, lse = capi.attn_packed_fwd(dq, dk, dv, dcu, dcu, scale, causal=causal)
    gq, gk, gv = capi.attn_packed_bwd(dq, dk, dv, o, ddo, lse, dcu, dcu, scale, causal=causal)
    for i in range(len(lens)):
        a, b = int(cu[i]), int(cu[i + 1])
        for c in range(H // 2):
            want, bound = torch.zeros((b - a, D), dtype=torch.float64), torch.zeros((b - a, D), dtype=torch.float64)
            for h in (2 * c, 2 * c + 1):
                (wo, bo), wl, (wv, bv) = of_head(q[a:b, h], k[a:b, c], v[a:b, c], do[a:b, h], causal)
                near("O", o[a:b, h], wo, bo)
                near("LSE", lse[h, a:b], wl, 1e-5 * (1 + wl))
                want, bound = want + wv, bound + bv
            near("dV", gv[a:b, c], want, bound)
    assert float(gq.abs().max()) <= 1e-25 * (scale > 1e-35) + 1e-30 and float(gk.abs().max()) <= 1e-25 * (scale > 1e-35) + 1e-30


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("B,H,Sq,Sk,D,causal", [(1, 2, 100, 77, 64, False), (2, 20, 700, 700, 128, True), (2, 40, 1024, 640, 64, False), (4, 32, 2048, 256, 128, False),
                                                (1, 2, 130, 300, 160, False), (2, 8, 512, 512, 256, False), (1, 4, 600, 400, 512, False)])
def test_dense(B, H, Sq, Sk, D, causal, scale):
    """Workgroups of 32, 128 and 256 queries, wide heads."""
    from flame_amd import capi
    print(f"[scale] dense {B=} {H=} {Sq=} {Sk=} {D=} {causal=} {scale=}", flush=True)
    q, k, v, do = rand(1, B, H, Sq, D), rand(2, B, H, Sk, D), rand(3, B, H, Sk, D), rand(4, B, H, Sq, D)
    dq, dk, dv, ddo = (t.cuda() for t in (q, k, v, do))
    o, lse = capi.attn_fwd(dq, dk, dv, scale, causal=causal)
    gv = capi.attn_bwd(dq, dk, dv, o, ddo, lse, scale, causal=causal)[2].cpu() if D <= 128 else None
    o, lse = o.cpu(), lse.view(B, H, Sq).cpu()
    for b, h in {(0, 0), (B - 1, H - 1), (0, H // 2)}:
        (wo, bo), wl, (wv, bv) = of_head(q[b, h], k[b, h], v[b, h], do[b, h], causal)
        near("O", o[b, h], wo, bo)
        near("LSE", lse[b, h], wl, 1e-5 * (1 + wl))
        if gv is not None:
            near("dV", gv[b, h], wv, bv)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("prefix", [0, 100])
def test_paged(prefix, scale):
    from flame_amd import capi
    print(f"[scale] paged {prefix=} {scale=}", flush=True)
    H, Hkv, D, page, lens = 4, 2, 64, 16, [100, 5, 3000]
    q, kc, vc = rand(1, 3, H, 1, D).cuda(), rand(2, 220, Hkv, page, D).cuda(), rand(3, 220, Hkv, page, D)
    table = torch.arange(3 * 200, dtype=torch.int32).view(3, 200) % 200
    pre = torch.arange(200, 207, dtype=torch.int32)
    extra = (pre.cuda(), torch.tensor([prefix], dtype=torch.int32).cuda()) if prefix else (None, None)
    o, lse = capi.attn_paged_fwd(q, kc, vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale, *extra, want_lse=True)
    for b, n in enumerate(lens):
        for h in range(H):
            v = torch.cat([vc[pre.long(), h // 2].reshape(-1, D)[:prefix], vc[table[b].long(), h // 2].reshape(-1, D)[:n]]).double()
            near("O", o[b, h, 0], v.mean(0), 2 * HALF * v.abs().mean(0))
            near("LSE", lse[b * H + h, 0], torch.tensor(math.log(prefix + n)), 1e-5 * (1 + math.log(prefix + n)))
