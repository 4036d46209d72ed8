"""Root-mean-square errors of the packed and paged calls, sequence by sequence and head by head.  A bound of every element has to cover the sum
of all roundings' magnitudes, and on long walks that exceeds the result itself, which is a sum of many terms of either sign: a step that is left
out of a walk stays below it.  The root of the mean square does not.

Expected error.  A rounding to bf16 is off by at most half a step, 2^-8 of the value, and evenly spread, so its variance is at most
r^2 = (2^-8)^2 / 3 of the value's square.  Roundings of different elements are independent, so variances add up:
  O   = round(sum_j round(P_ij) v_j):                          V(O)  = r^2 sum_j P^2 v^2 + r^2 O^2
  delta = sum_d dO O with the O above:                         V(delta_i) = r^2 sum_j P^2 (dO v_j)^2 + r^2 sum_d (dO O)^2
  dQ  = round(scale sum_j round(P (dO v - delta)) k_j):        V(dQ) = scale^2 (r^2 sum_j dS^2 k^2 + V(delta_i) (sum_j P k)^2) + r^2 dQ^2
  dK  = round(scale sum_h sum_i round(dS) q_i):                V(dK) = scale^2 sum_h sum_i (r^2 dS^2 + P^2 V(delta_i)) q^2 + r^2 dK^2
  dV  = round(sum_h sum_i round(P) dO_i):                      V(dV) = r^2 sum_h sum_i P^2 dO^2 + r^2 dV^2
Everything else is fp32, 2^-16 of that.  Over the rows of a sequence and head, at least 64 of them, the mean of the squared errors may exceed the mean of
these variances by chance only: by less than four times (a factor of two of the root), also where ten rows make up most of it (a sum of ten squares is seven times
its expectation, as the spread of real mantissas makes the true r^2 0.54 of the one above, once in 10^9)."""
import math

import pytest
import torch

from tests.test_gpu_packed import make

R2 = (2.0 ** -8) ** 2 / 3


def bf(x):
    return x.to(torch.bfloat16).to(x.dtype)


def parts_of(q, k, v, do, scale, causal, rounded=False, skip=None):
    """One sequence and head in 64 bits (rounded: with the roundings that the kernels make): O, dQ, what it adds to dK and dV, and the variances.
    skip: (name, rows) of the walked rows whose products the named result leaves out."""
    n = bf if rounded else (lambda x: x)
    s = q @ k.T * scale
    if causal:
        s = s.masked_fill(~torch.ones(s.shape, dtype=torch.bool, device=s.device).tril(s.shape[1] - s.shape[0]), -math.inf)
    p = torch.exp(s - torch.nan_to_num(torch.logsumexp(s, 1, keepdim=True), neginf=0.0))

    def walk(name, size):
        w = torch.ones(size, dtype=q.dtype, device=q.device)
        if skip and skip[0] == name:
            w[skip[1]] = 0
        return w[:, None]

    o = n((n(p) * walk("O", len(k)).T) @ v)
    delta = (do * o).sum(1, keepdim=True)
    dp = do @ v.T
    ds = n(p * (dp - delta))
    dq = n((ds * walk("dQ", len(k)).T) @ k * scale)
    dk = (ds * walk("dK", len(q))).T @ q * scale
    dv = (n(p) * walk("dV", len(q))).T @ do
    if rounded:
        return o, dq, dk, dv
    p2 = p * p
    var_delta = R2 * ((p2 * dp * dp).sum(1, keepdim=True) + (do * do * o * o).sum(1, keepdim=True))
    return (o, dq, dk, dv), (R2 * (p2 @ v ** 2 + o ** 2), scale ** 2 * (R2 * (ds * ds) @ k ** 2 + var_delta * (p @ k) ** 2) + R2 * dq ** 2,
                             scale ** 2 * (R2 * ds * ds + p2 * var_delta).T @ q ** 2, R2 * p2.T @ do ** 2)


def ratios(got, q, k, v, do, cq, ck, scale, causal):
    """(name, sequence, head, root of mean square error over mean variance) of O, dQ, dK, dV, where a sequence has 64 rows or more."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    G = q.shape[1] // k.shape[1]
    out = []

    def put(name, i, h, value, want, var):
        if len(want) >= 64:
            out.append((name, i, h, float(((value.double() - want) ** 2).mean() / var.mean()) ** 0.5))

    for i in range(len(cq) - 1):
        Q, K = slice(int(cq[i]), int(cq[i + 1])), slice(int(ck[i]), int(ck[i + 1]))
        if Q.stop == Q.start or K.stop == K.start:
            continue
        for c in range(k.shape[1]):
            sums = [0.0] * 4
            for h in range(c * G, c * G + G):
                (o, dq, dk, dv), (vo, vq, vk, vv) = parts_of(q[Q, h], k[K, c], v[K, c], do[Q, h], scale, causal)
                put("O", i, h, got[0][Q, h], o, vo)
                put("dQ", i, h, got[1][Q, h], dq, vq)
                sums = [a + b for a, b in zip(sums, (dk, vk, dv, vv))]
            dk, vk, dv, vv = sums
            put("dK", i, c, got[2][K, c], dk, vk + R2 * dk ** 2)
            put("dV", i, c, got[3][K, c], dv, vv + R2 * dv ** 2)
    return out


# ------------------------------------------------------------------------------------------------ the check itself, without a GPU
def imitated(q, k, v, do, scale, causal, skip=None, head=0):
    """What the kernels compute of one sequence whose heads share one key head, the step in `skip` left out for one head."""
    heads = [parts_of(q[:, h], k[:, 0], v[:, 0], do[:, h], scale, causal, rounded=True, skip=skip if h == head else None) for h in range(q.shape[1])]
    o, dq = (torch.stack([x[i] for x in heads], 1) for i in (0, 1))
    return (o, dq, *(bf(sum(x[i] for x in heads))[:, None] for i in (2, 3)))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [(100, 5000), (700, 700), (64, 64), (129, 700)])
def test_the_check_passes_the_roundings_and_nothing_else(lq, lk, causal):
    q, k, v, do, cq, ck = make(lq, [lq], [lk], 2, 1, 64)
    args = [t.double() for t in (q, k, v, do)]
    right = ratios(imitated(*args, 0.125, causal), q, k, v, do, cq, ck, 0.125, causal)
    assert {r[0] for r in right} == {"O", "dQ", "dK", "dV"} and max(r[3] for r in right) <= 1.2, right
    for name, n in (("O", lk), ("dQ", lk), ("dK", lq), ("dV", lq)):
        at = 64 * (n // 128)                    # one step of 64 rows in the middle (under the causal flag most rows have it)
        wrong = ratios(imitated(*args, 0.125, causal, (name, slice(at, at + 64))), q, k, v, do, cq, ck, 0.125, causal)
        off = [r for r in wrong if r[0] == name and (name in ("dK", "dV") or r[2] == 0)]
        assert off and min(r[3] for r in off) > 4, (name, off)


# ------------------------------------------------------------------------------------------------ the kernels
def fine(found):
    worst = max(found, key=lambda r: r[3])
    print(f"[rms] {len(found)} sequences and heads, worst {worst}", flush=True)
    assert worst[3] <= 2, worst


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("lq,lk,H,Hkv,behind", [
    ([100, 5, 129], [5000, 1300, 129], 4, 2, 0), ([4200], [4200], 4, 2, 0), ([2500, 40, 1700], [2500, 40, 1600], 4, 2, 0),       # walks in parts
    ([4096, 1101, 333], [4096, 1101, 333], 16, 4, 0), ([300, 64, 513], [300, 640, 513], 20, 4, 2200),                              # whole walks of 128 rows
    ([700, 65, 400], [700, 65, 400], 10, 5, 0), ([31] * 70 + [700], [31] * 70 + [700], 4, 1, 40)])                                # few rows; a search for the sequence
def test_packed(lq, lk, H, Hkv, behind, D, causal):
    from flame_amd import capi
    print(f"[rms] {lq[-3:]=} {lk[-3:]=} {H=} {Hkv=} {D=} {causal=} {behind=}", flush=True)
    q, k, v, do, cq, ck = (t.cuda() for t in make(sum(lq) + D, lq, lk, H, Hkv, D, behind))
    o, lse = capi.attn_packed_fwd(q, k, v, cq, ck, D ** -0.5, causal=causal)
    grads = capi.attn_packed_bwd(q, k, v, o, do, lse, cq, ck, D ** -0.5, causal=causal)
    fine(ratios((o, *grads), q, k, v, do, cq.tolist(), ck.tolist(), D ** -0.5, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("lens,H,Hkv,N,prefix", [([900, 1000, 700], 16, 4, 1, 0), ([20001, 9000], 16, 4, 1, 0), ([5000] * 5, 32, 8, 4, 0), ([300, 4000, 70], 16, 4, 1, 5000),
                                                 ([37 * i % 500 + 70 for i in range(40)], 8, 2, 1, 8000), ([3000, 500] * 10, 32, 32, 1, 0)])
def test_paged(lens, H, Hkv, N, prefix, D):
    """Walks by one workgroup and in units, a prefix whose units take up to 64 rows and 128; the rows of a sequence (its heads and tokens) together."""
    from flame_amd import capi
    print(f"[rms] paged {lens[:3]=} {H=} {Hkv=} {N=} {D=} {prefix=}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(D + N)
    page = 16
    need = [-(-n // page) for n in [prefix] + lens]
    order = torch.randperm(sum(need), device="cuda", generator=g).to(torch.int32)
    kc, vc = (torch.randn((sum(need), Hkv, page, D), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((len(lens), H, N, D), device="cuda", generator=g).to(torch.bfloat16)
    rows = list(order.split(need))
    table = torch.zeros((len(lens), max(need[1:])), dtype=torch.int32, device="cuda")
    for b, r in enumerate(rows[1:]):
        table[b, :len(r)] = r
    extra = (rows[0], torch.tensor([prefix], dtype=torch.int32, device="cuda")) if prefix else (None, None)
    o, _ = capi.attn_paged_fwd(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), D ** -0.5, *extra)
    found = []
    for b, n in enumerate(lens):
        error = variance = 0.0
        for c in range(Hkv):
            k, v = (torch.cat([x[rows[0].long(), c].reshape(-1, D)[:prefix], x[rows[1 + b].long(), c].reshape(-1, D)[:n]]).double() for x in (kc, vc))
            for h in range(c * (H // Hkv), (c + 1) * (H // Hkv)):
                s = (q[b, h].double() @ k.T * D ** -0.5).masked_fill(~torch.ones((N, len(k)), dtype=torch.bool, device="cuda").tril(len(k) - N), -math.inf)
                p = torch.softmax(s, 1)
                want = p @ v
                error += float(((o[b, h].double() - want) ** 2).sum())
                variance += float((R2 * (p ** 2 @ v ** 2 + want ** 2)).sum())
        found.append(("O", b, "all", (error / variance) ** 0.5))
    fine(found)
