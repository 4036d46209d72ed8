"""Rotary positions against the formula in 64 bits on the CPU, forward and backward, the gradients against differences, too.

Tolerance.  Sine and cosine: the fraction of a turn is cut to 2^-32 of one (1.5e-9), its eighth becomes fp32 (2^-24 of at most pi / 4), the series
leaves out 2e-9 and each of its last two operations rounds by 2^-24: less than 2.5e-7 together.  The two products and their sum round three times by
2^-24, the size once more: fp32 results are off by at most 5e-7 size (|a| + |b|), which also bounds what is rounded; rounding to the type adds half a step."""
import math

import pytest
import torch

from flame_amd import capi, functional
from flame_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def reference(x, pos, rope, back=False):
    """(turned, bound) of x [..., tokens, heads, D] at pos [..., tokens]; float64"""
    R = rope.rotary_dim
    x = x.double().cpu()
    angle = pos.double().cpu()[..., None, None] * torch.tensor(rope.frequencies, dtype=torch.float64)
    c, s = angle.cos() * rope.size, angle.sin() * rope.size * (-1 if back else 1)
    first, second = (slice(0, R, 2), slice(1, R, 2)) if rope.interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., first], x[..., second]
    y, bound = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    bound[..., first] = bound[..., second] = 5e-7 * rope.size * (a.abs() + b.abs())
    return y, bound


def close(got, want, bound, dtype):
    half = torch.finfo(dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)       # half of the smallest step
    off = (got.double().cpu() - want).abs()
    assert (off <= bound + half * (want.abs() + bound) + tiny).all(), float((off / (bound + half * want.abs() + 1e-30)).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 64), (96, 64), (128, 32), (80, 80), (72, 24), (20, 6), (2, 2), (90, 46), (256, 192), (7, 4)])
def test_rows(dtype, interleaved, D, R):
    """Wide and narrow heads, whole and in part, positions near and far, in no order, negative."""
    g = torch.Generator().manual_seed(D + R)
    rope = Rotary(D, rotary_dim=R, interleaved=interleaved)
    pos = torch.tensor([0, 1, 2, 3, 7, 100, 4095, 65537, 1000003, 2 ** 24 + 1, 2 ** 31 - 1, -1, -12345, -2 ** 31, 5, 5, 9], dtype=torch.int32)
    q, k = (torch.randn((len(pos), H, D), generator=g).to(dtype) for H in (5, 2))
    print(f"[rotary] {dtype=} {interleaved=} {D=} {R=}", flush=True)
    yq, yk = functional.rotary(rope, q.cuda(), k.cuda(), positions=pos.cuda())
    alone = functional.rotary(rope, k.cuda(), positions=pos.cuda())
    assert yq.dtype == dtype and torch.equal(alone, yk)
    for x, y in ((q, yq), (k, yk)):
        close(y, *reference(x, pos, rope), dtype)
        assert torch.equal(y[..., R:].cpu(), x[..., R:])


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 32.0), ("bands", 8.0)])
def test_scaled(scaling, factor):
    rope = Rotary(128, base=500000.0, scaling=scaling, factor=factor, original_length=8192)
    pos = torch.arange(0, 262144, 4099, dtype=torch.int32)
    x = torch.randn((len(pos), 3, 128))
    close(functional.rotary(rope, x.cuda(), positions=pos.cuda()), *reference(x, pos, rope), torch.float32)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (32, 8), (24, 24), (5, 3)])
@pytest.mark.parametrize("lens,start", [([1], [0]), ([5, 0, 17, 300, 1], [0, 9, 1000, 3, 70000]), ([1] * 70, list(range(70))), ([3000], [131000])])
def test_packed(H, Hkv, lens, start):
    """Few rows and many (one head of a thread, and four), rows behind the last sequence."""
    rope = Rotary(128)
    n = sum(lens)
    pos = torch.cat([torch.arange(a, a + m) for a, m in zip(start, lens)]).to(torch.int32)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    q, k = (torch.randn((n + 3, h, 128)).to(torch.bfloat16) for h in (H, Hkv))
    yq, yk = functional.rotary(rope, q.cuda(), k.cuda(), cu_seqlens=cu, start=torch.tensor(start, dtype=torch.int32, device="cuda"))
    for x, y in ((q, yq), (k, yk)):
        close(y[:n], *reference(x[:n], pos, rope), torch.bfloat16)
        assert (y[n:] == 0).all()
    from_zero = functional.rotary(rope, q.cuda(), cu_seqlens=cu)
    pos0 = torch.cat([torch.arange(m) for m in lens]).to(torch.int32)
    close(from_zero[:n], *reference(q[:n], pos0, rope), torch.bfloat16)


@pytest.mark.parametrize("form", ["positions of all", "positions of each"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_batches(form, interleaved):
    """[B, H, S, D], contiguous, as a view of [B, S, H, D] (whose order the result keeps), with other strides."""
    B, H, S, D = 3, 4, 37, 64
    rope = Rotary(D, interleaved=interleaved, rotary_dim=48)
    pos = torch.randint(0, 5000, (B, S) if form.endswith("each") else (S,), dtype=torch.int32)
    x = torch.randn((B, S, H, D)).to(torch.bfloat16)
    want, bound = reference(x, pos if pos.dim() == 2 else pos.expand(B, S), rope)
    want, bound = want.transpose(1, 2), bound.transpose(1, 2)
    view = x.cuda().transpose(1, 2)
    y = functional.rotary(rope, view, positions=pos.cuda())
    assert y.stride() == view.stride()
    close(y, want, bound, torch.bfloat16)
    assert torch.equal(functional.rotary(rope, view.contiguous(), positions=pos.cuda()), y)
    odd = torch.zeros((B, H, S, D + 3), dtype=torch.bfloat16, device="cuda")[..., 1:D + 1]
    odd.copy_(view)
    assert torch.equal(functional.rotary(rope, odd, positions=pos.cuda()), y)          # not on 16 bytes: number by number
    apart = torch.zeros((B, H, S, 2 * D), dtype=torch.bfloat16, device="cuda")[..., ::2]
    apart.copy_(view)
    assert torch.equal(functional.rotary(rope, apart, positions=pos.cuda()), y)
    both = torch.zeros((B, 2 * S), dtype=torch.int32, device="cuda")[:, ::2]
    if pos.dim() == 2:
        wide = torch.zeros((B, S + 5), dtype=torch.int32, device="cuda")
        wide[:, 2:S + 2] = pos.cuda()
        assert torch.equal(functional.rotary(rope, view, positions=wide[:, 2:S + 2]), y)
        with pytest.raises(AssertionError):
            functional.rotary(rope, view, positions=both)
    one = functional.rotary(rope, view[:1, :1], positions=pos.cuda()[:1] if pos.dim() == 2 else pos.cuda())
    assert torch.equal(one, y[:1, :1])


def test_what_is_not_finite_stays_in_its_pair():
    rope = Rotary(64)
    x = torch.randn((4, 2, 64), device="cuda")
    x[1, 0, 3], x[2, 1, 40] = math.nan, math.inf
    y = functional.rotary(rope, x, positions=torch.arange(4, dtype=torch.int32, device="cuda"))
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 0, 3] = want[1, 0, 35] = want[2, 1, 40] = want[2, 1, 8] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (96, 64), (30, 14)])
def test_gradients(dtype, interleaved, D, R):
    """Against the formula: the turn backwards; rows behind the last sequence have none."""
    rope = Rotary(D, rotary_dim=R, interleaved=interleaved, scaling="yarn", factor=4.0)
    lens = [40, 3, 100]
    n = sum(lens)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    start = torch.tensor([0, 70000, 9], dtype=torch.int32)
    pos = torch.cat([torch.arange(int(a), int(a) + m) for a, m in zip(start, lens)])
    q, k = (torch.randn((n + 2, H, D), device="cuda").to(dtype).requires_grad_(True) for H in (6, 2))
    dq, dk = (torch.randn_like(x) for x in (q, k))
    out = functional.rotary(rope, q, k, cu_seqlens=cu, start=start.cuda())
    gq, gk = torch.autograd.grad(out, (q, k), (dq, dk))
    for d, g in ((dq, gq), (dk, gk)):
        close(g[:n], *reference(d[:n], pos, rope, back=True), dtype)
        assert (g[n:] == 0).all()
    for x, y in ((q, out[0]), (k, out[1])):
        close(y[:n].detach(), *reference(x[:n].detach(), pos, rope), dtype)


def test_gradients_against_differences():
    """The operator is linear: (f(x + e d) - f(x)) . w / e is <grad, d> up to fp32 rounding, 1e-5 of the sum of magnitudes."""
    rope = Rotary(32, rotary_dim=20)
    pos = torch.tensor([[0, 5, 1000], [3, 77777, 1]], dtype=torch.int32, device="cuda")
    x = torch.randn((2, 3, 3, 32), device="cuda", requires_grad=True)
    w, d = torch.randn_like(x), torch.randn_like(x)
    y = functional.rotary(rope, x, positions=pos)
    (g,) = torch.autograd.grad(y, x, w)
    with torch.no_grad():
        change = (functional.rotary(rope, x + d, positions=pos).double() - y.double()) * w.double()
    assert abs(float(change.sum() - (g.double() * d.double()).sum())) <= 1e-5 * float(change.abs().sum())


def test_broadcast_leaves_and_second_derivatives():
    """A leaf expanded over heads gets the sum of their gradients; of an upstream gradient without strides too; f is derived as often as wanted."""
    rope = Rotary(64)
    pos = torch.arange(10, dtype=torch.int32, device="cuda")
    leaf = torch.randn((10, 1, 64), device="cuda", requires_grad=True)
    y = functional.rotary(rope, leaf.expand(10, 6, 64), positions=pos)
    (g,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    want, bound = reference(torch.ones((10, 1, 64)), pos, rope, back=True)
    assert ((g.double().cpu() - 6 * want).abs() <= 6 * bound + 2.0 ** -20).all()
    x = torch.randn((10, 2, 64), device="cuda", requires_grad=True)
    w = torch.randn((10, 2, 64), device="cuda", requires_grad=True)
    (gx,) = torch.autograd.grad(functional.rotary(rope, x, positions=pos), x, w, create_graph=True)
    v = torch.randn_like(gx)
    (gw,) = torch.autograd.grad(gx, w, v)
    want, bound = reference(v, pos, rope)
    close(gw, want, bound, torch.float32)
    q = torch.randn((10, 2, 64), device="cuda", requires_grad=True)
    yq, yk = functional.rotary(rope, q, x.detach(), positions=pos)
    yq.sum().backward()                                    # the other result has no gradient
    assert q.grad is not None
    yq, yk = functional.rotary(rope, q.detach(), x, positions=pos)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        pos += 1
        yk.sum().backward()


@pytest.mark.parametrize("which", [0, 1])
def test_only_one_requires_a_gradient(which):
    """The other's result requires none, and is taken where that is refused."""
    rope = Rotary(64)
    pos = torch.arange(10, dtype=torch.int32, device="cuda")
    x = [torch.randn((10, 4, 64), device="cuda"), torch.randn((10, 2, 64), device="cuda")]
    both = functional.rotary(rope, *x, positions=pos)
    x[which].requires_grad_(True)
    y = functional.rotary(rope, *x, positions=pos)
    assert y[which].requires_grad and not y[1 - which].requires_grad and all(torch.equal(a, b) for a, b in zip(y, both))
    w = torch.randn_like(y[which])
    (g,) = torch.autograd.grad((y[which] * w).sum() + y[1 - which].sum(), x[which])
    close(g, *reference(w, pos, rope, back=True), torch.float32)


def test_captured():
    """Forward and backward in a graph, replayed on new inputs and positions; an eager graph of the same leaf that lives on is refused."""
    rope = Rotary(128, interleaved=True)
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    leaf = torch.randn((50, 4, 128), device="cuda").to(torch.bfloat16).requires_grad_(True)
    w = torch.randn_like(leaf)

    def step():
        y = functional.rotary(rope, leaf, positions=pos)
        return y.detach(), torch.autograd.grad(y, leaf, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = step()
    for _ in range(4):
        with torch.no_grad():
            leaf.normal_()
            w.normal_()
            pos += 31
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(g, want[1])
    alive = functional.rotary(rope, leaf, positions=pos)
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive


def test_as_packed_attention_takes_it():
    """Rotary positions and packed attention in training: the gradients of the chain are those of the parts."""
    rope = Rotary(64)
    lens = [33, 5, 70]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    n = sum(lens)
    q, k, v = (torch.randn((n, H, 64), device="cuda").to(torch.bfloat16).requires_grad_(True) for H in (4, 2, 2))
    do = torch.randn((n, 4, 64), device="cuda").to(torch.bfloat16)
    tq, tk = functional.rotary(rope, q, k, cu_seqlens=cu)
    o = functional.sdpa_packed(tq, tk, v, cu, is_causal=True)
    gq, gk, gv = torch.autograd.grad(o, (q, k, v), do)
    leaves = [t.detach().requires_grad_(True) for t in (tq, tk, v)]
    hq, hk, hv = torch.autograd.grad(functional.sdpa_packed(*leaves, cu, is_causal=True), leaves, do)
    assert torch.equal(gv, hv)
    assert torch.equal(gq, capi.rotary(hq, None, rope.turns_on(hq.device), cu_seqlens=cu, inverse=True))
    assert torch.equal(gk, capi.rotary(hk, None, rope.turns_on(hq.device), cu_seqlens=cu, inverse=True))
