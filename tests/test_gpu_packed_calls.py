"""The calls around the kernels of packed sequences: autograd, other dtypes and layouts, captured graphs, another stream,
differences of the function itself."""
import math

import pytest
import torch

from tests.test_gpu_packed import check, make, reference

pytestmark = pytest.mark.gpu


def inputs(seed=1, lens=(100, 1, 70), H=4, Hkv=2, D=64):
    q, k, v, do, cq, ck = make(seed, list(lens), list(lens), H, Hkv, D)
    return (q, k, v, do, cq, ck), [t.cuda() for t in (q, k, v, do, cq, ck)]


def test_autograd_gives_the_gradients_of_the_calls():
    from flame_amd import capi, functional
    host, (q, k, v, do, cq, ck) = inputs()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = functional.sdpa_packed(*leaves, cq, is_causal=True)
    o.backward(do)
    want, lse = capi.attn_packed_fwd(q, k, v, cq, ck, 0.125)
    grads = capi.attn_packed_bwd(q, k, v, want, do, lse, cq, ck, 0.125)
    assert torch.equal(o, want) and all(torch.equal(x.grad, g) for x, g in zip(leaves, grads))
    z, _ = reference(*host, 0.125, True)
    check("O", o.detach().cpu(), *z["O"])
    with torch.no_grad():
        assert torch.equal(functional.sdpa_packed(*leaves, cq, ck, is_causal=True), want)
    # only one input wants a gradient; no causal flag; another scale
    k2 = k.clone().requires_grad_(True)
    functional.sdpa_packed(q, k2, v, cq, scale=0.3).backward(do)
    o3, l3 = capi.attn_packed_fwd(q, k, v, cq, ck, 0.3, causal=False)
    assert torch.equal(k2.grad, capi.attn_packed_bwd(q, k, v, o3, do, l3, cq, ck, 0.3, causal=False)[1])


def test_other_dtypes_and_layouts():
    from flame_amd import functional
    host, (q, k, v, do, cq, ck) = inputs()
    want = functional.sdpa_packed(q, k, v, cq, is_causal=True)
    f = [t.float().requires_grad_(True) for t in (q, k, v)]
    o = functional.sdpa_packed(*f, cq, is_causal=True)
    assert o.dtype == torch.float32 and torch.equal(o.bfloat16(), want)
    o.backward(do.float())
    b = [t.clone().requires_grad_(True) for t in (q, k, v)]
    functional.sdpa_packed(*b, cq, is_causal=True).backward(do)
    assert all(x.grad.dtype == torch.float32 and torch.equal(x.grad.bfloat16(), y.grad) for x, y in zip(f, b))
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(q).copy_(q)      # two bytes past 16
    turned = k.permute(2, 0, 1).contiguous().permute(1, 2, 0)                                           # D not contiguous
    assert torch.equal(functional.sdpa_packed(odd, turned, v, cq, is_causal=True), want)
    b[0].grad = None
    functional.sdpa_packed(*b, cq, is_causal=True).backward(do.permute(2, 0, 1).contiguous().permute(1, 2, 0))
    g = b[0].grad.clone()
    b[0].grad = None
    functional.sdpa_packed(*b, cq, is_causal=True).backward(do)
    assert torch.equal(g, b[0].grad)


def test_broadcast_inputs():
    """Keys and values expanded over the heads: one gradient of the sum."""
    from flame_amd import functional
    host, (q, k, v, do, cq, ck) = inputs(H=4, Hkv=1)
    a = [t.clone().requires_grad_(True) for t in (k, v)]
    functional.sdpa_packed(q, *(t.expand(-1, 4, -1) for t in a), cq, is_causal=True).backward(do)
    z, _ = reference(*host, 0.125, True)
    for name, t in zip(("dK", "dV"), a):       # four heads' gradients, rounded one by one, and their sum rounded again
        value, bound = z[name]
        assert ((t.grad.cpu().double() - value).abs() <= 2 * bound + 2.0 ** -8 * value.abs()).all()


def test_differences():
    """The gradients along a direction against differences of L = sum(O dO) in 64 bits: off by at most their own bound along the
    direction, and by what the difference is off the derivative (third order in the step; taken from the 64-bit gradient)."""
    from flame_amd import functional
    (q, k, v, do, cq, ck), _ = inputs(5, lens=(60, 33))
    z, _ = reference(q, k, v, do, cq, ck, 0.125, True)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    functional.sdpa_packed(*leaves, cq.cuda(), is_causal=True).backward(do.cuda())
    for i, name in enumerate(("dQ", "dK", "dV")):
        step = z[name][0].sign() / 64
        ends = []
        for s in (1, -1):
            moved = [t.double() for t in (q, k, v)]
            moved[i] = moved[i] + s * step
            ends.append((reference(*moved, do, cq, ck, 0.125, True)[0]["O"][0] * do.double()).sum())
        difference = float(ends[0] - ends[1]) / 2
        off = abs(float((z[name][0] * step).sum()) - difference)
        assert off <= 0.02 * abs(difference)
        assert abs(float((leaves[i].grad.cpu().double() * step).sum()) - difference) <= off + float((z[name][1] * step.abs()).sum()), name


def test_graph_of_forward_and_backward_calls():
    from flame_amd import capi
    _, (q, k, v, do, cq, ck) = inputs(2, lens=(300, 77, 129))
    ws = torch.empty(capi.packed_bwd_workspace_bytes(3, len(q), len(k), 4, 2, 64), dtype=torch.uint8, device="cuda")
    o, grads = torch.empty_like(q), tuple(torch.empty_like(t) for t in (q, k, v))

    def step(o, grads, ws):
        _, lse = capi.attn_packed_fwd(q, k, v, cq, ck, 0.125, out=o)
        capi.attn_packed_bwd(q, k, v, o, do, lse, cq, ck, 0.125, workspace=ws, grads=grads)
        return lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(o, grads, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        lse = step(o, grads, ws)
    for rep in range(3):
        g = torch.Generator(device="cuda").manual_seed(rep)
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g) * (1 + rep))
        cut = torch.tensor([0, 100 + rep, 250, 506 - rep], dtype=torch.int32, device="cuda")       # other lengths in the same buffers
        cq.copy_(cut)
        ck.copy_(cut)
        graph.replay()
        torch.cuda.synchronize()
        o2, g2 = torch.empty_like(o), tuple(torch.empty_like(t) for t in grads)
        l2 = step(o2, g2, torch.empty_like(ws))
        torch.cuda.synchronize()
        assert torch.equal(o, o2) and torch.equal(lse, l2) and all(torch.equal(a, b) for a, b in zip(grads, g2))


def test_graph_of_autograd():
    """A captured backward, and the refusal of one whose leaves a graph of another stream holds."""
    from flame_amd import functional
    _, (q, k, v, do, cq, ck) = inputs(3)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        functional.sdpa_packed(*leaves, cq, is_causal=True).backward(do)
        for t in leaves:
            t.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = functional.sdpa_packed(*leaves, cq, is_causal=True)
        o.backward(do)
    for rep in range(3):
        with torch.no_grad():
            for t, seed in zip(leaves, (1, 2, 3)):
                t.copy_(torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + rep)))
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
        functional.sdpa_packed(*fresh, cq, is_causal=True).backward(do)
        torch.cuda.synchronize()
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(leaves, fresh))
    held = [t.detach().clone().requires_grad_(True) for t in leaves]
    eager = functional.sdpa_packed(*held, cq, is_causal=True)          # on the default stream, alive
    torch.cuda.synchronize()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other, stream=side):
        with pytest.raises(RuntimeError, match="another stream"):
            functional.sdpa_packed(*held, cq, is_causal=True)
    del eager
    both = torch.cat([q, k, v], 1).requires_grad_(True)                # one leaf, seen by views
    parts = lambda: (both[:, :4], both[:, 4:4 + k.shape[1]], both[:, 4 + k.shape[1]:])
    eager = functional.sdpa_packed(*parts(), cq, is_causal=True)
    torch.cuda.synchronize()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other, stream=side):
        with pytest.raises(RuntimeError, match="another stream"):
            functional.sdpa_packed(*parts(), cq, is_causal=True)
    del eager


def test_a_second_derivative_is_refused():
    from flame_amd import functional
    _, (q, k, v, do, cq, ck) = inputs()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = functional.sdpa_packed(*leaves, cq, is_causal=True)
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(o, leaves, do, create_graph=True)
    again = torch.autograd.grad(o, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_another_stream():
    from flame_amd import functional
    _, (q, k, v, do, cq, ck) = inputs(4, lens=(500, 300))
    want = functional.sdpa_packed(q, k, v, cq, is_causal=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fresh = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = functional.sdpa_packed(*fresh, cq, is_causal=True)
        o.backward(do)
    side.synchronize()
    assert torch.equal(o, want)


def test_refusals_on_the_device():
    from flame_amd import capi, functional
    _, (q, k, v, do, cq, ck) = inputs()
    for bad in ((q, k.cpu(), v, cq), (q, k, v, cq.cpu()), (q, k[:-1], v, cq), (q[:, :3], k, v, cq), (q, k, v, cq[::2][:2]), (q, k, v, cq.to(torch.int64))):
        with pytest.raises(AssertionError):
            functional.sdpa_packed(*bad)
    with pytest.raises(AssertionError):
        functional.sdpa_packed(q, k, v, cq, cq[:3])
    with pytest.raises(AssertionError):
        capi.attn_packed_fwd(q.float(), k, v, cq, ck, 0.1)
    with pytest.raises(AssertionError):
        capi.attn_packed_fwd(q, k, v, cq, ck, 0.1, lse_out=torch.empty((len(q), 4), device="cuda"))
    with pytest.raises(capi.FlameAttnError):
        capi.attn_packed_fwd(q, k, v, cq, ck, -1.0)
    with pytest.raises(capi.FlameAttnError):
        functional.sdpa_packed(*(torch.zeros((10, 2, 136), dtype=torch.bfloat16, device="cuda") for _ in range(3)), torch.tensor([0, 10], dtype=torch.int32, device="cuda"))
    with pytest.raises(capi.FlameAttnError):
        capi.attn_packed_fwd(q, k, v, cq, ck, 0.1, out=torch.empty((1, 4, 64), dtype=torch.bfloat16, device="cuda").expand(len(q), 4, 64))


def test_bounds_that_lead_outside_touch_nothing_outside():
    """cu cannot be refused; what it says is cut to the tensors (the rows of a wider buffer around them stay as they were)."""
    from flame_amd import capi
    _, (q, k, v, do, cq, ck) = inputs(6, lens=(60, 40))
    room = torch.full((300, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    for wild in ([0, 60, 500], [0, -5, 100], [9, 90, 20], [0, 2 ** 31 - 1, -2 ** 31]):
        cu = torch.tensor(wild, dtype=torch.int32, device="cuda")
        out = room[100:200]
        o, lse = capi.attn_packed_fwd(q, k, v, cu, cu, 0.125, out=out)
        capi.attn_packed_bwd(q, k, v, torch.nan_to_num(o), do, lse, cu, cu, 0.125)
        torch.cuda.synchronize()
        assert bool((room[:100] == 7).all()) and bool((room[200:] == 7).all())
