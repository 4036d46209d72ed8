"""Bounds on the device that fall or lead outside: every kernel of the packed calls, its outputs and its workspace between guards.  And the gradients
of a backward on another stream, whose inputs arrive late."""
import random

import pytest
import torch

from tests.test_gpu_packed import make

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


class Guarded:
    """Tensors in the middle of larger ones."""

    def __init__(self):
        self.made = []

    def like(self, shape, dtype, value):
        n = 1
        for s in shape:
            n *= s
        room = torch.full((n + 2 * GUARD,), value, dtype=dtype, device="cuda")
        self.made.append((room, n, value))
        return room[GUARD:GUARD + n].view(shape)

    def intact(self):
        return all(bool((room[:GUARD] == value).all()) and bool((room[GUARD + n:] == value).all()) for room, n, value in self.made)


def wild(rng, n, T):
    """n + 1 bounds that nobody should pass."""
    yield [0] + [T + 400] * n
    yield [rng.choice([-5, 2 ** 31 - 1, -2 ** 31, T]) for _ in range(n + 1)]
    yield [T if i % 2 else 0 for i in range(n + 1)]
    yield [0 if i % 2 else T for i in range(n + 1)]
    yield sorted((rng.randint(-T, 2 * T) for _ in range(n + 1)), reverse=True)
    yield [rng.randint(-10, T + 10) for _ in range(n + 1)]


# few rows whose wavefronts share the keys (eight and four), walks in parts, whole walks of 128 rows, a search among more than 64 sequences
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T_q,T_k,n,H,Hkv,D,room", [(100, 100, 2, 4, 2, 64, False), (700, 650, 3, 10, 5, 96, False), (4200, 4200, 3, 4, 2, 128, True), (130, 5000, 2, 4, 2, 64, True),
                                                   (1200, 1100, 2, 10, 5, 128, False), (2600, 2500, 5, 20, 4, 128, False), (2600, 2600, 64, 20, 4, 64, False), (2600, 2500, 70, 4, 2, 64, False),
                                                   (300, 300, 4200, 2, 1, 96, False)])
def test_wild_bounds(T_q, T_k, n, H, Hkv, D, room, causal):
    from flame_amd import capi
    rng = random.Random(T_q + n)
    q, k, v, do, _, _ = (t.cuda() for t in make(n, [T_q], [T_k], H, Hkv, D))
    kept = [t.clone() for t in (q, k, v, do)]
    fwd_bytes, bwd_bytes = capi.packed_fwd_workspace_bytes(n, T_q, T_k, H, D), capi.packed_bwd_workspace_bytes(n, T_q, T_k, H, Hkv, D)
    assert (fwd_bytes > 0) == room
    for a, b in zip(wild(rng, n, T_q), list(wild(rng, n, T_k))[::-1 if n % 2 else 1]):
        print(f"[wild] {T_q=} {T_k=} {n=} {H=} {Hkv=} {D=} {causal=} {a[:4]=} {b[:4]=}", flush=True)
        cq, ck = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (a, b))
        g = Guarded()
        o, lse = g.like((T_q, H, D), torch.bfloat16, 7.0), g.like((H, T_q), torch.float32, 7.0)
        ws = g.like((max(fwd_bytes, 16),), torch.uint8, 7)
        capi.attn_packed_fwd(q, k, v, cq, ck, 0.125, causal=causal, out=o, lse_out=lse, workspace=ws)
        torch.cuda.synchronize()
        assert g.intact()
        grads = tuple(g.like(t.shape, torch.bfloat16, 7.0) for t in (q, k, v))
        capi.attn_packed_bwd(q, k, v, torch.nan_to_num(o), do, torch.nan_to_num(lse), cq, ck, 0.125, causal=causal, workspace=g.like((bwd_bytes,), torch.uint8, 7), grads=grads)
        torch.cuda.synchronize()
        assert g.intact() and all(torch.equal(x, y) for x, y in zip(kept, (q, k, v, do)))


def test_right_bounds_between_guards():
    """... and the guards do not keep a right call from its results."""
    from flame_amd import capi
    lens = [4000, 100, 100]
    q, k, v, do, cq, ck = (t.cuda() for t in make(1, lens, lens, 4, 2, 128))
    want = capi.attn_packed_fwd(q, k, v, cq, ck, 0.1)
    want_g = capi.attn_packed_bwd(q, k, v, want[0], do, want[1], cq, ck, 0.1)
    g = Guarded()
    o, lse = g.like(q.shape, torch.bfloat16, 7.0), g.like((4, len(q)), torch.float32, 7.0)
    capi.attn_packed_fwd(q, k, v, cq, ck, 0.1, out=o, lse_out=lse, workspace=g.like((capi.packed_fwd_workspace_bytes(3, len(q), len(k), 4, 128),), torch.uint8, 7))
    grads = tuple(g.like(t.shape, torch.bfloat16, 7.0) for t in (q, k, v))
    capi.attn_packed_bwd(q, k, v, o, do, lse, cq, ck, 0.1, workspace=g.like((capi.packed_bwd_workspace_bytes(3, len(q), len(k), 4, 2, 128),), torch.uint8, 7), grads=grads)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and all(torch.equal(x, y) for x, y in zip(grads, want_g)) and g.intact()


@pytest.mark.parametrize("lens,H", [((500, 300), 4), ((4200,), 2)])
def test_gradients_on_another_stream(lens, H):
    """The inputs are written on that stream after a wait of some milliseconds: a kernel on any other stream would read what was there before."""
    from flame_amd import functional
    q, k, v, do, cq, _ = (t.cuda() for t in make(4, list(lens), list(lens), H, H // 2, 64))
    want = []
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = functional.sdpa_packed(*leaves, cq, is_causal=True)
    o.backward(do)
    want = [o.detach(), *(t.grad for t in leaves)]
    late = [torch.zeros_like(t) for t in (q, k, v, do)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        for x, t in zip(late, (q, k, v, do)):
            x.copy_(t)
        leaves = [t.detach().requires_grad_(True) for t in late[:3]]
        o = functional.sdpa_packed(*leaves, cq, is_causal=True)
    o.backward(late[3])                     # called under the default stream: autograd goes back to the forward's
    side.synchronize()
    torch.cuda.synchronize()
    for name, a, b in zip(("O", "dQ", "dK", "dV"), want, (o.detach(), *(t.grad for t in leaves))):
        assert torch.equal(a, b), name
