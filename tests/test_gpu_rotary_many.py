"""Rotary positions of so many rows that a thread serves several heads (csrc/rotary_rule.hpp), in every form: types, halves and neighbours, parts of the head, 16-byte and narrow
accesses, numbers of heads that four does not divide, positions of rows, of all tokens and of each, bounds.  Against the formula in 64 bits with the
tolerance of test_gpu_rotary, and bit for bit against the same rows in small pieces, which one head of a thread serves."""
import pytest
import torch

from flame_amd import functional
from flame_amd.rotary import Rotary
from tests.test_gpu_rotary import DTYPES, close, reference

pytestmark = pytest.mark.gpu


def rand(*shape, dtype):
    return torch.randn(shape, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,H,Hkv,rows", [(128, 128, 9, 2, 9000), (64, 32, 5, 1, 32000), (30, 14, 6, 3, 6000), (96, 24, 3, 0, 12000)])
def test_rows(dtype, interleaved, D, R, H, Hkv, rows):
    rope = Rotary(D, rotary_dim=R, interleaved=interleaved, base=500000.0)
    pos = torch.randint(-2 ** 24, 2 ** 24, (rows,)).to(torch.int32)
    x = [rand(rows, h, D, dtype=dtype) for h in (H, Hkv) if h]
    print(f"[rotary] {dtype=} {interleaved=} {D=} {R=} {H=} {Hkv=} {rows=}", flush=True)
    y = functional.rotary(rope, *x, positions=pos.cuda())
    y = y if Hkv else (y,)
    for a, b in zip(x, y):
        close(b, *reference(a, pos, rope), dtype)
        assert torch.equal(b[..., R:], a[..., R:])
        for at in range(0, rows, 997):
            assert torch.equal(functional.rotary(rope, a[at:at + 100], positions=pos[at:at + 100].cuda()), b[at:at + 100])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("each", [False, True])
def test_batches_of_views(dtype, interleaved, each):
    """[B, H, S, D] out of [B, S, H, D]: 16-byte rows, and one number off them; positions of each token with a step between the rows."""
    B, S, H, D = 5, 4000, 7, 80
    rope = Rotary(D, rotary_dim=48, interleaved=interleaved)
    pos = torch.randint(0, 200000, (B, S + 3), device="cuda").to(torch.int32)[:, 1:S + 1] if each else torch.randint(0, 200000, (S,), device="cuda").to(torch.int32)
    x = rand(B, S, H, D, dtype=dtype).transpose(1, 2)
    print(f"[rotary] {dtype=} {interleaved=} {each=}", flush=True)
    y = functional.rotary(rope, x, positions=pos)
    close(y.transpose(1, 2), *reference(x.transpose(1, 2), (pos if each else pos.expand(B, S)).cpu(), rope), dtype)
    odd = torch.zeros((B, H, S, D + 8), dtype=dtype, device="cuda")[..., 1:D + 1]
    odd.copy_(x)
    assert torch.equal(functional.rotary(rope, odd, positions=pos), y)
    for b in range(B):
        assert torch.equal(functional.rotary(rope, x[b:b + 1, :, 100:200], positions=pos[b:b + 1, 100:200] if each else pos[100:200]), y[b:b + 1, :, 100:200])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,seqs", [(128, 128, 3), (64, 32, 90), (128, 20, 90), (36, 20, 90)])
def test_bounds_and_gradients(dtype, interleaved, D, R, seqs):
    rope = Rotary(D, rotary_dim=R, interleaved=interleaved)
    lens = [(37 * i) % 300 + (3000 if i == 1 else 0) for i in range(seqs)]
    lens[0] = 12000
    n = sum(lens)
    start = torch.tensor([(i * 70001) % 1000000 for i in range(seqs)], dtype=torch.int32)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    pos = torch.cat([torch.arange(a, a + m) for a, m in zip(start.tolist(), lens)])
    x = [rand(n + 3, h, D, dtype=dtype).requires_grad_(True) for h in (5, 2)]
    d = [torch.randn_like(t) for t in x]
    print(f"[rotary] {dtype=} {interleaved=} {D=} {R=} {seqs=}", flush=True)
    y = functional.rotary(rope, *x, cu_seqlens=cu, start=start.cuda())
    g = torch.autograd.grad(y, x, d)
    for a, b, da, db in zip(x, y, d, g):
        close(b[:n].detach(), *reference(a[:n].detach(), pos, rope), dtype)
        close(db[:n], *reference(da[:n], pos, rope, back=True), dtype)
        assert (b[n:] == 0).all() and (db[n:] == 0).all()
        assert torch.equal(functional.rotary(rope, a.detach()[:50], positions=pos[:50].to(torch.int32).cuda()), b[:50].detach())
