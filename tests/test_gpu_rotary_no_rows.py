"""A step without new tokens goes through all calls of a serving loop; rotary positions of no rows are tensors of no rows, with their gradients."""
import pytest
import torch

from flame_amd import functional
from flame_amd.paged_cache import PagedCache
from flame_amd.rotary import Rotary

pytestmark = pytest.mark.gpu


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_a_step_without_tokens(dtype):
    rope = Rotary(64)
    cache = PagedCache(1, 8, 32, 2, 64, dtype=dtype)
    seqs = [cache.new() for _ in range(3)]
    for counts in ([0, 0, 0], [5, 40, 0], [0, 0, 0]):
        n = sum(counts)
        batch, held = cache.extend(seqs, counts), cache.held(seqs)
        q, k, v = (torch.randn((n, h, 64), device="cuda").to(torch.bfloat16) for h in (4, 2, 2))
        q, k = functional.rotary(rope, q, k, cu_seqlens=batch.cu, start=batch.past)
        cache.store(0, k, v, batch)
        assert cache.attend_rows(0, q, batch, held).shape == (n, 4, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,more", [((0, 4, 64), dict(positions=(0,))), ((2, 4, 0, 64), dict(positions=(2, 0))), ((2, 4, 0, 64), dict(positions=(0,))),
                                        ((0, 4, 5, 64), dict(positions=(5,))), ((0, 4, 64), dict(cu=1)), ((0, 4, 64), dict(cu=3))])
def test_no_rows(dtype, shape, more):
    where = dict(positions=torch.zeros(more["positions"], dtype=torch.int32, device="cuda")) if "positions" in more else dict(cu_seqlens=ints(*[0] * (more["cu"] + 1)))
    rope = Rotary(64)
    q = torch.zeros(shape, dtype=dtype, device="cuda", requires_grad=True)
    k = torch.zeros((shape[0], 1, *shape[2:]), dtype=dtype, device="cuda")
    y = functional.rotary(rope, q, **where)
    assert y.shape == q.shape and y.dtype == dtype and y.requires_grad
    (g,) = torch.autograd.grad(y.sum(), q)
    assert g.shape == q.shape
    yq, yk = functional.rotary(rope, q, k, **where)
    assert yq.requires_grad and not yk.requires_grad and yk.shape == k.shape


def test_still_refused():
    rope = Rotary(64)
    q, k = torch.zeros((0, 4, 64), device="cuda"), torch.zeros((0, 2, 64), device="cuda")
    for bad in (dict(), dict(positions=ints(1)), dict(positions=ints(1)[0]), dict(positions=ints(1)[:0].long()), dict(positions=ints(1)[:0], cu_seqlens=ints(0, 0)),
                dict(cu_seqlens=ints(0)), dict(cu_seqlens=ints(0, 0), start=ints(0, 0)), dict(k=k[:, :0], positions=ints(1)[:0]), dict(k=k.half(), positions=ints(1)[:0]),
                dict(k=torch.zeros((1, 2, 64), device="cuda"), positions=ints(1)[:0])):
        with pytest.raises(AssertionError):
            functional.rotary(rope, q, **bad)
    with pytest.raises(AssertionError):
        functional.rotary(rope, q[:, :0], positions=ints(1)[:0])
