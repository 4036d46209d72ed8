"""The frequencies of a Rotary outlive it while calls on other streams than the first still wait to read them."""
import pytest
import torch

from flame_amd import functional
from flame_amd.rotary import Rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_goes_away_while_another_stream_is_late(graph):
    rope = Rotary(64)
    pos = torch.arange(1, 101, dtype=torch.int32, device="cuda")
    x = torch.randn((100, 4, 64), device="cuda", requires_grad=graph)
    w = torch.randn((100, 4, 64), device="cuda")

    def step():
        y = functional.rotary(rope, x, positions=pos)
        return (y.detach(), *torch.autograd.grad(y, x, w)) if graph else (y,)

    want = step()
    turns = rope.turns_on(x.device)
    address, size, zeros = turns.data_ptr(), turns.shape, torch.zeros_like(turns)
    del turns
    work = torch.empty(1 << 28, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(100):                       # of the order of 20 ms
            work.zero_()
        got = step()
    del rope                                       # the side stream has not come to it
    held = [torch.empty(size, dtype=torch.int64, device="cuda") for _ in range(50)]
    for t in held:
        t.copy_(zeros)                             # on the stream that the frequencies were made on
    if not side.query():                           # still not
        assert all(t.data_ptr() != address for t in held)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
