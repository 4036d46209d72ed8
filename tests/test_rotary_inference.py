"""The frequencies on a device are ordinary tensors, whatever mode they are made or first asked for in."""
import pytest
import torch

from flame_amd.rotary import Rotary


@pytest.mark.parametrize("made,asked", [(False, True), (True, False), (True, True)])
def test_frequencies_can_be_saved_for_a_backward(made, asked):
    with torch.inference_mode(made):
        rope = Rotary(64)
    with torch.inference_mode(asked):
        first = rope.turns_on(torch.device("cpu"))
    again = rope.turns_on(torch.device("cpu"))
    assert first is again and not again.is_inference() and again.dtype == torch.int64
    x = torch.ones(32, requires_grad=True)
    (x * again).sum().backward()               # saves them
    assert torch.equal(x.grad, again.float())
