"""A model's Rotary serves evaluation and training in any order."""
import pytest
import torch

from flame_amd import functional
from flame_amd.rotary import Rotary
from tests.test_gpu_rotary import close, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("made_in_inference", [False, True])
def test_training_after_inference(made_in_inference):
    with torch.inference_mode(made_in_inference):
        rope = Rotary(64)
    pos = torch.arange(10, dtype=torch.int32, device="cuda")
    x = torch.randn((10, 4, 64), device="cuda")
    with torch.inference_mode():
        y = functional.rotary(rope, x, positions=pos)
    leaf, w = x.clone().requires_grad_(True), torch.randn_like(x)
    z = functional.rotary(rope, leaf, positions=pos)
    assert torch.equal(y, z.detach())
    (g,) = torch.autograd.grad(z, leaf, w)
    close(g, *reference(w, pos, rope, back=True), torch.float32)
