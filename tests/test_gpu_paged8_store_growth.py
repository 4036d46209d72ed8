"""A block's scale grows by any factor that bf16 numbers can ask for: from a block of zeros, whose scale is the least, to the largest numbers, and by
every power of two on the way, next to the borders.  Codes and scales are compared with the 64-bit arithmetic of paged8_reference for equality."""
import math

import pytest
import torch

from tests.test_gpu_paged8_store import CODES, Cache
from tests import paged8_reference as ref

pytestmark = pytest.mark.gpu
LARGEST_BF16 = float(torch.finfo(torch.bfloat16).max)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("first", [0.0, 2.0 ** -120, 2.0 ** -60, 1.0])
@pytest.mark.parametrize("then", [1.0, 2.0 ** 34, 2.0 ** 36, 2.0 ** 60, LARGEST_BF16])
def test_from_small_to_large(code, first, then):
    c = Cache(11, code, 2, 2, 2, 16, 64, 16)
    x = c.rows(6, size=0.0)
    x[:, ::2] = first
    c.store(x, [4, 2], [0, 16])
    c.check()
    y = c.rows(2, size=0.0)
    y[:, :, :, ::5], y[:, :, :, 1::5] = then, -then / 3.0
    print(f"[growth] {code=} {first=} {then=}", flush=True)
    c.store(y, [1, 1], [5, 18])
    c.check()


@pytest.mark.parametrize("code", CODES)
def test_every_power_of_two(code):
    """First token one, then a number on, just above and just below what the block holds, 2^k times as large."""
    above, below = 1.0 + 2.0 ** -7, 1.0 - 2.0 ** -8
    steps = [(k, f) for k in range(0, 120, 7) for f in (1.0, above, below)]
    c = Cache(12, code, len(steps), 1, 1, 16, 16, 16)
    x = c.rows(len(steps), size=0.0)
    x[:] = 7.0
    c.store(x, [1] * len(steps), [0] * len(steps))
    holds = ref.LARGEST[code] * float(c.want[0][1][c.table[0][0], 0, 0])
    y = c.rows(len(steps), size=0.0)
    for i, (k, f) in enumerate(steps):
        y[:, i] = float(torch.tensor(holds * f * 2.0 ** k).to(torch.bfloat16))
    assert math.isfinite(float(y.float().max()))
    c.store(y, [1] * len(steps), [3] * len(steps))
    c.check()
