"""Rotary positions: how fast the pairs of a head turn, also where a model runs on contexts longer than it was trained on.

    rope = Rotary(head_dim=128, base=500000.0, scaling="yarn", factor=8.0, original_length=8192)
    q, k = functional.rotary(rope, q, k, cu_seqlens=cu)             # packed rows, each sequence from position 0
    q, k = functional.rotary(rope, q, k, positions=positions)       # a position for every row or token

Pair i of R / 2 turns by f_i = base^(-2 i / R) radians per position; `scaling` slows that down by `factor`:
  "linear"  f_i / factor: positions are pressed together
  "ntk"     base * factor^(R / (R - 2)) in place of base: the first pair keeps its pace, the last is `factor` times slower
  "yarn"    pairs that turn `fast` times or more within original_length keep their pace, those that turn `slow` times or less are `factor` times
            slower, those between by their index; the result is multiplied by 0.1 ln(factor) + 1
  "bands"   pairs whose wave is original_length / high or shorter keep their pace, from original_length / low on they are `factor` times
            slower, those between by their number of turns
The frequencies are formed in 64 bits and kept as fractions of a turn in 64-bit whole numbers: the kernel's angles are exact for every int32
position.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

# 1 / (2 pi), 50 digits
_TURNS_PER_RADIAN = Fraction(15915494309189533576888376337251436203445964574046, 10 ** 50)


class Rotary:
    """head_dim elements of a head, of which the first rotary_dim (omitted: all; even) turn: pairs (i, i + rotary_dim / 2), interleaved: (2 i, 2 i + 1)."""

    def __init__(self, head_dim, base=10000.0, rotary_dim=None, interleaved=False, scaling=None, factor=1.0, original_length=4096, fast=32.0, slow=1.0,
                 low=1.0, high=4.0):
        R = head_dim if rotary_dim is None else rotary_dim
        if R < 2 or R % 2 or R > head_dim:
            raise ValueError("rotary_dim is even, at least 2 and at most head_dim")
        if not (base > 1.0 and math.isfinite(base)):
            raise ValueError("base is a number above 1")
        if not (factor >= 1.0 and math.isfinite(factor)):
            raise ValueError("factor is at least 1")
        if original_length < 1 or not 0.0 < slow < fast or not 0.0 < low < high:
            raise ValueError("original_length is positive, 0 < slow < fast and 0 < low < high")
        self.head_dim, self.rotary_dim, self.interleaved, self.size = head_dim, R, bool(interleaved), 1.0
        if scaling == "ntk":
            if R < 4:
                raise ValueError("a base is scaled for two pairs or more")
            base = base * factor ** (R / (R - 2))
        f = [base ** (-2.0 * i / R) for i in range(R // 2)]
        if scaling == "linear":
            f = [x / factor for x in f]
        elif scaling == "yarn":
            # index of the pair that turns so often within original_length
            first, last = (R * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base)) for turns in (fast, slow))
            first, last = max(math.floor(first), 0), min(math.ceil(last), R - 1)
            slowed = [min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0) for i in range(R // 2)]
            f = [x / factor * s + x * (1.0 - s) for x, s in zip(f, slowed)]
            self.size = 0.1 * math.log(factor) + 1.0
        elif scaling == "bands":
            kept = [min(max((original_length * x / (2.0 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
            f = [x / factor * (1.0 - s) + x * s for x, s in zip(f, kept)]
        elif scaling not in (None, "ntk"):
            raise ValueError('scaling is None, "linear", "ntk", "yarn" or "bands"')
        self.frequencies = f                                    # radians per position
        turns = [round(Fraction(x) * _TURNS_PER_RADIAN * 2 ** 64) for x in f]
        self._turns = [t - 2 ** 64 if t >= 2 ** 63 else t for t in turns]
        self._on = {}

    def turns_on(self, device) -> torch.Tensor:
        """int64 [rotary_dim / 2] on the device: 2^64 turns per position.  Copied there by the first call, which a captured graph therefore
        has behind it."""
        turns = self._on.get(device)
        if turns is None:
            with torch.inference_mode(False):           # a recorded graph saves them, whatever mode the first call is made in
                turns = self._on[device] = torch.tensor(self._turns, dtype=torch.int64, device=device)
        return turns
