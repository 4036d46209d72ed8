"""The frequencies of rotary positions, and what the calls refuse; nothing here reaches a device."""
import ctypes
import math
import os
from fractions import Fraction

import pytest
import torch
import torch.autograd.forward_ad as fwad

from flame_amd import capi, functional
from flame_amd.rotary import Rotary

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flame_amd", "lib", "libflame_attn_hip.so")
INVALID, UNSUPPORTED = -1, -2
P, P2, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(1 << 20), ctypes.c_void_p(0)


def test_frequencies():
    base, D = 10000.0, 128
    plain = Rotary(D)
    assert plain.frequencies == [base ** (-2.0 * i / D) for i in range(64)] and plain.size == 1.0
    assert Rotary(D, rotary_dim=32).frequencies == [base ** (-2.0 * i / 32) for i in range(16)]
    assert Rotary(D, scaling="linear", factor=4.0).frequencies == [f / 4.0 for f in plain.frequencies]
    ntk = Rotary(D, scaling="ntk", factor=8.0).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1] * 8.0, plain.frequencies[-1], rel_tol=1e-12) and all(a <= b for a, b in zip(ntk, plain.frequencies))
    for kind in ("yarn", "bands"):
        rope = Rotary(D, scaling=kind, factor=16.0, original_length=4096)
        ratio = [b / a for a, b in zip(rope.frequencies, plain.frequencies)]
        assert ratio[0] == 1.0 and math.isclose(ratio[-1], 16.0, rel_tol=1e-12) and all(a <= b + 1e-12 for a, b in zip(ratio, ratio[1:]))
        turns = [4096 * f / (2 * math.pi) for f in plain.frequencies]
        kept, slowed = (32.0, 1.0) if kind == "yarn" else (4.0, 1.0)
        for t, r in zip(turns, ratio):                     # (yarn: by the pair's number, rounded to whole ones)
            assert r == 1.0 if t >= kept * 1.2 else math.isclose(r, 16.0, rel_tol=1e-12) if t < slowed / 1.2 else 1.0 <= r <= 16.0 + 1e-9
        assert rope.size == (0.1 * math.log(16.0) + 1.0 if kind == "yarn" else 1.0)


def test_fractions_of_a_turn():
    """Against pi to 60 digits, to half a unit of 2^-64; the sign bit is the fraction's first."""
    pi = Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)
    for rope in (Rotary(128), Rotary(64, base=500000.0, scaling="bands", factor=8.0), Rotary(2, base=1.5)):
        for f, t in zip(rope.frequencies, rope.turns_on(torch.device("cpu")).tolist()):
            exact = Fraction(f) / (2 * pi) * 2 ** 64
            assert abs((t % 2 ** 64) - exact) <= Fraction(51, 100)


@pytest.mark.parametrize("bad", [dict(rotary_dim=130), dict(rotary_dim=3), dict(rotary_dim=0), dict(base=1.0), dict(base=math.inf), dict(factor=0.5), dict(factor=math.nan),
                                 dict(scaling="other"), dict(scaling="ntk", rotary_dim=2), dict(original_length=0), dict(fast=1.0), dict(low=4.0)])
def test_refused_frequencies(bad):
    with pytest.raises(ValueError):
        Rotary(128, **bad)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        from flame_amd import build
        build.build_lib()
    return ctypes.CDLL(LIB)


def call(lib, q=P, yq=P2, H=4, qs=(640, 64, 64, 1), qo=(640, 64, 64, 1), k=NULL, yk=NULL, H_kv=0, ks=(1280, 640, 64, 1), dtype=0, turns=P, R=64, size=1.0, pos=P, step=0,
         cu=NULL, start=NULL, n=0, B=2, S=10, D=64):
    st = lambda v: (ctypes.c_int64 * 4)(*v) if v else None
    return lib.flame_rotary(q, yq, H, st(qs), st(qo), k, yk, H_kv, st(ks), st(ks), dtype, turns, R, 0, ctypes.c_float(size), 0, pos, ctypes.c_int64(step), cu, start, n, B, S,
                            D, NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(q=NULL), INVALID), (dict(yq=NULL), INVALID), (dict(H=0), INVALID), (dict(qs=None), INVALID), (dict(turns=NULL), INVALID), (dict(R=0), INVALID),
    (dict(size=math.inf), INVALID), (dict(H_kv=2), INVALID), (dict(H_kv=2, k=P), INVALID), (dict(k=P, yk=P), INVALID), (dict(H_kv=2, k=P, yk=P2), INVALID),
    (dict(pos=NULL), INVALID), (dict(cu=P, n=1), INVALID), (dict(pos=NULL, cu=P, n=1, B=2), INVALID), (dict(pos=NULL, cu=P, n=0, B=1), INVALID), (dict(start=P), INVALID),
    (dict(step=-1), INVALID), (dict(B=0), INVALID), (dict(S=0), INVALID), (dict(R=63), UNSUPPORTED), (dict(R=66), UNSUPPORTED), (dict(dtype=3), UNSUPPORTED),
    (dict(qs=(640, 64, 64, 2)), UNSUPPORTED), (dict(qs=(-640, 64, 64, 1)), UNSUPPORTED), (dict(qo=(640, 0, 64, 1)), UNSUPPORTED), (dict(q=ctypes.c_void_p(4097)), UNSUPPORTED),
    (dict(qo=(0, 640, 64, 1)), UNSUPPORTED), (dict(B=1 << 16, S=1 << 16), UNSUPPORTED), (dict(S=1 << 30, H=64, B=1, qs=(0, 64, 4096, 1), qo=(0, 64, 4096, 1)), UNSUPPORTED)])
def test_refused_by_the_library(lib, bad, code):
    bad = dict(bad)
    if "qo" not in bad and "qs" not in bad:
        bad.setdefault("qo", (640 * 4, 640, 64, 1))
        bad.setdefault("qs", (640 * 4, 640, 64, 1))
    assert call(lib, **bad) == code


def test_refused_by_python():
    rope = Rotary(64)
    q, pos, cu = torch.zeros((5, 4, 64)), torch.arange(5, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="head dim"):
        functional.rotary(rope, torch.zeros((5, 4, 32)), positions=pos)
    with pytest.raises(ValueError, match="expect"):
        functional.rotary(rope, torch.zeros((4, 64)), positions=pos)
    for bad in (dict(), dict(positions=pos, cu_seqlens=cu)):
        with pytest.raises(AssertionError, match="GPU"):           # no tensor is on one: the first check
            functional.rotary(rope, q, **bad)
    with pytest.raises(AssertionError, match="bf16, fp16 or fp32"):
        functional.rotary(rope, q.double(), positions=pos)
    with pytest.raises(AssertionError, match="at least one"):
        functional.rotary(rope, q[:0], positions=pos)
    for which in range(2):
        with fwad.dual_level():
            x = [q.clone(), q.clone()]
            x[which] = fwad.make_dual(x[which], torch.ones_like(q))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                functional.rotary(rope, *x, positions=pos)


@pytest.mark.gpu
def test_refused_on_the_device():
    rope = Rotary(64)
    q, k = torch.zeros((5, 4, 64), device="cuda"), torch.zeros((5, 2, 64), device="cuda")
    pos, cu, start = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 2, 3, 4], [0, 2, 5], [0, 7]))
    for bad in (dict(), dict(positions=pos, cu_seqlens=cu), dict(positions=pos, start=start), dict(positions=pos[:4]), dict(positions=pos.long()), dict(positions=pos.cpu()),
                dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu, start=start[:1]), dict(cu_seqlens=cu[:1]), dict(k=k[:4], positions=pos), dict(k=k.half(), positions=pos),
                dict(k=k.cpu(), positions=pos), dict(k=k[None], positions=pos), dict(positions=pos[None])):
        with pytest.raises(AssertionError):
            functional.rotary(rope, q, **bad)
    four = q[None]
    for bad in (dict(cu_seqlens=cu), dict(positions=torch.zeros((2, 4), dtype=torch.int32, device="cuda"))):
        with pytest.raises(AssertionError):
            functional.rotary(rope, four.transpose(1, 2).expand(3, 4, 5, 64), **bad)
    with pytest.raises(AssertionError):
        capi.rotary(q, None, rope.turns_on(q.device).repeat(2), positions=pos)
    with pytest.raises(capi.FlameAttnError):
        capi.rotary(q, None, rope.turns_on(q.device), size=math.inf, positions=pos)
