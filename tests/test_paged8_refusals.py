"""What the entry points of the paged cache in 8 bits refuse, through the C ABI and through Python, and that its workspace holds every part that the
device can cut; nothing here reaches a device."""
import ctypes
import os
import random

import pytest
import torch
import torch.autograd.forward_ad as fwad

from flame_amd import capi, functional
from flame_amd.paged_cache import PagedCache

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flame_amd", "lib", "libflame_attn_hip.so")
INVALID, UNSUPPORTED = -1, -2
BF16, I8, E4M3 = 0, 3, 4
P, P2, ODD, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(1 << 20), ctypes.c_void_p(4104), ctypes.c_void_p(0)        # never dereferenced
S, S2 = ctypes.c_void_p(8192), ctypes.c_void_p(1 << 21)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        from flame_amd import build
        build.build_lib()
    lib = ctypes.CDLL(LIB)
    lib.flame_attn_paged_q8_workspace_bytes.restype = ctypes.c_size_t
    return lib


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def attend(lib, q=P, kc=P, dtype=I8, ks=S, vs=S2, block=16, o=P, table=P, stride=8, pages=8, kv_len=P, prefix=NULL, prefix_pages=0, prefix_len=NULL, B=2, H=4,
           H_kv=2, N=1, D=64, n_pages=20, page=16, scale=0.1, qs=(256, 64, 64, 1), cs=(2048, 1024, 64, 1), ss=(2, 1, 1), os_=(256, 64, 64, 1), ws=P, ws_bytes=1 << 30):
    return lib.flame_attn_paged_fwd_q8(q, kc, P2, dtype, ks, vs, block, o, NULL, table, ctypes.c_int64(stride), pages, kv_len, prefix, prefix_pages, prefix_len, B, H,
                                       H_kv, N, D, n_pages, page, ctypes.c_float(scale), i64(*qs), i64(*cs), i64(*cs), i64(*ss), i64(*ss), i64(*os_), ws,
                                       ctypes.c_size_t(ws_bytes), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(q=NULL), INVALID), (dict(kc=NULL), INVALID), (dict(ks=NULL), INVALID), (dict(vs=NULL), INVALID), (dict(table=NULL), INVALID), (dict(kv_len=NULL), INVALID),
    (dict(pages=0), INVALID), (dict(B=0), INVALID), (dict(H=5), INVALID), (dict(block=0), INVALID), (dict(scale=float("nan")), INVALID), (dict(prefix=P), INVALID),
    (dict(pages=100, ws=NULL), INVALID), (dict(pages=100, ws_bytes=100), INVALID), (dict(ws=ODD), UNSUPPORTED), (dict(dtype=BF16), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED),
    (dict(D=72), UNSUPPORTED), (dict(D=144), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(block=32), UNSUPPORTED), (dict(block=3), UNSUPPORTED),
    (dict(page=256, block=256), UNSUPPORTED), (dict(kc=ODD), UNSUPPORTED), (dict(cs=(2048, 1024, 72, 1)), UNSUPPORTED), (dict(cs=(2048, 1024, 64, 2)), UNSUPPORTED),
    (dict(cs=(2048, 1024, 1 << 24, 1)), UNSUPPORTED), (dict(ss=(-2, 1, 1)), UNSUPPORTED), (dict(ss=(1 << 30, 1, 1)), UNSUPPORTED), (dict(ss=(2, 1, 1 << 30)), UNSUPPORTED),
    (dict(ks=ctypes.c_void_p(8194)), UNSUPPORTED), (dict(os_=(0, 64, 64, 1)), UNSUPPORTED), (dict(page=65536, pages=1 << 20), UNSUPPORTED), (dict(N=1 << 30), UNSUPPORTED)])
def test_attention(lib, bad, code):
    assert attend(lib, **bad) == code


def store(lib, k=P, v=P2, kc=P, vc=P2, dtype=I8, ks=S, vs=S2, block=16, table=P, stride=8, pages=8, cu=P, start=P, n=2, T=10, H_kv=2, D=64, n_pages=20, page=16,
          xs=(128, 64, 1), cs=(2048, 1024, 64, 1), ss=(2, 1, 1)):
    return lib.flame_kv_store_q8(k, v, kc, vc, dtype, ks, vs, block, table, ctypes.c_int64(stride), pages, cu, start, n, T, H_kv, D, n_pages, page, i64(*xs), i64(*xs),
                                 i64(*cs), i64(*cs), i64(*ss), i64(*ss), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(k=NULL), INVALID), (dict(vc=NULL), INVALID), (dict(ks=NULL), INVALID), (dict(cu=NULL), INVALID), (dict(start=NULL), INVALID), (dict(T=0), INVALID),
    (dict(n=0), INVALID), (dict(block=0), INVALID), (dict(vc=P), INVALID), (dict(vs=S), INVALID), (dict(dtype=BF16), UNSUPPORTED), (dict(D=24), UNSUPPORTED),
    (dict(D=144), UNSUPPORTED), (dict(block=5), UNSUPPORTED), (dict(block=32), UNSUPPORTED), (dict(page=12), UNSUPPORTED), (dict(xs=(128, 60, 1)), UNSUPPORTED),
    (dict(cs=(2048, 1024, 0, 1)), UNSUPPORTED), (dict(cs=(2048, 1000, 64, 1)), UNSUPPORTED), (dict(ss=(2, 0, 1)), UNSUPPORTED), (dict(ss=(1, 1, 1)), UNSUPPORTED),
    (dict(T=2 ** 31 - 1, block=1, H_kv=8, xs=(512, 64, 1), cs=(8192, 1024, 64, 1), ss=(128, 16, 1)), UNSUPPORTED)])
def test_stores(lib, bad, code):
    assert store(lib, **bad) == code


def load(lib, kc=P, dtype=I8, ks=S, vs=S2, block=16, k=P, v=P2, cu=P, start=P, n=2, T=10, H_kv=2, D=64, page=16, ys=(128, 64, 1), cs=(2048, 1024, 64, 1), ss=(2, 1, 1)):
    return lib.flame_kv_load(kc, P2, dtype, ks, vs, block, k, v, P, ctypes.c_int64(8), 8, cu, start, n, T, H_kv, D, 20, page, i64(*cs), i64(*cs), i64(*ss), i64(*ss),
                             i64(*ys), i64(*ys), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(kc=NULL), INVALID), (dict(ks=NULL), INVALID), (dict(dtype=BF16), INVALID), (dict(k=NULL), INVALID), (dict(v=P), INVALID), (dict(cu=NULL), INVALID),
    (dict(T=0), INVALID), (dict(block=0), INVALID), (dict(dtype=1), INVALID), (dict(dtype=1, ks=NULL, vs=NULL), UNSUPPORTED), (dict(D=24), UNSUPPORTED),
    (dict(D=20, dtype=BF16, ks=NULL, vs=NULL), UNSUPPORTED), (dict(block=6), UNSUPPORTED), (dict(page=10), UNSUPPORTED), (dict(ys=(64, 64, 1)), UNSUPPORTED),
    (dict(ys=(128, 0, 1)), UNSUPPORTED), (dict(cs=(2048, 1024, 72, 1)), UNSUPPORTED), (dict(ss=(-1, 1, 1)), UNSUPPORTED), (dict(T=2 ** 31 - 1), UNSUPPORTED)])
def test_loads(lib, bad, code):
    assert load(lib, **bad) == code


def copies(lib, kc=P, vc=P2, ks=S, vs=S2, layers=2, page=16, D=64, block=16, cs=(40960, 2048, 1024, 64, 1), ss=(40, 2, 1, 1), src=(0,), dst=(1,)):
    a = lambda x: (ctypes.c_int32 * len(x))(*x)
    return lib.flame_kv_copy_pages_q8(kc, vc, ks, vs, layers, 20, 2, page, D, block, i64(*cs), i64(*cs), i64(*ss), i64(*ss), a(src), a(dst), len(src), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(kc=NULL), INVALID), (dict(ks=NULL), INVALID), (dict(vs=S), INVALID), (dict(block=0), INVALID), (dict(src=(20,)), INVALID), (dict(src=(0, 1), dst=(2, 2)), INVALID),
    (dict(src=(1,)), INVALID), (dict(D=72), UNSUPPORTED), (dict(block=64), UNSUPPORTED), (dict(cs=(40960, 2048, 1024, 72, 1)), UNSUPPORTED),
    (dict(ss=(40, 2, 0, 1)), UNSUPPORTED), (dict(cs=(0, 2048, 1024, 64, 1)), UNSUPPORTED)])
def test_copies(lib, bad, code):
    assert copies(lib, **bad) == code


def test_workspace_holds_every_range(lib):
    """Each workgroup has two places for the parts of walks that it shares: as many ranges as there can be workgroups, whatever the lengths are."""
    f = lib.flame_attn_paged_q8_workspace_bytes
    assert f(4, 32, 8, 1, 128, 16, 64, 0) == 0                     # a short table: one workgroup takes all keys
    assert f(4, 32, 8, 1, 72, 16, 100, 0) == f(4, 32, 7, 1, 64, 16, 100, 0) == f(0, 8, 8, 1, 64, 16, 100, 0) == 0
    rng = random.Random(1)
    for _ in range(300):
        B, H_kv, G, N, page = rng.randint(1, 300), rng.choice([1, 2, 8]), rng.choice([1, 4, 8, 40]), rng.choice([1, 4, 9]), 2 ** rng.randint(4, 8)
        D, pages = rng.choice([64, 128]), rng.randint(1, 300)
        have = f(B, H_kv * G, H_kv, N, D, page, pages, 0)
        if not have:
            continue
        rows = N * G
        walks, tiles = B * H_kv * -(-rows // 32), -(-pages * page // 32)
        for most in (walks * tiles, rng.randint(1, walks * tiles)):       # tiles of all walks together
            for groups in (512, 768):
                grid = max(1, min(groups, -(-walks * tiles // 4)))
                share = max(4, -(-most // grid))
                ranges = -(-most // share)
                assert ranges <= grid and have >= 2 * ranges * min(32, rows) * (4 * D + 8) + 8 * (B + 1)


def tensors(dtype=torch.int8, D=64, page=16, block=16, heads=2):
    cache = lambda: torch.zeros((4, heads, page, D)).to(dtype)
    scale = lambda: torch.ones((4, heads, page // block))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    return dict(k=torch.zeros((5, heads, D), dtype=torch.bfloat16), v=torch.zeros((5, heads, D), dtype=torch.bfloat16), kc=cache(), vc=cache(), table=ints([2], [3]),
                cu=ints(0, 2, 5), start=ints(0, 3), ks=scale(), vs=scale())


CALLS = {
    "store": lambda x: capi.kv_store(x["k"], x["v"], x["kc"], x["vc"], x["table"], x["cu"], x["start"], x["ks"], x["vs"]),
    "load": lambda x: capi.kv_load(x["kc"], x["vc"], x["table"], x["cu"], x["start"], 5, x["ks"], x["vs"]),
    "copy": lambda x: capi.kv_copy_pages(x["kc"], x["vc"], [0], [1], x["ks"], x["vs"]),
    "attend": lambda x: functional.sdpa_paged(torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16), x["kc"], x["vc"], x["table"], torch.tensor([3, 4], dtype=torch.int32),
                                              k_scale=x["ks"], v_scale=x["vs"]),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,match", [
    (dict(vs=None), "both caches have scales"), (dict(ks=None, vs=None), "bf16"), (dict(kc=torch.bfloat16), "int8 or both"), (dict(vc=torch.float8_e4m3fn), "int8 or both"),
    (dict(kc=torch.uint8, vc=torch.uint8), "int8 or both"), (dict(ks=torch.float64), "fp32"), (dict(ks=(4, 2)), "fp32"), (dict(ks=(4, 3, 1)), "pages and heads"),
    (dict(vs=(3, 2, 1)), "pages and heads"), (dict(ks=(4, 2, 3), vs=(4, 2, 3)), "into blocks"), (dict(vs=(4, 2, 2)), "into blocks"), (dict(), "GPU")])
def test_python(call, change, match):
    x = tensors()
    for name, to in change.items():
        x[name] = None if to is None else x[name].to(to) if isinstance(to, torch.dtype) else torch.ones(to)
    with pytest.raises(AssertionError, match=match):
        CALLS[call](x)


@pytest.mark.parametrize("call", CALLS)
def test_gradients_and_tangents_of_scales(call):
    for name in ("ks", "vs"):
        x = tensors()
        x[name].requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            CALLS[call](x)
        with torch.no_grad(), pytest.raises(AssertionError, match="GPU"):
            CALLS[call](x)
        x = tensors()
        with fwad.dual_level():
            x[name] = fwad.make_dual(x[name], torch.ones_like(x[name]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                CALLS[call](x)


def test_paged_cache():
    make = lambda **k: PagedCache(2, 8, 16, 2, k.pop("head_dim", 64), device="cpu", **k)
    for bad in (dict(dtype=torch.float16), dict(dtype=torch.int8, block=32), dict(dtype=torch.int8, block=3), dict(dtype=torch.int8, block=0),
                dict(dtype=torch.float8_e4m3fn, head_dim=72)):
        with pytest.raises(ValueError):
            make(**bad)
    cache = make(dtype=torch.int8, block=4)
    assert cache.k.dtype == torch.int8 and cache.k_scale.shape == (2, 8, 2, 4) and make().k_scale is None
    a, b = cache.new(), cache.new()
    batch = cache.extend([a, b], [3, 20])
    assert batch.past.tolist() == [0, 0]
    batch = cache.extend([b, a], [1, 2])
    assert batch.past.tolist() == [20, 3]
    held = cache.held([b, a])
    assert held.counts == [21, 5] and held.start.tolist() == [0, 0] and held.cu.tolist() == [0, 21, 26] and held.prefix_table is None
    with pytest.raises(ValueError):
        cache.held([a, a])
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    for rows, other in ((q[:2], held), (q, cache.held([a]))):
        with pytest.raises(ValueError):
            cache.attend_rows(0, rows, batch, other)
    with pytest.raises(RuntimeError, match="no backward"):
        cache.attend_rows(0, q.clone().requires_grad_(True), batch, held)
    whole = cache.new()
    cache.extend([whole], [32])
    forks = cache.extend([whole, cache.fork(whole)], [1, 2])
    assert forks.past.tolist() == [32, 32] and forks.start.tolist() == [0, 0] and forks.prefix_len.tolist() == [32]
