"""What the entry points of packed sequences and of the paged cache refuse, through the C ABI and through Python; nothing
here reaches a device."""
import ctypes
import os

import pytest
import torch

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flame_amd", "lib", "libflame_attn_hip.so")
INVALID, UNSUPPORTED = -1, -2


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        from flame_amd import build
        build.build_lib()
    lib = ctypes.CDLL(LIB)
    for name in ("flame_attn_packed_fwd_workspace_bytes", "flame_attn_packed_bwd_workspace_bytes", "flame_attn_paged_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_size_t
    return lib


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


P = ctypes.c_void_p(4096)            # never dereferenced: the checks come first
P2 = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p(4104)          # not on 16 bytes
NULL = ctypes.c_void_p(0)


def packed_fwd(lib, q=P, k=P, v=P, o=P, lse=P, cu_q=P, cu_k=P, n=2, T_q=10, T_kv=10, H=4, H_kv=2, D=64, scale=0.1, qs=(256, 64, 1), ks=(128, 64, 1),
               vs=(128, 64, 1), os_=(256, 64, 1), ws=NULL, ws_bytes=0):
    return lib.flame_attn_packed_fwd_bf16(q, k, v, o, lse, cu_q, cu_k, n, T_q, T_kv, H, H_kv, D, ctypes.c_float(scale), i64(*qs), i64(*ks), i64(*vs),
                                          i64(*os_), 1, ws, ctypes.c_size_t(ws_bytes), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(q=NULL), INVALID), (dict(o=NULL), INVALID), (dict(cu_q=NULL), INVALID), (dict(cu_k=NULL), INVALID), (dict(n=0), INVALID), (dict(T_q=0), INVALID),
    (dict(T_kv=-1), INVALID), (dict(H=0), INVALID), (dict(H_kv=0), INVALID), (dict(H=5), INVALID), (dict(scale=0.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(D=60), UNSUPPORTED), (dict(D=136), UNSUPPORTED), (dict(q=ODD), UNSUPPORTED), (dict(qs=(256, 64, 2)), UNSUPPORTED),
    (dict(ks=(129, 64, 1)), UNSUPPORTED), (dict(vs=(128, 60, 1)), UNSUPPORTED), (dict(qs=(1 << 24, 64, 1)), UNSUPPORTED), (dict(qs=(-256, 64, 1)), UNSUPPORTED),
    (dict(ws=ODD, ws_bytes=100), UNSUPPORTED), (dict(os_=(0, 64, 1)), UNSUPPORTED), (dict(os_=(256, 0, 1)), UNSUPPORTED), (dict(os_=(128, 64, 1)), UNSUPPORTED), (dict(os_=(64, 576, 1)), UNSUPPORTED)])
def test_packed_forward(lib, bad, code):
    assert packed_fwd(lib, **bad) == code


def packed_bwd(lib, lse=P, ws=P, ws_bytes=1 << 20, dqs=(256, 64, 1), dks=(128, 64, 1), D=64, H_kv=2):
    q, k = i64(256, 64, 1), i64(128, 64, 1)
    return lib.flame_attn_packed_bwd_bf16(P, P, P, P, P, lse, P, P, P, P, P, 2, 10, 10, 4, H_kv, D, ctypes.c_float(0.1), q, k, k, q, q, i64(*dqs), i64(*dks), k,
                                          1, ws, ctypes.c_size_t(ws_bytes), NULL)


@pytest.mark.parametrize("bad,code", [(dict(lse=NULL), INVALID), (dict(ws=NULL), INVALID), (dict(ws_bytes=64), INVALID), (dict(ws=ODD), UNSUPPORTED),
                                      (dict(dqs=(256, 32, 1)), UNSUPPORTED), (dict(dks=(64, 64, 1)), UNSUPPORTED), (dict(D=12), UNSUPPORTED), (dict(H_kv=3), INVALID)])
def test_packed_backward(lib, bad, code):
    assert packed_bwd(lib, **bad) == code


def test_packed_workspace(lib):
    f = lib.flame_attn_packed_bwd_workspace_bytes
    assert f(3, 1000, 1000, 8, 2, 64) >= 2 * 8 * 1000 * 4
    assert f(0, 10, 10, 8, 2, 64) == f(1, 10, 10, 8, 3, 64) == f(1, 10, 10, 8, 2, 63) == 0


def cut(lens_tile, lens_walk, heads, rep, causal, room, least, gain, scale):
    """Units per head as the packed kernels make them: (tiles, longest walk, mean walk) of every sequence, parts of the longest."""
    rows = []
    for t, w in zip(lens_tile, lens_walk):
        tiles, walk = -(-t // 128), -(-w // 64) * rep
        less = 0.5 * min(t, w) / max(t, w, 1) if causal else 0.0
        rows.append((tiles, walk, max((walk + 1) // 2, int(walk * (1 - less) + 1e-3))))
    steps, units = sum(t * m for t, _, m in rows) * heads, sum(t for t, _, _ in rows) * heads
    if max(w for _, w, _ in rows) - steps // 256 <= gain:
        return sum(t for t, _, _ in rows)
    n = steps / max(room - units // 2, room // 4)
    share = int(n) + 1 if n >= 16 else max(least, min(16, int(scale * n)))
    return sum(t * max(1, -(-w // share)) for t, w, _ in rows)


@pytest.mark.parametrize("lens_q,lens_k", [([1], [100000]), ([128] * 3, [5000, 300, 1]), ([4000], [4000]), ([1000, 5], [1000, 1 << 20]), ([7] * 60, [9000] * 60),
                                           ([129, 0, 257], [16000, 4, 0]), ([1] * 64, [1 << 24] * 64)])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (2, 1), (3, 3), (8, 2), (12, 4)])
@pytest.mark.parametrize("causal", [False, True])
def test_workspaces_hold_every_part(lib, lens_q, lens_k, H, Hkv, causal):
    """The grids and the room for partial sums cover the parts that the device cuts, whatever the lengths are."""
    Tq, Tk, n, D = sum(lens_q), sum(lens_k), len(lens_q), 64
    have = lib.flame_attn_packed_fwd_workspace_bytes(n, Tq, Tk, H, D)
    if have:
        assert have >= cut(lens_q, lens_k, H, 1, causal, 512, 16, 16, 1.6) * H * 128 * (4 * D + 8)
    more = lib.flame_attn_packed_bwd_workspace_bytes(n, Tq, Tk, H, Hkv, D) - 2 * -(-H * Tq * 4 // 256) * 256
    assert more >= 0
    slots = Tk // 128 + n + 1
    walked = Tq * (H // Hkv)
    if walked // n >= 768 and slots * Hkv * 2 < 3 * 256 and -(-walked // 64) - (slots - n) * Hkv * (walked // n // 128) // 256 > 12:
        assert more >= cut(lens_k, lens_q, Hkv, H // Hkv, causal, 256, 8, 12, 0.65) * Hkv * 2 * 128 * D * 4
    slots = Tq // 128 + n + 1
    if Tk // n >= 768 and slots * H * 2 < 3 * 256 and -(-Tk // 64) - (slots - n) * H * (Tk // n // 128) // 256 > 12:
        assert more >= cut(lens_q, lens_k, H, 1, causal, 512, 8, 12, 1.6) * H * 128 * D * 4


def paged(lib, q=P, kc=P, o=P, table=P, stride=8, pages=8, kv_len=P, prefix=NULL, prefix_pages=0, prefix_len=NULL, B=2, H=4, H_kv=2, N=1, D=64, n_pages=20,
          page=16, scale=0.1, qs=(256, 64, 64, 1), ks=(2048, 1024, 64, 1), os_=(256, 64, 64, 1), ws=P, ws_bytes=1 << 30):
    return lib.flame_attn_paged_fwd_bf16(q, kc, P, o, NULL, table, ctypes.c_int64(stride), pages, kv_len, prefix, prefix_pages, prefix_len, B, H, H_kv, N, D,
                                         n_pages, page, ctypes.c_float(scale), i64(*qs), i64(*ks), i64(*ks), i64(*os_), ws, ctypes.c_size_t(ws_bytes), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(q=NULL), INVALID), (dict(kc=NULL), INVALID), (dict(table=NULL), INVALID), (dict(kv_len=NULL), INVALID), (dict(pages=0), INVALID), (dict(B=0), INVALID),
    (dict(N=0), INVALID), (dict(H=5), INVALID), (dict(n_pages=0), INVALID), (dict(scale=-1.0), INVALID), (dict(prefix=P), INVALID),
    (dict(prefix=P, prefix_pages=3), INVALID), (dict(prefix_len=P, prefix_pages=3), INVALID), (dict(stride=-1), INVALID), (dict(pages=100, ws=NULL), INVALID),
    (dict(pages=100, ws_bytes=100), INVALID), (dict(ws=ODD), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(page=1 << 17), UNSUPPORTED),
    (dict(D=20), UNSUPPORTED), (dict(D=160), UNSUPPORTED), (dict(kc=ODD), UNSUPPORTED), (dict(ks=(2048, 1024, 64, 2)), UNSUPPORTED),
    (dict(ks=(2048, 1024, 1 << 24, 1)), UNSUPPORTED), (dict(os_=(0, 64, 64, 1)), UNSUPPORTED), (dict(os_=(256, 32, 64, 1)), UNSUPPORTED),
    (dict(page=65536, pages=1 << 20), UNSUPPORTED), (dict(B=1 << 20, pages=1 << 20), UNSUPPORTED), (dict(N=1 << 30), UNSUPPORTED)])
def test_paged_attention(lib, bad, code):
    assert paged(lib, **bad) == code


def test_paged_workspace(lib):
    f = lib.flame_attn_paged_workspace_bytes
    assert f(4, 32, 8, 1, 128, 16, 64, 0) == 0                     # a short table: one workgroup takes all keys
    assert f(4, 32, 8, 1, 128, 16, 65, 0) > 0
    assert f(4, 32, 8, 1, 128, 16, 65, 512) > f(4, 32, 8, 1, 128, 16, 65, 0) and f(4, 32, 8, 1, 128, 16, 64, 1) > 0
    assert f(0, 32, 8, 1, 128, 16, 64, 0) == f(4, 32, 7, 1, 128, 16, 64, 0) == f(4, 32, 8, 1, 128, 17, 64, 0) == 0
    need = f(2, 4, 2, 1, 64, 16, 100, 0)
    assert paged(lib, pages=100, ws_bytes=need - 1) == INVALID


def units(tiles, walks):
    """Most tiles of a unit, as the kernels cut `tiles` tiles (32 keys each) of `walks` walks."""
    if walks < 256:
        return max(4, -(-tiles // (512 - walks)) + 3 & ~3)
    return max(64, -(-tiles // max(2048 - walks, 256)) + 3 & ~3)


def splits(tiles, unit, walks):
    """Units of a walk: as even as they come if there are many walks."""
    if walks >= 256 and tiles > unit:
        n = -(-tiles // unit)
        unit = -(-tiles // n) + 3 & ~3
    return -(-tiles // unit)


@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [4096] * 7, [100000, 3], [7] * 500, [60000] * 64, [0, 0, 5], [9000, 1, 4000] * 30, [2100] * 300])
@pytest.mark.parametrize("H,Hkv,N", [(32, 8, 1), (4, 4, 1), (8, 1, 5)])
@pytest.mark.parametrize("wider", [1, 3])
def test_workspace_holds_every_unit(lib, lens, H, Hkv, N, wider):
    """The units that the device cuts lie within the room that the host asks for, whatever the lengths under a table's width."""
    rows = N * (H // Hkv)
    rt, D, page = -(-rows // 32), 64, 16
    pages = wider * max(129, max(-(-n // page) for n in lens))     # (of at most 128 pages there may be no units)
    tiles, walks = [-(-n // 32) for n in lens], len(lens) * Hkv * rt
    made = sum(splits(t, units(sum(tiles) * Hkv * rt, walks), walks) for t in tiles) * Hkv * rt
    have = lib.flame_attn_paged_workspace_bytes(len(lens), H, Hkv, N, D, page, pages, 0)
    assert have >= made * min(32, rows) * (4 * D + 8)
    all_rows = len(lens) * rows
    for prefix in (1, 100, 5000, 200000):
        t = -(-prefix // 32)
        if all_rows > 64:          # units of 128 rows
            per_split, height = Hkv * -(-all_rows // 128), 128
            n = -(-t * per_split // 256)
            unit = max(n, min(16, 2 * n), 4)
        else:
            per_split, height = Hkv * -(-all_rows // 32), 32
            unit = units(t * per_split, per_split)
        more = lib.flame_attn_paged_workspace_bytes(len(lens), H, Hkv, N, D, page, pages, -(-prefix // page)) - have
        assert more >= -(-t // unit) * per_split * height * (4 * D + 8) - 512


def store(lib, k=P, kc=P, vc=P2, table=P, cu=P, start=P, n=2, T=10, H_kv=2, D=64, n_pages=20, page=16, pages=4, ks=(128, 64, 1), kcs=(2048, 1024, 64, 1)):
    return lib.flame_kv_store_bf16(k, P, kc, vc, table, ctypes.c_int64(4), pages, cu, start, n, T, H_kv, D, n_pages, page, i64(*ks), i64(*ks), i64(*kcs), i64(*kcs), NULL)


@pytest.mark.parametrize("bad,code", [
    (dict(k=NULL), INVALID), (dict(kc=NULL), INVALID), (dict(table=NULL), INVALID), (dict(cu=NULL), INVALID), (dict(start=NULL), INVALID), (dict(n=0), INVALID),
    (dict(T=0), INVALID), (dict(n_pages=0), INVALID), (dict(pages=0), INVALID), (dict(page=12), UNSUPPORTED), (dict(D=4), UNSUPPORTED), (dict(k=ODD), UNSUPPORTED),
    (dict(ks=(128, 64, 2)), UNSUPPORTED), (dict(kcs=(0, 1024, 64, 1)), UNSUPPORTED), (dict(kcs=(2048, 1024, 32, 1)), UNSUPPORTED), (dict(vc=P), INVALID)])
def test_store(lib, bad, code):
    assert store(lib, **bad) == code


def copies(lib, src, dst, kc=P, layers=2, n_pages=20, D=64, ks=(40960, 2048, 1024, 64, 1)):
    a, b = (ctypes.c_int32 * max(1, len(src)))(*src), (ctypes.c_int32 * max(1, len(dst)))(*dst)
    return lib.flame_kv_copy_pages_bf16(kc, P, layers, n_pages, 2, 16, D, i64(*ks), i64(*ks), a, b, len(src), NULL)


def test_copies(lib):
    assert copies(lib, [], []) == 0
    for src, dst in (([0], [20]), ([20], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [5, 5]), ([0, 1], [1, 2]), ([3], [3]), ([1, 0], [2, 1])):
        assert copies(lib, src, dst) == INVALID, (src, dst)
    assert copies(lib, [0], [1], kc=NULL) == INVALID
    assert copies(lib, [0], [1], layers=0) == INVALID
    assert copies(lib, [0], [1], kc=ODD) == UNSUPPORTED
    assert copies(lib, [0], [1], D=65) == UNSUPPORTED
    assert copies(lib, [0], [1], ks=(0, 2048, 1024, 64, 1)) == UNSUPPORTED
    assert copies(lib, [0], [1], ks=(40960, 1024, 1024, 64, 1)) == UNSUPPORTED


def test_python_checks_what_it_can_see():
    """Tensors that are not on a GPU, of other types, shapes and dimensions."""
    from flame_amd import capi, functional
    q, k = torch.zeros((10, 4, 64), dtype=torch.bfloat16), torch.zeros((10, 2, 64), dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], dtype=torch.int32)
    for args, err in (((q, k, k, cu), AssertionError), ((q[0], k, k, cu), ValueError), ((q, k, k[:5], cu), AssertionError), ((q, k[..., :32], k[..., :32], cu), AssertionError),
                      ((q[:, :3], k, k, cu), AssertionError), ((q, k, k, cu.long()), AssertionError), ((q, k, k, cu[:1]), AssertionError), ((q[:0], k, k, cu), AssertionError)):
        with pytest.raises(err):
            functional.sdpa_packed(*args)
    c = torch.zeros((6, 2, 16, 64), dtype=torch.bfloat16)
    table, n = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q = torch.zeros((3, 4, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        functional.sdpa_paged(q[0], c, c, table, n)
    with pytest.raises(AssertionError):
        functional.sdpa_paged(q, c, c, table, n)
    with pytest.raises(AssertionError):
        capi.kv_store(q[:, :2, 0], q[:, :2, 0], c, c, table, torch.arange(4, dtype=torch.int32), n)
    with pytest.raises(AssertionError):
        capi.kv_copy_pages(c, c, [0], [1])
