"""The largest sizes that the packed and paged calls take: tiles, steps and places are counted in 32 bits, and a launch has fewer than
2^32 threads.  Broadcast inputs (stride 0) reach such sizes without memory.  No call here reaches a launch: sizes that are taken come with a null
pointer, which is another refusal."""
import ctypes

import pytest

from tests.test_packed_paged_refusals import INVALID, NULL, P, UNSUPPORTED, copies, i64, lib, packed_fwd, paged, store  # noqa: F401 (lib: a fixture)

MOST = 2 ** 31 - 1024


def packed_bwd(lib, n=2, T_q=10, T_kv=10, H=4, H_kv=2, D=64, null=False):
    q, k = i64(H * D, D, 1), i64(H_kv * D, D, 1)
    return lib.flame_attn_packed_bwd_bf16(P, P, P, P, P, NULL if null else P, P, P, P, P, P, n, T_q, T_kv, H, H_kv, D, ctypes.c_float(0.1), q, k, k, q, q, q, k, k, 1, P,
                                          ctypes.c_size_t(2 ** 62), NULL)


@pytest.mark.parametrize("T", [MOST + 1, 2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 1])
def test_packed_rows(lib, T):  # noqa: F811
    """(T + 127) / 128 and the like must not overflow: a negative number of tiles becomes a negative place."""
    one = dict(H=1, H_kv=1, D=8, qs=(8, 8, 1), os_=(8, 8, 1), ks=(0, 8, 1), vs=(0, 8, 1))
    assert packed_fwd(lib, T_kv=T, **one) == UNSUPPORTED
    assert packed_fwd(lib, T_q=T, **one) == UNSUPPORTED
    assert packed_bwd(lib, T_kv=T, H=1, H_kv=1, D=8) == UNSUPPORTED
    assert packed_bwd(lib, T_q=T, H=1, H_kv=1, D=8) == UNSUPPORTED
    assert lib.flame_attn_packed_fwd_workspace_bytes(1, 100, T, 1, 8) == lib.flame_attn_packed_fwd_workspace_bytes(1, T, 100, 1, 8) == 0
    assert lib.flame_attn_packed_bwd_workspace_bytes(1, 100, T, 1, 1, 8) == lib.flame_attn_packed_bwd_workspace_bytes(1, T, 100, 1, 1, 8) == 0


def test_packed_sizes_below(lib):  # noqa: F811
    assert packed_fwd(lib, q=NULL, T_q=MOST, T_kv=MOST, H=1, H_kv=1, D=8) == INVALID
    assert packed_bwd(lib, null=True, T_q=MOST, T_kv=MOST, H=1, H_kv=1, D=8) == INVALID


def test_packed_grids(lib):  # noqa: F811
    """Workgroups of 256 threads for T / 128 + n + 1 tiles of every head: at most 2^24 - 1."""
    heads = 4096
    T = 128 * ((2 ** 24 - 1) // heads - 3)          # 4095 tiles of every head
    for more, code in ((0, INVALID), (128, UNSUPPORTED)):
        assert packed_fwd(lib, q=NULL, T_q=T + more, H=heads, H_kv=1) == code
        assert packed_bwd(lib, null=True, T_q=T + more, H=heads, H_kv=1) == code
        assert packed_bwd(lib, null=True, T_kv=T + more, H=heads, H_kv=heads) == code
    assert packed_fwd(lib, q=NULL, n=2 ** 23, H=1, H_kv=1) == INVALID and packed_fwd(lib, q=NULL, n=2 ** 24, H=1, H_kv=1) == UNSUPPORTED
    assert packed_fwd(lib, q=NULL, T_kv=T + 128, H=heads, H_kv=heads) == INVALID          # the forward has no tiles of keys


@pytest.mark.parametrize("H_kv,D,rows", [(1, 8, 64), (1, 64, 8), (3, 40, 4), (8, 128, 1), (2, 256, 1)])
def test_stored_rows(lib, H_kv, D, rows):  # noqa: F811
    """`rows` rows in a wavefront, four of these in a workgroup of 256 threads."""
    size = dict(H_kv=H_kv, D=D, k=NULL)
    most = min(MOST, (2 ** 24 - 1) * 4 * rows)
    assert store(lib, T=most, **size) == INVALID
    for T in (most + 1, 2 ** 31 - 1):
        assert store(lib, T=T, **size) == UNSUPPORTED


def test_paged_grids(lib):  # noqa: F811
    """One workgroup of 256 threads for every sequence, key head and 32 rows where a table is short; else one for four rows of the result."""
    assert paged(lib, B=2 ** 18, H=64, H_kv=64, D=8, pages=1) == UNSUPPORTED
    one = dict(H=2 ** 10, H_kv=1, D=8, qs=(2 ** 13, 8, 8, 1), os_=(2 ** 13, 8, 8, 1), pages=129, ws=NULL)
    assert paged(lib, B=2 ** 16 - 1, **one) == INVALID and paged(lib, B=2 ** 16, **one) == UNSUPPORTED
    f = lib.flame_attn_paged_workspace_bytes
    assert f(2 ** 16 - 1, 2 ** 10, 1, 1, 8, 16, 129, 0) > 0 and f(2 ** 16, 2 ** 10, 1, 1, 8, 16, 129, 0) == 0


def test_copied_pages(lib):  # noqa: F811
    """Pages of up to 2^30 elements, 65535 layers: their grids are within the limits."""
    assert copies(lib, [0], [1], kc=NULL, layers=65535) == INVALID and copies(lib, [0], [1], kc=NULL, layers=65536) == UNSUPPORTED
