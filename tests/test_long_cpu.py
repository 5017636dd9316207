"""What the long-cache operators refuse before anything touches a device, and their plain definitions' own corners."""

import ctypes as C

import pytest

from btb_b200 import build as B
from btb_b200 import capi

from .longref import kept_rows, path_keys, rows_keys


@pytest.fixture(scope="module")
def lib():
    B.build()
    return capi.lib()


@pytest.fixture(scope="module")
def p():
    buf = C.create_string_buffer(64)
    return (C.addressof(buf) + 15) & ~15, buf


GOOD = dict(T=4, Hq=8, Hk=2, D=128, hs=128, rs=256, scale=0.1, cap=512, win=0, ts=512)
BAD = [dict(T=0), dict(T=33), dict(T=-1), dict(Hq=6), dict(Hq=0), dict(Hk=0), dict(Hk=3), dict(Hq=32), dict(D=96), dict(D=256),
       dict(hs=120), dict(hs=132), dict(rs=260), dict(rs=248), dict(cap=0), dict(cap=-1), dict(scale=float("nan")), dict(hs=0),
       dict(rs=0), dict(hs=-128), dict(hs=256 * 511, rs=256), dict(hs=256 * 512 + 8, rs=256)]  # fmt: skip


def shared(lib, a, ptrs):
    q, K, V, out, rw, ws, sinks = ptrs
    return lib.btb_b200_attn_shared(q, K, V, out, rw, a["T"], a["Hq"], a["Hk"], a["D"], a["hs"], a["rs"], a["scale"], ws,
                                    a["win"], sinks, a["cap"], None)  # fmt: skip


def scored(lib, a, ptrs):
    q, K, V, out, n0, par, tot, ws = ptrs
    return lib.btb_b200_attn_scored(q, K, V, out, n0, par, a["T"], a["Hq"], a["Hk"], a["D"], a["hs"], a["rs"], a["scale"], tot,
                                    a["ts"], ws, None, None, a["cap"], None)  # fmt: skip


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_attention_shapes_are_refused(lib, p, bad):
    a = {**GOOD, **bad}
    assert shared(lib, a, [p[0]] * 7) == capi.ERR_DOMAIN
    assert scored(lib, a, [p[0]] * 8) == capi.ERR_DOMAIN
    if set(bad) <= {"T", "Hq", "Hk", "D"}:
        dims = [a[k] for k in ("T", "Hq", "Hk", "D")]
        assert lib.btb_b200_attn_shared_workspace_bytes(*dims) == 0
        assert lib.btb_b200_attn_scored_workspace_bytes(*dims, 512) == 0


def test_attention_pointers_and_totals_are_refused(lib, p):
    for i in range(6):
        ptrs = [p[0]] * 7
        ptrs[i] = None
        assert shared(lib, GOOD, ptrs) == capi.ERR_NULL
        if i != 4:  # (the layout is read a word at a time)
            ptrs[i] = p[0] + 2
            assert shared(lib, GOOD, ptrs) == capi.ERR_DOMAIN
    for i in range(8):
        ptrs = [p[0]] * 8
        ptrs[i] = None
        assert scored(lib, GOOD, ptrs) == capi.ERR_NULL
    assert scored(lib, {**GOOD, "ts": 511}, [p[0]] * 8) == capi.ERR_DOMAIN
    dims = [GOOD[k] for k in ("T", "Hq", "Hk", "D")]
    assert lib.btb_b200_attn_shared_workspace_bytes(*dims) > 0
    assert lib.btb_b200_attn_scored_workspace_bytes(*dims, 0) == 0 < lib.btb_b200_attn_scored_workspace_bytes(*dims, 512)


EV = dict(layers=2, ls=4096, ld=4096, Hk=2, D=64, hs=64, rs=128, cap=32, cap_d=32, keep=16, recent=4)


def evict(lib, a, ptrs, tbl=None, tbl_d=None):
    K, V, tot, n0, Kd, Vd, td, n_out, idx, ws = ptrs
    return lib.btb_b200_kv_evict(K, V, tot, n0, Kd, Vd, td, n_out, idx, a["layers"], a["ls"], a["ld"], a["Hk"], a["D"], a["hs"],
                                 a["rs"], a["cap"], a["cap_d"], a["keep"], a["recent"], tbl, tbl_d, ws, None)  # fmt: skip


@pytest.mark.parametrize("bad", [dict(layers=0), dict(Hk=0), dict(D=0), dict(D=12), dict(cap=0), dict(cap_d=0), dict(keep=0),
                                 dict(keep=33), dict(recent=-1), dict(recent=17), dict(hs=60), dict(hs=68), dict(rs=60), dict(rs=130),
                                 dict(ls=4100), dict(ld=4100), dict(ld=8192), dict(cap_d=31)], ids=str)  # fmt: skip
def test_evict_shapes_are_refused(lib, p, bad):
    assert evict(lib, {**EV, **bad}, [p[0]] * 10) == capi.ERR_DOMAIN


def test_evict_pointers_and_half_in_place_calls_are_refused(lib, p):
    for i in range(10):
        ptrs = [p[0]] * 10
        ptrs[i] = None
        assert evict(lib, EV, ptrs) == capi.ERR_NULL
    for i in (0, 1, 2, 4, 5, 6):  # one of the three caches in place, the others not
        ptrs = [p[0]] * 10
        ptrs[i] = p[0] + 16
        assert evict(lib, EV, ptrs) == capi.ERR_DOMAIN
    assert evict(lib, EV, [p[0]] * 10, tbl=p[0]) == capi.ERR_DOMAIN  # in place through two maps
    assert evict(lib, EV, [p[0]] * 10, tbl_d=p[0]) == capi.ERR_DOMAIN
    for dims in ((0, 2, 32), (2, 0, 32), (2, 2, 0)):
        assert lib.btb_b200_kv_evict_workspace_bytes(*dims) == 0
    assert lib.btb_b200_kv_evict_workspace_bytes(2, 2, 32) > 0


def test_the_definitions_themselves():
    lay = [10, 2, 4, 0, 0, 5, 1, 5, 3]  # two rows: prefixes [0, 5) and [5, 8), the third step
    assert rows_keys(lay, 0) == [0, 1, 2, 3, 4, 10, 14, 18] and rows_keys(lay, 1) == [5, 6, 7, 11, 15, 19]
    assert rows_keys(lay, 0, 2) == [14, 18] and rows_keys(lay, 1, 4) == [7, 11, 15, 19]
    assert path_keys([-1, 0, 0, 2], 3, 2) == [0, 1, 2, 4, 5] and path_keys([-1], 0, 0) == [0]
    nan = float("nan")
    assert kept_rows([1, 3, 2, 3, 0], 3, 1) == [1, 3, 4] and kept_rows([1, 1, 1, 1], 2, 0) == [0, 1]
    assert kept_rows([5, nan, 7, float("inf"), 0], 2, 0) == [1, 3] and kept_rows([-0.0, 0.0, 0.0], 2, 0) == [0, 1]
    assert kept_rows([1, 2], 5, 1) == [0, 1]
