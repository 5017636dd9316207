"""Evictions over maps and layouts that `test_gpu_long.py` does not walk."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from btb_b200 import capi  # noqa: E402
from btb_b200.capi import call, ptr  # noqa: E402

from .test_gpu_long import BF, DEV, check_evict, evict, gen, some_totals, workspace  # noqa: E402


@pytest.mark.parametrize("into", ["another", "itself"])
def test_a_row_that_its_map_puts_outside_is_not_moved(into):
    """its place is left as it was, every other row moves"""
    g = gen(23)
    L, cap, Hk, D, keep, recent = 1, 100, 2, 64, 50, 10
    K0, V0 = (torch.randn(L, cap, Hk, D, generator=g, device=DEV).to(BF) for _ in range(2))
    t0 = torch.rand(L, Hk, cap, generator=g, device=DEV)
    t0[0, :, 60] = 9.0  # kept by both heads
    for v in (-1, cap, 1 << 30):
        tbl = torch.randperm(cap, generator=g, device=DEV).int()
        good = tbl.clone()
        tbl[60] = v
        K, V, t = K0.clone(), V0.clone(), t0.clone()
        if into == "itself":
            Kd, Vd, td, to = K, V, t, tbl
        else:
            Kd, Vd = (torch.full_like(K0, 3.0) for _ in range(2))
            td, to = torch.zeros_like(t0), None
        old = Kd.clone(), Vd.clone()
        idx, n_out = evict(K, V, t, cap, keep, recent, Kd, Vd, td, tbl=tbl, tbl_d=to)
        torch.cuda.synchronize()
        assert capi.status() == capi.ERR_DOMAIN and int(n_out) == keep
        for h in range(Hk):
            rows = idx[0, h].long()
            at = torch.arange(keep, device=DEV) if to is None else good[:keep].long()
            moved = rows != 60
            assert int((~moved).sum()) == 1
            for src, dst, was in ((K0, Kd, old[0]), (V0, Vd, old[1])):
                assert torch.equal(dst[0, at[moved], h], src[0, good[rows[moved]].long(), h])
                assert torch.equal(dst[0, at[~moved], h], was[0, at[~moved], h])


# ---- evictions over any layout ------------------------------------------------------------------------------------------
def strided(storage, L, cap, Hk, D, ls, hs, rs):
    return storage.as_strided((L, cap, Hk, D), (ls, rs, hs, 1))


def layouts(kind, L, cap, Hk, D):
    """(ls, hs, rs, elements) of a cache of L layers"""
    if kind == "heads":  # each head's rows on their own
        hs, rs = (cap + 3) * D, D
        return Hk * hs + 16, hs, rs, L * (Hk * hs + 16)
    if kind == "wide":  # position-major in wider rows
        hs, rs = D + 8, Hk * (D + 8) + 24
        return cap * rs + 40, hs, rs, L * (cap * rs + 40)
    hs, rs = D, L * Hk * D  # "layers": all layers of a row side by side
    return Hk * D, hs, rs, cap * rs


def evict_strided(K, V, totals, n0, keep, recent, Kd, Vd, td, tbl=None, tbl_d=None):
    L, cap, Hk, D = K.shape
    n0 = torch.tensor([n0], dtype=torch.int32, device=DEV)
    n_out = torch.full((1,), -7, dtype=torch.int32, device=DEV)
    idx = torch.full((L, Hk, keep), -9, dtype=torch.int32, device=DEV)
    ws = workspace("btb_b200_kv_evict_workspace_bytes", L, Hk, cap)
    call("btb_b200_kv_evict", ptr(K), ptr(V), ptr(totals), ptr(n0), ptr(Kd), ptr(Vd), ptr(td), ptr(n_out), ptr(idx), L, K.stride(0),
         Kd.stride(0), Hk, D, K.stride(2), K.stride(1), cap, td.shape[2], keep, recent, ptr(tbl), ptr(tbl_d), ptr(ws),
         capi.stream_ptr())  # fmt: skip
    return idx, n_out


@pytest.mark.parametrize("kind", ["heads", "wide", "layers"])
@pytest.mark.parametrize("L,Hk,D,n0,keep,recent", [(3, 2, 64, 1500, 700, 33), (1, 1, 128, 5000, 2500, 0), (2, 5, 96, 333, 332, 332),
                                                   (2, 3, 8, 90, 120, 7)])  # fmt: skip
def test_evictions_over_any_layout(kind, L, Hk, D, n0, keep, recent):
    g = gen(n0 + D)
    cap = max(n0, keep) + 9
    ls, hs, rs, n = layouts(kind, L, cap, Hk, D)
    stores = [torch.randn(n, generator=g, device=DEV).to(BF) for _ in range(2)]
    first = [x.clone() for x in stores]
    view = lambda x: strided(x, L, cap, Hk, D, ls, hs, rs)  # noqa: E731
    K, V = (view(x) for x in stores)
    K0, V0 = (view(x) for x in first)
    t = some_totals(g, L, Hk, cap, "ties")
    t0 = t.clone()
    # into another cache, laid out alike, of sentinels
    dst = [torch.full((n,), 3.0, dtype=BF, device=DEV) for _ in range(2)]
    Kd, Vd, td = view(dst[0]), view(dst[1]), torch.full((L, Hk, cap), 3.0, device=DEV)
    idx, n_out = evict_strided(K, V, t, n0, keep, recent, Kd, Vd, td)
    three = view(torch.full((n,), 3.0, dtype=BF, device=DEV))
    check_evict(K0, V0, t0, n0, keep, recent, idx, n_out, Kd, Vd, td, (three, three, torch.full_like(td, 3.0)))
    assert all(torch.equal(a, b) for a, b in zip(stores, first))
    # in place
    idx, n_out = evict_strided(K, V, t, n0, keep, recent, K, V, t)
    check_evict(K0, V0, t0, n0, keep, recent, idx, n_out, K, V, t, (K0, V0, t0))
    for d, a, f in ((dst[0], stores[0], first[0]), (dst[1], stores[1], first[1])):  # what lies between rows and heads: as it was
        between = torch.ones(n, dtype=torch.bool, device=DEV)
        view(between)[:] = False
        assert bool((d[between] == 3).all()) and torch.equal(a[between], f[between])
    assert capi.status() == 0
