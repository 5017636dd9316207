"""Evictions over maps that `test_gpu_long.py` does not walk."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from btb_b200 import capi  # noqa: E402

from .test_gpu_long import BF, DEV, evict, gen  # noqa: E402


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
