"""What `RowsEngine(shared=True)` refuses before it takes anything on a card, and what it takes."""

from types import SimpleNamespace

import pytest

from btb_b200 import build as B
from btb_b200 import capi
from btb_b200 import engine as E
from btb_b200.batch import RowsEngine


@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 256), (6, 2, 128), (12, 2, 64), (32, 2, 128), (8, 2, 96)])
def test_shapes_that_the_shared_attention_does_not_take_are_refused(Hq, Hk, D):
    B.build()
    cfg = E.DenseConfig("odd", hidden=256, layers=1, q_heads=Hq, kv_heads=Hk, head_dim=D, inter=512, vocab=100)
    with pytest.raises(ValueError, match="shared"):
        RowsEngine(SimpleNamespace(cfg=cfg), shared=True)


@pytest.mark.parametrize("T,Hq,Hk,D", [(32, 64, 8, 128), (32, 32, 8, 128), (1, 64, 8, 64), (9, 8, 8, 128), (32, 8, 1, 64), (4, 256, 32, 64)])
def test_workspaces_are_no_larger_than_their_states(T, Hq, Hk, D):
    """a CTA's parts take a kv head's queries of rows, the next CTA's begin that many further on; then a set of all heads' for the
    stretches that run on into the next head, and the rows' own units: f32 [D] and two words each"""
    B.build()
    L = capi.lib()
    G = Hq // Hk
    units = max(16, min(64, 1024 // (T * Hk)))
    most = (160 * T * G + T * Hq + T * Hq * units) * (D * 4 + 8) + 1024
    assert 0 < int(L.btb_b200_attn_shared_workspace_bytes(T, Hq, Hk, D)) <= most
    kept = T * Hq * 512 * 4 + 16 if T * G <= 32 else 0
    assert 0 < int(L.btb_b200_attn_scored_workspace_bytes(T, Hq, Hk, D, 512)) <= most + T * Hq * 33 * 4 + kept
