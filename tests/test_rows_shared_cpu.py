"""What `RowsEngine(shared=True)` refuses before it takes anything on a card."""

from types import SimpleNamespace

import pytest

from btb_b200 import build as B
from btb_b200 import engine as E
from btb_b200.batch import RowsEngine


@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 256), (6, 2, 128), (12, 2, 64), (32, 2, 128), (8, 2, 96)])
def test_shapes_that_the_shared_attention_does_not_take_are_refused(Hq, Hk, D):
    B.build()
    cfg = E.DenseConfig("odd", hidden=256, layers=1, q_heads=Hq, kv_heads=Hk, head_dim=D, inter=512, vocab=100)
    with pytest.raises(ValueError, match="shared"):
        RowsEngine(SimpleNamespace(cfg=cfg), shared=True)
