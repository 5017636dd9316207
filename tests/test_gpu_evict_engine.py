"""The evicting engine on the card where a call asks for more than its cache can be cut to."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from btb_b200 import capi  # noqa: E402
from btb_b200 import engine as E  # noqa: E402
from btb_b200.evict import EvictEngine  # noqa: E402

from .util import LAYER_STD  # noqa: E402

CFG = E.DenseConfig("evict", hidden=256, layers=2, q_heads=8, kv_heads=2, head_dim=128, inter=512, vocab=1000)


def prompt(n):
    return torch.randint(0, CFG.vocab, (n,), generator=torch.Generator().manual_seed(n))


def test_more_steps_a_graph_than_the_cache_can_be_cut_for():
    """refused before the capture and at a replay, with the cache as it was; as many as fit evict and go on, replay after replay"""
    mw = E.synth_weights(CFG, seed=3, on_cpu=True, layer_std=LAYER_STD)
    eng = EvictEngine(mw, budget=160, keep=64, recent=16, positions=4096)
    eng.prefill(prompt(100))
    before = eng.K.clone(), eng.totals.clone()
    with pytest.raises(ValueError):
        eng.step_graph(97)
    assert eng.rows == int(eng.n0) == 100 and eng.dropped == 0
    assert torch.equal(eng.K, before[0]) and torch.equal(eng.totals, before[1])
    graph = eng.step_graph(96)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert eng.rows == int(eng.n0) == 160 and eng.rows + eng.dropped == 100 + 96 * (i + 1) and capi.status() == 0
    # a graph that fitted an empty cache once
    eng.reset()
    long = eng.step_graph(150)
    long.replay()
    with pytest.raises(ValueError):
        long.replay()
    torch.cuda.synchronize()
    assert eng.rows == int(eng.n0) == 150 and eng.dropped == 0 and capi.status() == 0
    eng.forward(prompt(20))
    torch.cuda.synchronize()
    assert eng.rows == int(eng.n0) == 84 and capi.status() == 0
