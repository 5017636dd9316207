"""The evicting engine's host side with the card's work taken out: what it makes room for, and what it refuses before
anything has moved."""

import pytest
import torch

from btb_b200.engine import CardEngine, pad_rows
from btb_b200.evict import EvictEngine
from btb_b200.session import Session


def bare(monkeypatch, rows, budget=160, keep=64, positions=2048):
    """an engine of host numbers only; `cuts` counts its evictions"""
    e = EvictEngine.__new__(EvictEngine)
    e.cap, e.keep, e.recent, e.positions, e.rows, e.dropped, e.cuts = budget, keep, 16, positions, rows, 0, 0

    def evict():
        if e.rows > e.keep:
            e.dropped, e.rows, e.cuts = e.dropped + e.rows - e.keep, e.keep, e.cuts + 1

    e.evict = evict
    monkeypatch.setattr(CardEngine, "forward", lambda self, ids, depth, parents: torch.zeros(pad_rows(int(ids.numel())), 4))
    return e


@pytest.mark.parametrize("rows,T,cut", [(0, 160, 0), (60, 100, 0), (61, 100, -1), (160, 96, 1), (160, 97, -1), (64, 97, -1),
                                        (65, 96, 1), (160, 161, -1), (0, 161, -1), (63, 98, -1)])  # fmt: skip
def test_room_is_made_or_refused_whole(monkeypatch, rows, T, cut):
    e = bare(monkeypatch, rows)
    if cut < 0:  # T rows would not fit beside the rows that stay
        with pytest.raises(ValueError):
            e.make_room(T)
        assert (e.rows, e.dropped, e.cuts) == (rows, 0, 0)
        return
    e.make_room(T)
    assert e.cuts == cut and e.rows + T <= e.cap and e.rows + e.dropped == rows


def test_a_graph_of_more_steps_than_fit_is_refused_at_its_replay_too(monkeypatch):
    from btb_b200.evict import _Steps

    class Graph:
        replays = 0

        def replay(self):
            self.replays += 1

    e, g = bare(monkeypatch, 0), Graph()
    steps = _Steps(e, g, 100)
    steps.replay()
    assert g.replays == 1 and e.rows == 100
    with pytest.raises(ValueError):
        steps.replay()
    assert g.replays == 1 and (e.rows, e.dropped, e.cuts) == (100, 0, 0)


def test_a_pass_of_too_many_rows_lets_none_go(monkeypatch):
    e = bare(monkeypatch, 160)
    with pytest.raises(ValueError):
        e.forward(torch.arange(33))
    assert (e.rows, e.dropped, e.cuts) == (160, 0, 0)
    e.forward(torch.arange(32))
    assert (e.rows, e.dropped, e.cuts) == (96, 96, 1)


def test_a_session_over_it_is_refused_however_it_is_made(monkeypatch):
    """a session moves the cache's length by itself, and goes back to rows that may have left"""
    e = bare(monkeypatch, 0)
    for make in (e.session, lambda: Session(e)):
        with pytest.raises(TypeError):
            make()
