"""Decoding over a cache of a fixed number of rows: when it is full, each kv head of each layer lets go of the rows its
attention has given least.

btb has no such cache: its one way with a long conversation is to move pages between the card, pinned RAM and the host
(btb/engine/kvpool.py), which a B200's memory makes unnecessary up to its size and which bounds nothing past it. Here
every pass runs its attention through `btb_b200_attn_scored`, which adds up the softmax weights each cache row is given,
and a pass that would not fit first cuts the cache to `keep` rows (`btb_b200_kv_evict`): the `recent` last ones and those
of the largest totals. The kept rows move together, still rotated to the positions they had; the tokens' positions go on
counting.
"""

from __future__ import annotations

from typing import Any

import torch

from . import capi
from .capi import ptr
from .engine import CardEngine, ModelWeights, pad_rows, rope_tables

PASS_ROWS = 32  # rows a pass at most


class _Steps:
    """the captured step, with room made for its row before each replay"""

    def __init__(self, eng: "EvictEngine", graph: Any, steps: int):
        self.eng, self.graph, self.steps = eng, graph, steps

    def replay(self) -> None:
        self.eng.make_room(self.steps)
        self.graph.replay()
        self.eng.rows += self.steps


class EvictEngine(CardEngine):
    """the card engine over a cache of `budget` rows that evicts down to `keep` of them (`recent` of those the last ones).
    Until the first eviction its tokens are the engine's own, to the attention's rounding. `positions`: the longest
    conversation, in tokens (rows of the rotary tables). A step of the 4 B dense model takes 2.04 ms over 128 rows and 2.18 over
    4000 (the card engine's 1.97 and 2.64), and the step that finds its 4096 rows full 0.12 ms more to halve them."""

    evicts = True  # rows of the cache may leave it: no `Session` stands over it

    def __init__(self, weights: ModelWeights, budget: int = 4096, keep: int | None = None, recent: int | None = None,
                 positions: int | None = None, device: Any = "cuda"):  # fmt: skip
        keep = int(budget) // 2 if keep is None else int(keep)
        recent = keep // 4 if recent is None else int(recent)
        positions = 16 * int(budget) if positions is None else int(positions)
        if not 0 <= recent <= keep or keep <= 0 or keep > int(budget) - PASS_ROWS:
            raise ValueError(f"keep {keep} (recent {recent}) of a budget of {budget}: 0 <= recent <= keep <= budget - {PASS_ROWS}")
        if positions < budget:
            raise ValueError(f"{positions} positions for a budget of {budget} rows")
        c = weights.cfg
        if c.head_dim not in (64, 128) or c.q_heads % c.kv_heads or c.q_heads // c.kv_heads not in (1, 2, 4, 8):
            raise ValueError(f"{c.q_heads} query heads over {c.kv_heads} kv heads of {c.head_dim}: no scored attention for them")
        super().__init__(weights, cap=budget, step_kernel=False, device=device)
        self.keep, self.recent, self.positions = keep, recent, positions
        self.fuse_attn_o = False
        self.cos, self.sin = rope_tables(c, positions, self.dev)
        self.totals = torch.zeros(c.layers, c.kv_heads, self.cap, dtype=torch.float32, device=self.dev)
        # the rows the last eviction kept, by their numbers before it
        self.kept = torch.full((c.layers, c.kv_heads, keep), -1, dtype=torch.int32, device=self.dev)
        L = capi.lib()
        D = c.head_dim
        need = max(int(L.btb_b200_attn_scored_workspace_bytes(T, c.q_heads, c.kv_heads, D, self.cap)) for T in range(1, PASS_ROWS + 1))
        need = max(need, int(L.btb_b200_kv_evict_workspace_bytes(c.layers, c.kv_heads, self.cap)))
        self._ws = torch.empty(need, dtype=torch.uint8, device=self.dev)
        self.rows = 0  # cache rows standing
        self.dropped = 0  # tokens whose rows have been evicted

    # -- room ----------------------------------------------------------------------------------------------------------
    def reset(self) -> None:
        super().reset()
        self.rows = 0
        self._moved(0)

    def _moved(self, dropped: int) -> None:
        """positions run `dropped` ahead of cache rows from here on"""
        self.dropped = dropped
        for M, g in self._bufs.items():
            g["depth"].copy_(torch.arange(M, dtype=torch.int32) + dropped)
        self._before.fill_(dropped - 1)

    def bufs(self, M: int) -> dict[str, torch.Tensor]:
        fresh = M not in self._bufs
        g = super().bufs(M)
        if fresh:
            g["depth"].add_(self.dropped)
        return g

    def make_room(self, T: int) -> None:
        """evicts if the cache does not hold T more rows; T that it would not hold even then are refused, and nothing leaves"""
        if self.dropped + self.rows + T > self.positions:
            raise ValueError(f"position {self.dropped + self.rows + T} of {self.positions}")
        if self.rows + T > self.cap:
            stay = min(self.rows, self.keep)
            if stay + T > self.cap:
                raise ValueError(f"{T} rows beside the {stay} that stay in a cache of {self.cap}")
            self.evict()

    def evict(self) -> None:
        """cuts the cache to `keep` rows a kv head (nothing moves if no more stand)"""
        if self.rows <= self.keep:
            return
        c = self.cfg
        layer = self.K.stride(0)
        capi.call("btb_b200_kv_evict", ptr(self.K), ptr(self.V), ptr(self.totals), ptr(self.n0), ptr(self.K), ptr(self.V),
                  ptr(self.totals), ptr(self.n0), ptr(self.kept), c.layers, layer, layer, c.kv_heads, c.head_dim, self.hs,
                  self.rs, self.cap, self.cap, self.keep, self.recent, 0, 0, ptr(self._ws), capi.stream_ptr())  # fmt: skip
        self._moved(self.dropped + self.rows - self.keep)
        self.rows = self.keep

    # -- passes --------------------------------------------------------------------------------------------------------
    def forward(self, ids: torch.Tensor, depth: Any = None, parents: Any = None, advance: bool = True) -> torch.Tensor:
        if depth is not None or not advance:
            raise TypeError("rows that may be given up again would count in the totals: an evicting cache takes chains it keeps")
        T = int(ids.numel())
        pad_rows(T)  # (more rows than a pass holds are refused before any leave)
        self.make_room(T)
        out = super().forward(ids, torch.arange(self.dropped, self.dropped + T, dtype=torch.int32), torch.arange(-1, T - 1))
        self.rows += T
        return out

    def _attention(self, g: dict, i: int, wq: Any, wk: Any, T: int, s: int, win: int = 0, sinks: Any = None,
                   out: Any = None, warm: tuple = ()) -> None:  # fmt: skip
        if win:
            raise ValueError("a sliding window counts rows: not over a cache that rows have left")
        c = self.cfg
        Hq, Hk, D = c.q_heads, c.kv_heads, c.head_dim
        out = g["att"] if out is None else out
        self._k("btb_b200_norm_rope_kv_pos", ptr(g["qkv"]), ptr(wq), ptr(wk), c.eps, ptr(self.cos), ptr(self.sin),
                ptr(self.n0), ptr(g["depth"]), ptr(self.K[i]), ptr(self.V[i]), ptr(g["q"]), T, Hq, Hk, D, self.hs,
                self.rs, 0, 0, self.cap, self.positions, s)  # fmt: skip
        self._k("btb_b200_attn_scored", ptr(g["q"]), ptr(self.K[i]), ptr(self.V[i]), ptr(out), ptr(self.n0), ptr(g["par"]),
                T, Hq, Hk, D, self.hs, self.rs, float(D**-0.5), ptr(self.totals[i]), self.cap, ptr(self._ws), 0,
                ptr(sinks), self.cap, s)  # fmt: skip

    def step_graph(self, steps: int = 1, publish: bool = True) -> Any:
        key = ("step", steps, publish, self.sampler.sampling.greedy, self.sampler.top_k)
        if key not in self._graphs:
            self.make_room(steps)
            totals = self.totals.clone()  # the capture's eager run puts the length back; what its steps gave the rows goes too
            super().step_graph(steps, publish)
            self.totals.copy_(totals)
        return _Steps(self, self._graphs[key], steps)

    # -- what a cache that rows leave cannot do --------------------------------------------------------------------------
    def prefill_gemm(self, prompt: torch.Tensor, chunk: int = 256) -> torch.Tensor:
        raise TypeError("prefill_gemm's attention adds up no totals: an evicting cache is filled by prefill")

    def generate_speculative(self, prompt: Any, max_new: int, budget: int = 8, v_max: int = 8) -> tuple[list[int], dict]:
        raise TypeError("a verify pass's rejected rows would count in the totals: no speculation over an evicting cache")


__all__ = ["EvictEngine"]
