"""The long-cache operators' less travelled paths on the card: passes whose scores are made again (more queries a kv head than
keep theirs), calls that mix prefixes of many and of few rows, caches longer than one turn of the totals' blocks."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from btb_b200 import capi  # noqa: E402
from btb_b200.capi import call, ptr  # noqa: E402

from .test_gpu_long import (  # noqa: E402
    BF, DEV, cache, chain, check_scored, check_shared, gen, scored, shared, tree, workspace,
)  # fmt: skip


def keeps_scores(T, Hq, Hk, D):
    """whether a pass keeps its scores for the totals: its workspace then grows with the cache"""
    n = [int(capi.lib().btb_b200_attn_scored_workspace_bytes(T, Hq, Hk, D, cap)) for cap in (1024, 4096)]
    assert 0 < n[0] <= n[1]
    return n[1] > n[0]


# ---- totals from scores made again --------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5, 1e-20])
@pytest.mark.parametrize("T,Hq,Hk,D", [(9, 8, 2, 128), (32, 8, 2, 64), (32, 16, 2, 128)])
def test_any_scale_where_scores_are_made_again(scale, T, Hq, Hk, D):
    assert not keeps_scores(T, Hq, Hk, D)
    g = gen(T + D)
    n0, cap = 600, 700
    K, V, hs, rs = cache(g, cap, Hk, D)
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    out, totals = torch.zeros(T, Hq * D, dtype=BF, device=DEV), torch.rand(Hk, cap, generator=g, device=DEV)
    before = totals.clone()
    ws = workspace("btb_b200_attn_scored_workspace_bytes", T, Hq, Hk, D, cap)
    n0p, par = torch.tensor([n0], dtype=torch.int32, device=DEV), torch.tensor(chain(T), dtype=torch.int32, device=DEV)
    call("btb_b200_attn_scored", ptr(q), ptr(K), ptr(V), ptr(out), ptr(n0p), ptr(par), T, Hq, Hk, D, hs, rs, scale, ptr(totals), cap,
         ptr(ws), 0, 0, cap, capi.stream_ptr())  # fmt: skip
    check_scored(q.double() * scale * D**0.5, K, V, n0, chain(T), before, out, totals)
    assert capi.status() == 0


@pytest.mark.parametrize("pdl", [0, 8, 15])
@pytest.mark.parametrize("D", [64, 128])
def test_overlapping_launches_where_scores_are_made_again(pdl, D):
    """the third launch reads its inputs ahead of its wait: the same bits with programmatic launches off and on, calls of both
    kinds back to back, each with inputs that a kernel just before it wrote"""
    T, Hq, Hk = 16, 8, 2
    assert not keeps_scores(T, Hq, Hk, D)
    g = gen(D)
    n0, cap = 800, 900
    K, V, hs, rs = cache(g, cap, Hk, D)
    qs = [torch.randn(T, Hq, D, generator=g, device=DEV).to(BF) for _ in range(2)]
    n0s = [n0, n0 - 311]
    ws = workspace("btb_b200_attn_scored_workspace_bytes", T, Hq, Hk, D, cap)
    wants = []
    for q, n in zip(qs, n0s):
        t = torch.zeros(Hk, cap, device=DEV)
        wants.append((scored(q, K, V, hs, rs, n, tree(T), t, cap, ws=ws), t))
    torch.cuda.synchronize()
    q, n0p, par = torch.zeros_like(qs[0]), torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor(tree(T), dtype=torch.int32, device=DEV)
    try:
        capi.set_tuning(pdl=pdl)
        got = []
        for i in range(30):
            t = torch.zeros(Hk, cap, device=DEV)
            q.copy_(qs[i & 1]), n0p.fill_(n0s[i & 1])
            got.append((scored(q, K, V, hs, rs, n0p, par, t, cap, ws=ws), t))
        torch.cuda.synchronize()
    finally:
        capi.set_tuning(pdl=13)
    for i, (o, t) in enumerate(got):
        assert torch.equal(o, wants[i & 1][0]) and torch.equal(t, wants[i & 1][1]), i
    assert capi.status() == 0


def test_many_rows_that_do_not_fit_write_nothing():
    g = gen(10)
    T, cap = 16, 300
    assert not keeps_scores(T, 8, 2, 128)
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(T, 8, 128, generator=g, device=DEV).to(BF)
    for n0 in (285, 300, 1 << 30, -1, -(1 << 31)):
        totals = torch.full((2, cap), 2.0, device=DEV)
        out = scored(q, K, V, hs, rs, n0, chain(T), totals, cap)
        torch.cuda.synchronize()
        assert capi.status() == capi.ERR_DOMAIN, n0
        assert bool(out.isnan().all()) and bool((totals == 2).all()), n0
    totals = torch.zeros(2, cap, device=DEV)
    got = scored(q, K, V, hs, rs, 284, chain(T), totals, cap)  # (the last count that fits)
    check_scored(q, K, V, 284, chain(T), torch.zeros_like(totals), got, totals)
    assert capi.status() == 0


def test_many_rows_over_a_bad_map():
    g = gen(9)
    n0, T, cap = 700, 12, 800
    assert not keeps_scores(T, 8, 2, 64)
    K, V, hs, rs = cache(g, cap, 2, 64)
    tbl = torch.randperm(cap, generator=g, device=DEV).int()
    q = torch.randn(T, 8, 64, generator=g, device=DEV).to(BF)
    totals = torch.zeros(2, cap, device=DEV)
    got = scored(q, K, V, hs, rs, n0, chain(T), totals, cap, tbl)
    check_scored(q, K, V, n0, chain(T), torch.zeros_like(totals), got, totals, tbl)
    assert capi.status() == 0
    for at, v in ((0, -1), (650, cap), (n0 + 1, 1 << 30), (699, -(1 << 31)), (n0 + T - 1, cap)):
        bad = tbl.clone()
        bad[at] = v
        scored(q, K, V, hs, rs, n0, chain(T), torch.zeros(2, cap, device=DEV), cap, bad)
        torch.cuda.synchronize()
        assert capi.status() == capi.ERR_DOMAIN, at


@pytest.mark.parametrize("T,Hq,Hk,D,n0", [(32, 64, 8, 64, 20011), (32, 16, 2, 128, 30001), (32, 64, 8, 128, 9000), (9, 64, 8, 64, 25000)])
def test_many_rows_over_a_long_cache(T, Hq, Hk, D, n0):
    """tiles of keys for several turns of every block that makes scores again"""
    assert not keeps_scores(T, Hq, Hk, D)
    g = gen(n0)
    cap = n0 + T
    K, V, hs, rs = cache(g, cap, Hk, D)
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    totals = torch.rand(Hk, cap, generator=g, device=DEV)
    before = totals.clone()
    got = scored(q, K, V, hs, rs, n0, chain(T), totals, cap)
    check_scored(q, K, V, n0, chain(T), before, got, totals)
    again = before.clone()
    assert torch.equal(scored(q, K, V, hs, rs, n0, chain(T), again, cap), got) and torch.equal(again, totals)
    assert capi.status() == 0


@pytest.mark.parametrize("T,Hk,n0", [(1, 64, 11000), (17, 64, 11000), (1, 128, 9300), (3, 100, 20000)])
def test_kept_scores_of_more_keys_than_the_blocks_take_at_once(T, Hk, n0):
    assert keeps_scores(T, Hk, Hk, 64)
    g = gen(n0 + T)
    cap = n0 + T + 300
    K, V, hs, rs = cache(g, cap, Hk, 64)
    q = torch.randn(T, Hk, 64, generator=g, device=DEV).to(BF)
    totals = torch.rand(Hk, cap, generator=g, device=DEV)
    before = totals.clone()
    got = scored(q, K, V, hs, rs, n0, chain(T), totals, cap)
    check_scored(q, K, V, n0, chain(T), before, got, totals)
    assert capi.status() == 0


# ---- prefixes of many and of few rows in one call -------------------------------------------------------------------------
@pytest.mark.parametrize("of", [[0] * 20 + [1] * 11 + [2], [2] + [1] * 11 + [0] * 20, [1] * 4 + [0] * 17 + [2] * 4 + [3] * 7,
                                [0, 1] * 6 + [2] * 20], ids=str)  # fmt: skip
@pytest.mark.parametrize("lens", [[20000, 9001, 5000, 777], [1, 8000, 64, 9999]], ids=str)
@pytest.mark.parametrize("D,Hk", [(64, 8), (128, 8), (128, 2)])
def test_prefixes_of_uneven_rows(of, lens, D, Hk):
    """eight query heads a kv head: a prefix of more than 16 rows takes both warpgroups' halves of its queries, one of fewer a
    tile each in turn. With the first lengths over 8 kv heads some CTAs hold parts of both kinds, in either order"""
    g = gen(D + len(lens))
    offs = [sum(lens[:p]) for p in range(len(lens))]
    step = 70
    base, cap = sum(lens), sum(lens) + (step + 1) * 32
    lay = [base, step, 32]
    for t, p in enumerate(of):
        lay += [t, offs[p], lens[p]]
    K, V, hs, rs = cache(g, cap, Hk, D)
    q = torch.randn(32, 8 * Hk, D, generator=g, device=DEV).to(BF)
    got = shared(q, K, V, hs, rs, lay, cap)
    check_shared(q, K, V, lay, got, 32)
    assert torch.equal(shared(q, K, V, hs, rs, lay, cap), got) and capi.status() == 0


# ---- the workspace --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,Hq,Hk,D,n", [(32, 64, 8, 128, 20000), (32, 8, 8, 64, 9000), (1, 8, 1, 128, 30000), (3, 256, 32, 64, 4000),
                                         (17, 16, 2, 128, 700), (4, 200, 200, 64, 300)])  # fmt: skip
@pytest.mark.parametrize("prefixes", [1, 5])
def test_nothing_is_written_behind_a_workspace(T, Hq, Hk, D, n, prefixes):
    g = gen(n + T)
    lens = [max(1, n - 64 * p) // min(prefixes, T) for p in range(min(prefixes, T))]
    offs = [sum(lens[:p]) for p in range(len(lens))]
    base, step = sum(lens), 40
    cap = base + (step + 1) * T
    lay = [base, step, T]
    for t in range(T):
        lay += [t, offs[t % len(lens)], lens[t % len(lens)]]
    K, V, hs, rs = cache(g, cap, Hk, D)
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    guard = 1 << 18  # words of a pattern behind it
    for name, dims in (("shared", (T, Hq, Hk, D)), ("scored", (T, Hq, Hk, D, cap))):
        size = int(getattr(capi.lib(), f"btb_b200_attn_{name}_workspace_bytes")(*dims))
        ws = torch.full(((size + 3) // 4 + guard,), 0x5A5A5A5A, dtype=torch.int32, device=DEV)
        if name == "shared":
            check_shared(q, K, V, lay, shared(q, K, V, hs, rs, lay, cap, ws=ws), T)
        else:
            totals = torch.zeros(Hk, cap, device=DEV)
            got = scored(q, K, V, hs, rs, base, chain(T), totals, cap, ws=ws)
            check_scored(q, K, V, base, chain(T), torch.zeros_like(totals), got, totals)
        assert bool((ws[-guard:] == 0x5A5A5A5A).all()), name
    assert capi.status() == 0


def test_two_streams_of_passes_and_tensor_core_matvecs():
    """on each of two streams a pass of totals (three launches), a shared pass and a tensor-core matvec of its output, all of which
    take tensor memory and start under programmatic launch, over and over beside one another: the bits of a run alone"""
    runs = []
    for D, Hq, Hk, T, n in ((64, 32, 4, 16, 900), (128, 16, 2, 32, 1500)):
        g = gen(D)
        lay, cap = [n, 9, T], n + 10 * T
        for t in range(T):
            lay += [t, 0, n]
        K, V, hs, rs = cache(g, cap, Hk, D)
        q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
        R, C = 2048, Hq * D
        W = (torch.randn(R, C, generator=g, device=DEV) / C**0.5).to(BF)
        rw = torch.tensor(lay, dtype=torch.int32, device=DEV)
        n0, par = torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor(tree(T), dtype=torch.int32, device=DEV)
        wss = [workspace("btb_b200_attn_shared_workspace_bytes", T, Hq, Hk, D), workspace("btb_b200_attn_scored_workspace_bytes", T, Hq, Hk, D, cap)]
        wtc = torch.zeros(max(4, int(capi.lib().btb_b200_gemv_tc_workspace_bytes(R, C)) // 4), dtype=torch.float32, device=DEV)
        assert not keeps_scores(T, Hq, Hk, D)

        def go(q=q, K=K, V=V, hs=hs, rs=rs, rw=rw, n0=n0, par=par, cap=cap, wss=wss, wtc=wtc, W=W, R=R, C=C, T=T, Hk=Hk):
            outs = [torch.empty(T, C, dtype=BF, device=DEV) for _ in range(2)]
            y, totals = torch.empty(2, T, R, dtype=BF, device=DEV), torch.zeros(Hk, cap, device=DEV)
            for i in range(2):
                if i == 0:
                    scored(q, K, V, hs, rs, n0, par, totals, cap, out=outs[0], ws=wss[1])
                else:
                    shared(q, K, V, hs, rs, rw, cap, out=outs[1], ws=wss[0])
                call("btb_b200_gemv_tc_bf16", ptr(W), ptr(outs[i]), ptr(y[i]), T, R, C, ptr(wtc), capi.stream_ptr())
            return outs[0], outs[1], y, totals

        want = go()
        torch.cuda.synchronize()
        runs.append((go, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(25):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(runs[i][0]())
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, runs[i][1]))
    assert capi.status() == 0
