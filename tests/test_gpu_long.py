"""The long-cache operators on the card against their definitions in 64 bits (tests/longref.py): attention with shared
prefixes, attention that adds up the rows' weights, eviction by those totals, and the engines that run them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from btb_b200 import capi  # noqa: E402
from btb_b200 import engine as E  # noqa: E402
from btb_b200.batch import RowsEngine  # noqa: E402
from btb_b200.capi import call, ptr  # noqa: E402
from btb_b200.evict import EvictEngine  # noqa: E402

from .longref import EPS_F32, attend, kept_rows, path_keys, rows_keys  # noqa: E402
from .util import LAYER_STD, lively  # noqa: E402

DEV = "cuda"
BF = torch.bfloat16
NAN = float("nan")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def cache(g, cap, Hk, D, layout="rows"):
    """K and V [Hk, cap, D] views with the layout's strides: (views, hs, rs)"""
    if layout == "rows":  # position-major, as the engine's arena
        k, v = (torch.randn(cap, Hk, D, generator=g, device=DEV).to(BF) for _ in range(2))
        return k.transpose(0, 1), v.transpose(0, 1), D, Hk * D
    if layout == "wide":  # position-major in wider rows: heads 8 elements apart, rows 24 past the last
        hs, rs = D + 8, Hk * (D + 8) + 24
        k, v = (torch.randn(cap, rs, generator=g, device=DEV).to(BF) for _ in range(2))
        return *(x.as_strided((Hk, cap, D), (hs, rs, 1)) for x in (k, v)), hs, rs
    k, v = (torch.randn(Hk, cap + 3, D, generator=g, device=DEV).to(BF) for _ in range(2))  # each head's rows on their own
    return k[:, :cap], v[:, :cap], (cap + 3) * D, D


def workspace(name, *dims):
    n = int(getattr(capi.lib(), name)(*dims))
    assert n > 0
    return torch.full(((n + 15) // 16 * 4,), NAN, dtype=torch.float32, device=DEV)  # (nothing may rest on its contents)


def shared(q, K, V, hs, rs, lay, cap, sinks=None, win=0, out=None, ws=None):
    T, Hq, D = q.shape
    Hk = K.shape[0]
    out = torch.full((T, Hq * D), NAN, dtype=BF, device=DEV) if out is None else out
    ws = workspace("btb_b200_attn_shared_workspace_bytes", T, Hq, Hk, D) if ws is None else ws
    rw = lay if isinstance(lay, torch.Tensor) else torch.tensor(lay, dtype=torch.int32, device=DEV)
    call("btb_b200_attn_shared", ptr(q), ptr(K), ptr(V), ptr(out), ptr(rw), T, Hq, Hk, D, hs, rs, D**-0.5, ptr(ws), win,
         ptr(sinks), cap, capi.stream_ptr())  # fmt: skip
    return out


def scored(q, K, V, hs, rs, n0, par, totals, cap, tbl=None, sinks=None, out=None, ws=None):
    T, Hq, D = q.shape
    Hk = K.shape[0]
    out = torch.full((T, Hq * D), NAN, dtype=BF, device=DEV) if out is None else out
    ws = workspace("btb_b200_attn_scored_workspace_bytes", T, Hq, Hk, D, cap) if ws is None else ws
    n0 = n0 if isinstance(n0, torch.Tensor) else torch.tensor([n0], dtype=torch.int32, device=DEV)
    par = par if isinstance(par, torch.Tensor) else torch.tensor(par, dtype=torch.int32, device=DEV)
    call("btb_b200_attn_scored", ptr(q), ptr(K), ptr(V), ptr(out), ptr(n0), ptr(par), T, Hq, Hk, D, hs, rs, D**-0.5,
         ptr(totals), totals.stride(0), ptr(ws), ptr(tbl), ptr(sinks), cap, capi.stream_ptr())  # fmt: skip
    return out


def layout(live, T, lens, step, gap=0):
    """prompts of `lens` rows end to end (row t a continuation of prompt t % len(lens)), then the steps; `gap` rows between"""
    offs = [gap + sum(lens[:p]) for p in range(len(lens))]
    base = gap + sum(lens) + gap
    lay = [base, step, T]
    for t in range(live):
        lay += [t, offs[t % len(lens)], lens[t % len(lens)]]
    return lay + [0, 0, -1] * (T - live), base + (step + 1) * T + gap


def check_shared(q, K, V, lay, got, live, sinks=None, win=0):
    T, Hq, D = q.shape
    for t in range(live):
        rows = torch.tensor(rows_keys(lay, t, win), device=DEV)
        ref, _, tol, _ = attend(q[t], K, V, rows, sinks)
        err = (got[t].reshape(Hq, D).double() - ref).abs()
        assert bool((err <= tol).all()), (t, float((err - tol).max()), float(err.max()))


# ---- attention with shared prefixes ------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,Hq,Hk", [(128, 32, 8), (128, 8, 8), (128, 16, 8), (128, 64, 8), (64, 64, 8), (64, 4, 1), (128, 8, 1),
                                     (64, 6, 3)])  # fmt: skip
@pytest.mark.parametrize("live,T,lens,step", [(1, 1, [1], 0), (3, 4, [129], 0), (8, 8, [700], 31), (5, 8, [64, 127, 1], 5),
                                              (32, 32, [300], 130), (17, 32, [128, 256, 511], 128)])  # fmt: skip
def test_shared_rows_equal_the_definition(D, Hq, Hk, live, T, lens, step):
    g = gen(live * 1000 + Hq + D)
    lay, cap = layout(live, T, lens, step)
    K, V, hs, rs = cache(g, cap, Hk, D)
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    got = shared(q, K, V, hs, rs, lay, cap)
    check_shared(q, K, V, lay, got, live)
    assert bool(got[live:].isnan().all())  # padding rows are left as they were
    assert capi.status() == 0


@pytest.mark.parametrize("lens,live,step", [([5000], 32, 300), ([9001, 777], 7, 12), ([33000], 2, 0), ([0], 3, 700), ([0, 4], 2, 0)])
def test_shared_rows_of_long_and_empty_prefixes(lens, live, step):
    g = gen(live)
    T = E.pad_rows(live)
    lay, cap = layout(live, T, lens, step)
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(T, 16, 128, generator=g, device=DEV).to(BF)
    got = shared(q, K, V, hs, rs, lay, cap)
    check_shared(q, K, V, lay, got, live)
    assert capi.status() == 0


@pytest.mark.parametrize("lens,live,Hq,Hk", [([30000], 32, 32, 4), ([20011, 9000], 31, 64, 8), ([40003], 3, 32, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_rows_many_tiles_a_block(lens, live, Hq, Hk, D):
    """long stretches of tiles a block, of 256 and of fewer query rows, several parts each; keys whose scores grow along the
    cache, so that the running maximum moves often"""
    g = gen(live + D)
    T = E.pad_rows(live)
    lay, cap = layout(live, T, lens, 40)
    K, V, hs, rs = cache(g, cap, Hk, D)
    K *= torch.linspace(0.2, 4, cap, device=DEV)[None, :, None].to(BF)
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    got = shared(q, K, V, hs, rs, lay, cap)
    check_shared(q, K, V, lay, got, live)
    assert torch.equal(shared(q, K, V, hs, rs, lay, cap)[:live], got[:live]) and capi.status() == 0


@pytest.mark.parametrize("win", [1, 7, 128, 500, 100000])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_rows_windows_and_sinks(win, D):
    g = gen(win)
    lay, cap = layout(6, 8, [900, 333], 140)
    K, V, hs, rs = cache(g, cap, 2, D)
    q = torch.randn(8, 8, D, generator=g, device=DEV).to(BF)
    sinks = torch.randn(8, generator=g, device=DEV) * 3
    check_shared(q, K, V, lay, shared(q, K, V, hs, rs, lay, cap, sinks, win), 6, sinks, win)
    check_shared(q, K, V, lay, shared(q, K, V, hs, rs, lay, cap, None, win), 6, None, win)
    assert capi.status() == 0


@pytest.mark.parametrize("kind", ["rows", "wide", "heads"])
def test_shared_reads_only_its_rows_and_any_layout(kind):
    """everything a row does not see - the gaps between prompts, padding columns' steps, later steps, other rows' steps -
    may hold anything, NaN and infinities among it, and other rows' results do not show it"""
    g = gen(5)
    lay, cap = layout(5, 8, [200, 131], 150, gap=9)
    K, V, hs, rs = cache(g, cap, 3, 128, kind)
    q = torch.randn(8, 12, 128, generator=g, device=DEV).to(BF)
    want = shared(q, K, V, hs, rs, lay, cap)
    check_shared(q, K, V, lay, want, 5)
    seen = {r for t in range(5) for r in rows_keys(lay, t)}
    rest = torch.tensor([r for r in range(cap) if r not in seen], device=DEV)
    K[:, rest], V[:, rest] = NAN, float("inf")
    assert torch.equal(shared(q, K, V, hs, rs, lay, cap)[:5], want[:5])
    # one row's own steps spoiled: only that row
    mine = torch.tensor([r for r in rows_keys(lay, 2) if r >= lay[0]], device=DEV)
    V[:, mine[3]] = NAN
    got = shared(q, K, V, hs, rs, lay, cap)
    others = [0, 1, 3, 4]
    assert torch.equal(got[others], want[others]) and bool(got[2].isnan().any())
    # one prompt's rows spoiled: only its rows
    V[:, 9 + 200 + 4] = NAN
    got = shared(q, K, V, hs, rs, lay, cap)
    assert torch.equal(got[[0, 4]], want[[0, 4]]) and bool(got[1].isnan().any()) and bool(got[3].isnan().any())


def test_shared_extreme_scores():
    """a first key so far below the next ones that its weight vanishes, and one so far above that it takes everything"""
    g = gen(6)
    lay, cap = layout(4, 4, [1000], 3)
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(4, 8, 128, generator=g, device=DEV).to(BF)
    for at, f in ((0, -60.0), (999, 60.0), (500, 60.0), (130, -60.0), (lay[0] + 5, 30.0)):
        keep = K[:, at].clone()
        K[:, at] = (f * q[0].reshape(2, 4, 128)[:, 0]).to(BF)
        check_shared(q, K, V, lay, shared(q, K, V, hs, rs, lay, cap), 4)
        K[:, at] = keep


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.5, 1e-20])
def test_any_scale(scale):
    g = gen(31)
    lay, cap = layout(5, 8, [700], 70)
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(8, 8, 128, generator=g, device=DEV).to(BF)
    out = torch.zeros(8, 8 * 128, dtype=BF, device=DEV)
    ws = workspace("btb_b200_attn_shared_workspace_bytes", 8, 8, 2, 128)
    rw = torch.tensor(lay, dtype=torch.int32, device=DEV)
    call("btb_b200_attn_shared", ptr(q), ptr(K), ptr(V), ptr(out), ptr(rw), 8, 8, 2, 128, hs, rs, scale, ptr(ws), 0, 0, cap,
         capi.stream_ptr())  # fmt: skip
    # the definition divides by sqrt(D): queries scaled in 64 bits stand for the scale
    check_shared(q.double() * scale * 128**0.5, K, V, lay, out, 5)
    for T in (1, 5):  # a pass that keeps its scores, and one that makes them again
        totals = torch.zeros(2, cap, device=DEV)
        ws = workspace("btb_b200_attn_scored_workspace_bytes", T, 8, 2, 128, cap)
        n0, par = torch.tensor([600], dtype=torch.int32, device=DEV), torch.tensor(chain(T), dtype=torch.int32, device=DEV)
        call("btb_b200_attn_scored", ptr(q), ptr(K), ptr(V), ptr(out), ptr(n0), ptr(par), T, 8, 2, 128, hs, rs, scale, ptr(totals),
             cap, ptr(ws), 0, 0, cap, capi.stream_ptr())  # fmt: skip
        check_scored(q[:T].double() * scale * 128**0.5, K, V, 600, chain(T), torch.zeros_like(totals), out[:T], totals)
    assert capi.status() == 0


@pytest.mark.parametrize("pdl", [0, 15])
def test_the_launches_overlap_changes_nothing(pdl):
    """with programmatic launches off, and on for every kind of kernel, the same bits, many calls back to back"""
    g = gen(32)
    lay, cap = layout(8, 8, [900], 40)
    K, V, hs, rs = cache(g, cap, 2, 64)
    q = torch.randn(8, 8, 64, generator=g, device=DEV).to(BF)
    ws = workspace("btb_b200_attn_shared_workspace_bytes", 8, 8, 2, 64)
    wt = workspace("btb_b200_attn_scored_workspace_bytes", 8, 8, 2, 64, cap)
    want, totals = shared(q, K, V, hs, rs, lay, cap), torch.zeros(2, cap, device=DEV)
    scored(q, K, V, hs, rs, 800, chain(8), totals, cap)
    torch.cuda.synchronize()
    try:
        capi.set_tuning(pdl=pdl)
        outs, sums = [], []
        for _ in range(30):
            t = torch.zeros(2, cap, device=DEV)
            outs.append(shared(q, K, V, hs, rs, lay, cap, ws=ws)), sums.append(t)
            scored(q, K, V, hs, rs, 800, chain(8), t, cap, ws=wt)
        torch.cuda.synchronize()
    finally:
        capi.set_tuning(pdl=13)
    assert all(torch.equal(o, want) for o in outs) and all(torch.equal(t, totals) for t in sums) and capi.status() == 0


def test_shared_is_captured_once_for_every_length_and_two_graphs_have_their_workspaces():
    g = gen(7)
    cap = 3000
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(8, 8, 128, generator=g, device=DEV).to(BF)
    a, b = layout(8, 8, [1500], 40)[0], layout(6, 8, [100, 800], 3)[0]
    wants = [shared(q, K, V, hs, rs, lay, cap) for lay in (a, b)]
    rws = [torch.tensor(a, dtype=torch.int32, device=DEV) for _ in range(2)]
    outs = [torch.zeros(8, 8 * 128, dtype=BF, device=DEV) for _ in range(2)]
    wss = [workspace("btb_b200_attn_shared_workspace_bytes", 8, 8, 2, 128) for _ in range(2)]
    graphs = []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            shared(q, K, V, hs, rs, rws[i], cap, out=outs[i], ws=wss[i])
        graphs.append(gr)
    rws[1].copy_(torch.tensor(b, dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1][:6], wants[1][:6])


def test_shared_layout_outside_the_cache_is_refused_by_the_status_word():
    g = gen(8)
    K, V, hs, rs = cache(g, 512, 2, 128)
    q = torch.randn(4, 8, 128, generator=g, device=DEV).to(BF)
    good = layout(4, 4, [300], 0)[0]
    for bad in ([300, 0, 4] + [0, 300, 300, 1, 0, 300, 2, 0, 300, 3, 0, 300],  # a prefix past the cache
                [600, 0, 4] + good[3:], [300, 60, 4] + good[3:],  # steps past it
                [300, 0, 4] + [0, -5, 300, 1, 0, 300, 2, 0, 300, 3, 0, 300],  # a prefix before it
                [300, 0, 4] + [-301, 0, 300, 1, 0, 300, 2, 0, 300, 3, 0, 300]):  # fmt: skip
        assert capi.status() == 0
        shared(q, K, V, hs, rs, bad, 512)
        torch.cuda.synchronize()
        assert capi.status() == capi.ERR_DOMAIN
    check_shared(q, K, V, good, shared(q, K, V, hs, rs, good, 512), 4)
    assert capi.status() == 0


# ---- attention that adds up what each row is given -----------------------------------------------------------------------
def chain(T):
    return list(range(-1, T - 1))


def tree(T):
    return [-1 if t == 0 else (t - 1) // 3 for t in range(T)]


def check_scored(q, K, V, n0, par, before, got, after, tbl=None, sinks=None):
    T, Hq, D = q.shape
    Hk = K.shape[0]
    want, tol_w = before.double().clone(), torch.zeros_like(before, dtype=torch.float64)
    want[:, n0 : n0 + T] = 0
    for t in range(T):
        j = torch.tensor(path_keys(par, t, n0), device=DEV)
        ref, w, tol, rel = attend(q[t], K, V, j if tbl is None else tbl[j].long(), sinks)
        err = (got[t].reshape(Hq, D).double() - ref).abs()
        assert bool((err <= tol).all()), (t, float((err - tol).max()), float(err.max()))
        given = w.reshape(Hk, Hq // Hk, -1).sum(1)
        want[:, j] += given
        tol_w[:, j] += given * (rel + (len(j) + T * Hq // Hk) * EPS_F32)
    # ... and a weight below f32's smallest normal number, 2^-126, may come out as zero (the powers flush): at most that much a
    # weight, T rows times the kv head's queries of them in a total. Scores that spread over 300 units show it: e^-88 is 2^-127
    tol_w += (T * Hq // Hk + 2) * EPS_F32 * want.abs() + T * Hq // Hk * torch.finfo(torch.float32).tiny
    err = (after.double() - want).abs()
    # (rows past the pass are left as they were: compared to the bit)
    assert bool((err[:, : n0 + T] <= tol_w[:, : n0 + T]).all()), float((err - tol_w)[:, : n0 + T].max())
    assert torch.equal(after[:, n0 + T :], before[:, n0 + T :])


@pytest.mark.parametrize("D,Hq,Hk", [(128, 32, 8), (64, 64, 8), (128, 4, 4), (128, 8, 1), (64, 6, 3), (64, 4, 4)])
@pytest.mark.parametrize("T,n0,par", [(1, 0, chain), (1, 1, chain), (1, 127, chain), (1, 128, chain), (1, 3001, chain),
                                      (2, 129, tree), (9, 613, tree), (32, 0, chain), (32, 257, chain), (31, 1030, tree)])  # fmt: skip
def test_scored_equals_the_definition(D, Hq, Hk, T, n0, par):
    g = gen(T * 10000 + n0 + Hq + D)
    cap = n0 + T + 5
    K, V, hs, rs = cache(g, cap, Hk, D)
    K[:, n0 + T :], V[:, n0 + T :] = NAN, NAN
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    totals = torch.rand(Hk, cap, generator=g, device=DEV)
    before = totals.clone()
    got = scored(q, K, V, hs, rs, n0, par(T), totals, cap)
    check_scored(q, K, V, n0, par(T), before, got, totals)
    again = before.clone()
    assert torch.equal(scored(q, K, V, hs, rs, n0, par(T), again, cap), got) and torch.equal(again, totals)
    assert capi.status() == 0


@pytest.mark.parametrize("kind", ["rows", "wide", "heads"])
@pytest.mark.parametrize("T,n0", [(1, 20000), (5, 4097), (2, 9000), (32, 30011)])
def test_scored_long_paged_sinks_and_layouts(kind, T, n0):
    g = gen(n0 + T)
    Hq, Hk, D, cap = 16, 2, 128, (n0 + T + 70) // 64 * 64
    K, V, hs, rs = cache(g, cap, Hk, D, kind)
    pages = torch.randperm(cap // 64, generator=g, device=DEV).int()
    tbl = (pages[:, None] * 64 + torch.arange(64, device=DEV, dtype=torch.int32)).reshape(-1).contiguous()
    q = torch.randn(T, Hq, D, generator=g, device=DEV).to(BF)
    sinks = torch.randn(Hq, generator=g, device=DEV)
    totals = torch.rand(Hk, cap + 11, generator=g, device=DEV)[:, :cap]  # (heads further apart than the cache is long)
    before = totals.clone()
    got = scored(q, K, V, hs, rs, n0, tree(T), totals, cap, tbl, sinks)
    check_scored(q, K, V, n0, tree(T), before, got, totals, tbl, sinks)
    assert capi.status() == 0


def test_scored_rows_mapped_one_by_one_and_a_bad_map():
    g = gen(9)
    n0, T, cap = 700, 3, 800
    K, V, hs, rs = cache(g, cap, 2, 64)
    tbl = torch.randperm(cap, generator=g, device=DEV).int()  # no pages: every row anywhere
    q = torch.randn(T, 8, 64, generator=g, device=DEV).to(BF)
    totals = torch.zeros(2, cap, device=DEV)
    got = scored(q, K, V, hs, rs, n0, chain(T), totals, cap, tbl)
    check_scored(q, K, V, n0, chain(T), torch.zeros_like(totals), got, totals, tbl)
    assert capi.status() == 0
    for at, v in ((0, -1), (650, cap), (n0 + 1, 1 << 30), (699, -(1 << 31))):
        bad = tbl.clone()
        bad[at] = v
        scored(q, K, V, hs, rs, n0, chain(T), torch.zeros(2, cap, device=DEV), cap, bad)
        torch.cuda.synchronize()
        assert capi.status() == capi.ERR_DOMAIN, at


def test_scored_pass_that_does_not_fit_writes_nothing():
    g = gen(10)
    cap = 300
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(4, 8, 128, generator=g, device=DEV).to(BF)
    for n0 in (297, 300, 1 << 30, -1, -(1 << 31)):
        totals = torch.full((2, cap), 2.0, device=DEV)
        out = scored(q, K, V, hs, rs, n0, chain(4), totals, cap)
        assert bool(out.isnan().all()) and bool((totals == 2).all())
        assert capi.status() == capi.ERR_DOMAIN
    totals = torch.zeros(2, cap, device=DEV)
    got = scored(q, K, V, hs, rs, 296, chain(4), totals, cap)
    check_scored(q, K, V, 296, chain(4), torch.zeros_like(totals), got, totals)
    assert capi.status() == 0


def test_scored_a_spoiled_row_spoils_only_the_rows_that_see_it():
    g = gen(11)
    n0, T, cap = 200, 4, 300
    K, V, hs, rs = cache(g, cap, 2, 128)
    q = torch.randn(T, 8, 128, generator=g, device=DEV).to(BF)
    par = [-1, 0, 0, 2]
    want = scored(q, K, V, hs, rs, n0, par, torch.zeros(2, cap, device=DEV), cap)
    V[:, n0 + 2] = NAN  # a draft: row 3 descends from it, row 1 does not
    got = scored(q, K, V, hs, rs, n0, par, torch.zeros(2, cap, device=DEV), cap)
    assert torch.equal(got[:2], want[:2]) and bool(got[2:].isnan().all())


def test_scored_totals_add_up_over_steps_in_one_captured_graph():
    """a decode captured once and replayed as the cache grows, on a stream of its own"""
    g = gen(12)
    Hq, Hk, D, cap, start, steps = 32, 8, 128, 700, 120, 24
    K, V, hs, rs = cache(g, cap, Hk, D)
    qs = torch.randn(steps, Hq, D, generator=g, device=DEV).to(BF)
    q = torch.zeros(1, Hq, D, dtype=BF, device=DEV)
    n0 = torch.tensor([start], dtype=torch.int32, device=DEV)
    totals = torch.zeros(Hk, cap, device=DEV)
    totals[:, start:] = NAN  # rows not written yet: set when they are
    out = torch.zeros(1, Hq * D, dtype=BF, device=DEV)
    ws = workspace("btb_b200_attn_scored_workspace_bytes", 1, Hq, Hk, D, cap)
    root = torch.tensor([-1], dtype=torch.int32, device=DEV)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        scored(q, K, V, hs, rs, n0, root, totals, cap, out=out, ws=ws)
    want = torch.zeros(Hk, cap, dtype=torch.float64, device=DEV)
    with torch.cuda.stream(st):
        for i in range(steps):
            q.copy_(qs[i : i + 1])
            graph.replay()
            n0.add_(1)
    torch.cuda.synchronize()
    rel = 0.0
    for i in range(steps):
        j = torch.arange(start + i + 1, device=DEV)
        _, w, _, r = attend(qs[i], K, V, j)
        want[:, j] += w.reshape(Hk, Hq // Hk, -1).sum(1)
        rel = max(rel, r)
    n = start + steps
    tol = want[:, :n] * (rel + (n + steps * 6) * EPS_F32)
    assert bool(((totals[:, :n].double() - want[:, :n]).abs() <= tol).all())
    assert bool(totals[:, n:].isnan().all())
    assert abs(float(totals[:, :n].double().sum()) - steps * Hq) < 1e-3


# ---- eviction -----------------------------------------------------------------------------------------------------------
def evict(K, V, totals, n0, keep, recent, Kd=None, Vd=None, td=None, tbl=None, tbl_d=None, n_out=None):
    """K, V [L, cap, Hk, D] position-major, totals [L, Hk, cap]; in place without Kd"""
    L, cap, Hk, D = K.shape
    Kd, Vd, td = (K, V, totals) if Kd is None else (Kd, Vd, td)
    n0 = n0 if isinstance(n0, torch.Tensor) else torch.tensor([n0], dtype=torch.int32, device=DEV)
    n_out = torch.full((1,), -7, dtype=torch.int32, device=DEV) if n_out is None else n_out
    idx = torch.full((L, Hk, keep), -9, dtype=torch.int32, device=DEV)
    ws = workspace("btb_b200_kv_evict_workspace_bytes", L, Hk, cap)
    call("btb_b200_kv_evict", ptr(K), ptr(V), ptr(totals), ptr(n0), ptr(Kd), ptr(Vd), ptr(td), ptr(n_out), ptr(idx), L,
         K.stride(0), Kd.stride(0), Hk, D, D, Hk * D, cap, Kd.shape[1], keep, recent, ptr(tbl), ptr(tbl_d), ptr(ws),
         capi.stream_ptr())  # fmt: skip
    return idx, n_out


def some_totals(g, L, Hk, cap, kind):
    t = torch.rand(L, Hk, cap, generator=g, device=DEV)
    if kind == "ties":
        t = (t * 4).floor()
    elif kind == "equal":
        t = torch.full_like(t, 0.25)
    elif kind == "close":  # totals that differ in their last bits
        t = 1 + (t * 64).floor() * 2**-23
    elif kind == "odd":
        t[..., ::7] = NAN
        t[..., 1::5] = float("inf")
        t[..., 2::11] = -0.0
        t[..., 3::11] = 0.0
        t[..., 4::13] = -float("inf")
        t[..., 5::13] *= -1
        t[..., 6::17] *= 1e-42
        t[..., 8::29] = -NAN
    return t


def check_evict(K0, V0, t0, n0, keep, recent, idx, n_out, Kd, Vd, td, old):
    L, cap, Hk, D = K0.shape
    n = min(n0, keep)
    assert int(n_out) == n
    for a in range(L):
        for h in range(Hk):
            rows = kept_rows(t0[a, h, :n0].tolist(), keep, recent)
            assert idx[a, h].tolist() == rows + [-1] * (keep - n), (a, h)
            r = torch.tensor(rows, dtype=torch.long, device=DEV)
            for src, dst in ((K0[a, :, h], Kd[a, :, h]), (V0[a, :, h], Vd[a, :, h])):
                assert torch.equal(dst[:n].view(torch.int16), src[r].view(torch.int16))
            assert torch.equal(td[a, h, :n].view(torch.int32), t0[a, h, r].view(torch.int32))
    for dst, o, dim in ((Kd, old[0], 1), (Vd, old[1], 1), (td, old[2], 2)):  # rows past the count: as they were
        m = dst.shape[dim] - n
        as_int = torch.int32 if dst.dtype == torch.float32 else torch.int16
        assert torch.equal(dst.narrow(dim, n, m).contiguous().view(as_int), o.narrow(dim, n, m).contiguous().view(as_int))


@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "close", "odd"])
@pytest.mark.parametrize("n0,keep,recent", [(1, 1, 0), (2, 1, 1), (2, 1, 0), (40, 40, 3), (7, 40, 3), (0, 5, 5), (300, 299, 0),
                                            (300, 100, 100), (1025, 513, 64), (2600, 1999, 7), (5000, 33, 1)])  # fmt: skip
def test_evict_keeps_the_rows_of_most_weight(kind, n0, keep, recent):
    g = gen(n0 + keep)
    L, Hk, D, cap = 2, 3, 64, n0 + 9
    K, V = (torch.randn(L, cap, Hk, D, generator=g, device=DEV).to(BF) for _ in range(2))
    t = some_totals(g, L, Hk, cap, kind)
    K0, V0, t0 = K.clone(), V.clone(), t.clone()
    capd = keep + 3
    Kd, Vd = (torch.full((L, capd, Hk, D), 3.0, dtype=BF, device=DEV) for _ in range(2))
    td = torch.full((L, Hk, capd), 3.0, device=DEV)
    old = Kd.clone(), Vd.clone(), td.clone()
    idx, n_out = evict(K, V, t, n0, keep, recent, Kd, Vd, td)
    check_evict(K0, V0, t0, n0, keep, recent, idx, n_out, Kd, Vd, td, old)
    for x, x0 in ((K, K0), (V, V0)):
        assert torch.equal(x, x0)
    if keep <= cap:  # in place, the count into n0's own word
        word = torch.tensor([n0], dtype=torch.int32, device=DEV)
        idx, n_out = evict(K, V, t, word, keep, recent, n_out=word)
        check_evict(K0, V0, t0, n0, keep, recent, idx, n_out, K, V, t, (K0, V0, t0))
    assert capi.status() == 0


@pytest.mark.parametrize("L,n0,keep,recent,Hk,D", [(36, 1000, 500, 100, 8, 128), (1, 40001, 20001, 64, 2, 128),
                                                   (3, 2049, 2048, 2047, 1, 256), (2, 700, 350, 0, 5, 8), (1, 70000, 3, 1, 1, 8),
                                                   (1, 60000, 30000, 1000, 2, 64), (2, 500, 250, 30, 2, 96)])  # fmt: skip
def test_evict_shapes_in_place(L, n0, keep, recent, Hk, D):
    g = gen(n0)
    K, V = (torch.randn(L, n0, Hk, D, generator=g, device=DEV).to(BF) for _ in range(2))
    t = torch.rand(L, Hk, n0, generator=g, device=DEV).pow(8)
    K0, V0, t0 = K.clone(), V.clone(), t.clone()
    for _ in range(2):  # (twice from the same start: the same rows)
        K.copy_(K0), V.copy_(V0), t.copy_(t0)
        idx, n_out = evict(K, V, t, n0, keep, recent)
        check_evict(K0, V0, t0, n0, keep, recent, idx, n_out, K, V, t, (K0, V0, t0))
    assert capi.status() == 0


def test_evict_through_row_maps():
    g = gen(21)
    L, Hk, D, pages, n0, keep, recent = 2, 2, 128, 12, 500, 190, 20
    cap = pages * 64
    K, V = (torch.randn(L, cap, Hk, D, generator=g, device=DEV).to(BF) for _ in range(2))
    t = torch.rand(L, Hk, cap, generator=g, device=DEV)

    def table(ids):
        return (torch.tensor(ids, device=DEV, dtype=torch.int32)[:, None] * 64 + torch.arange(64, device=DEV, dtype=torch.int32)).reshape(-1).contiguous()

    tbl = table([7, 2, 9, 0, 4, 11, 3, 8])
    logical = lambda x: x[:, tbl.long()]  # noqa: E731
    K0, V0, t0 = K.clone(), V.clone(), t.clone()
    want = [logical(K0).clone(), logical(V0).clone()]
    # in place through one map
    full = torch.cat([tbl, table([1, 5, 6, 10])])
    idx, n_out = evict(K, V, t, n0, keep, recent, tbl=full, tbl_d=full)
    Kl, Vl = K[:, full.long()], V[:, full.long()]
    check_evict(K0[:, full.long()], V0[:, full.long()], t0, n0, keep, recent, idx, n_out, Kl, Vl, t,
                (K0[:, full.long()], V0[:, full.long()], t0))  # fmt: skip
    # from one map's pages into another cache's
    to = table([3, 0, 2])
    Kd, Vd = (torch.zeros(L, 4 * 64, Hk, D, dtype=BF, device=DEV) for _ in range(2))
    td = torch.zeros(L, Hk, 4 * 64, device=DEV)
    dst_map = torch.cat([to, table([1])])
    idx, n_out = evict(K0.clone(), V0.clone(), t0.clone(), n0, keep, recent, Kd, Vd, td, tbl=full, tbl_d=dst_map)
    zero = torch.zeros_like(Kd)
    check_evict(K0[:, full.long()], V0[:, full.long()], t0, n0, keep, recent, idx, n_out, Kd[:, dst_map.long()],
                Vd[:, dst_map.long()], td, (zero, zero, torch.zeros_like(td)))  # fmt: skip
    assert torch.equal(want[0], logical(K0)) and capi.status() == 0


def test_evict_refuses_a_count_outside_the_cache_and_a_bad_map():
    g = gen(22)
    K, V = (torch.randn(1, 100, 2, 64, generator=g, device=DEV).to(BF) for _ in range(2))
    t = torch.rand(1, 2, 100, generator=g, device=DEV)
    K0, V0, t0 = K.clone(), V.clone(), t.clone()
    for n0 in (101, -1, 1 << 30, -(1 << 31)):
        _, n_out = evict(K, V, t, n0, 50, 10)
        assert torch.equal(K, K0) and torch.equal(V, V0) and torch.equal(t, t0) and int(n_out) == -7
        assert capi.status() == capi.ERR_DOMAIN
    for v in (-1, 100, 1 << 30):
        tbl = torch.arange(100, dtype=torch.int32, device=DEV)
        tbl[99] = v
        evict(K.clone(), V.clone(), t.clone(), 100, 50, 10, torch.zeros_like(K), torch.zeros_like(V), torch.zeros_like(t), tbl=tbl)
        torch.cuda.synchronize()
        assert capi.status() == capi.ERR_DOMAIN


# ---- the engines that run them ---------------------------------------------------------------------------------------------
CFG = E.DenseConfig("long", hidden=256, layers=3, q_heads=8, kv_heads=2, head_dim=128, inter=512, vocab=1000)


def near(a, b):
    """rows of logits of two decodes that differ in the attention's rounding: the engine's own bound"""
    a, b = a.float(), b.float()
    assert float((a - b).abs().max()) <= 2.0**-5 * max(1.0, float(b.abs().max()))


@pytest.mark.parametrize("B,n,steps", [(3, 40, 6), (8, 300, 5), (17, 130, 4)])
def test_forks_over_a_shared_prefix_decode_as_one_sequence_does(B, n, steps):
    mw = E.synth_weights(CFG, seed=1, on_cpu=True, layer_std=LAYER_STD)
    prompt = torch.randint(0, CFG.vocab, (n,), generator=torch.Generator().manual_seed(B))
    plain, eng = RowsEngine(mw, cap=1024), RowsEngine(mw, cap=1024, shared=True)
    assert torch.equal(plain.fork(prompt, B), eng.fork(prompt, B))  # (a prompt's rows go through the same kernels)
    toks = [(7 * b + 1) % CFG.vocab for b in range(B)]
    for i in range(steps):
        a, b = plain.rows_step(toks), eng.rows_step(toks)
        near(b, a)
        toks = a.float().argmax(-1).tolist()
    assert capi.status() == 0
    # a batch of prompts end to end, one row each, in the same engine and the same captured graph
    prompts = [torch.randint(0, CFG.vocab, (20 + 3 * b,), generator=torch.Generator().manual_seed(b)) for b in range(B)]
    for a, b in zip(plain.batch(prompts), eng.batch(prompts)):
        assert torch.equal(a, b)
    for i in range(3):
        a, b = plain.rows_step(toks), eng.rows_step(toks)
        near(b, a)
    assert capi.status() == 0


def test_an_evicting_cache_that_never_fills_decodes_as_the_engine_does():
    mw = E.synth_weights(CFG, seed=2, on_cpu=True, layer_std=LAYER_STD)
    prompt = torch.randint(0, CFG.vocab, (90,), generator=torch.Generator().manual_seed(4))
    flat, eng = E.CardEngine(mw, cap=512), EvictEngine(mw, budget=512)
    near(eng.prefill(prompt), flat.prefill(prompt))
    assert int(eng.n0) == eng.rows == 90 and eng.dropped == 0
    # a chain of rows gives 1 a query head each
    t = eng.totals[:, :, :90].double().sum(-1)
    assert float((t - 90 * 4).abs().max()) < 1e-2
    tok = int(flat.generate_greedy(prompt, 1)[0])
    flat.reset(), flat.prefill(prompt)
    for _ in range(6):
        a, b = flat.forward(torch.tensor([tok])), eng.forward(torch.tensor([tok]))
        near(b, a)
        tok = int(a.float().argmax())
    lively(eng.generate_greedy(prompt, 24))
    assert capi.status() == 0


def test_a_full_cache_lets_rows_go_and_positions_go_on():
    mw = E.synth_weights(CFG, seed=3, on_cpu=True, layer_std=LAYER_STD)
    budget, keep, recent = 160, 64, 16
    eng = EvictEngine(mw, budget=budget, keep=keep, recent=recent, positions=2048)
    prompt = torch.randint(0, CFG.vocab, (budget,), generator=torch.Generator().manual_seed(5))
    eng.prefill(prompt)
    assert eng.rows == budget and eng.dropped == 0
    K0, V0, t0 = eng.K.clone(), eng.V.clone(), eng.totals.clone()
    eng.forward(torch.tensor([11]))  # does not fit: the cache is cut first
    assert eng.rows == int(eng.n0) == keep + 1 and eng.dropped == budget - keep
    for a in range(CFG.layers):
        for h in range(CFG.kv_heads):
            rows = kept_rows(t0[a, h].tolist(), keep, recent)
            assert eng.kept[a, h].tolist() == rows
            assert torch.equal(eng.K[a, :keep, h], K0[a, rows, h]) and torch.equal(eng.V[a, :keep, h], V0[a, rows, h])
    # the new row stands at its own position: the first layer's key depends on the token and the position alone
    flat = E.CardEngine(mw, cap=512)
    flat.prefill(torch.cat([prompt, torch.tensor([11])]))
    assert torch.equal(eng.K[0, keep], flat.K[0, budget]) and torch.equal(eng.V[0, keep], flat.V[0, budget])
    # the captured step evicts by itself as often as it must, and gives the passes' tokens
    eng.reset()
    assert eng.rows == 0 and eng.dropped == 0
    got = eng.generate_greedy(prompt, 300)
    assert eng.dropped > 0 and eng.rows <= budget and eng.dropped + eng.rows == budget + 299
    lively(got)
    two = EvictEngine(mw, budget=budget, keep=keep, recent=recent, positions=2048)
    want, lg = [], two.prefill(prompt)
    for _ in range(300):
        want.append(int(lg[-1].float().argmax()))
        lg = two.forward(torch.tensor(want[-1:]))
    assert got == want
    assert torch.isfinite(eng.totals[:, :, : eng.rows]).all() and capi.status() == 0


def test_an_evicting_cache_refuses_what_it_cannot_do():
    mw = E.synth_weights(CFG, seed=3, on_cpu=True, layer_std=LAYER_STD)
    for kw in (dict(budget=64, keep=64), dict(budget=128, keep=50, recent=51), dict(budget=128, keep=0), dict(budget=128, positions=100)):
        with pytest.raises(ValueError):
            EvictEngine(mw, **kw)
    eng = EvictEngine(mw, budget=128, keep=64, positions=140)
    for f in (lambda: eng.prefill_gemm(torch.arange(4)), eng.session, lambda: eng.generate_speculative(torch.arange(4), 4),
              lambda: eng.forward(torch.arange(4), advance=False), lambda: eng.forward(torch.arange(4), [0, 1, 1, 2], [-1, 0, 0, 1])):  # fmt: skip
        with pytest.raises(TypeError):
            f()
    eng.prefill(torch.arange(138))
    eng.forward(torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        eng.forward(torch.tensor([3]))
    assert eng.rows + eng.dropped == 140 and capi.status() == 0
