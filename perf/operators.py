"""Cases for timing the long-cache operators: the attention of rows that share a prefix (`btb_b200_attn_shared`), the
attention that adds up what each cache row is given (`btb_b200_attn_scored`) and the eviction by those totals
(`btb_b200_kv_evict`). `run` computes a case in elementary torch operations, or with `own` set through the library."""

import math

import torch

own = False

# (query heads, kv heads, head dim): the configurations' models - 4 B dense, 30 B and 20 B mixtures, 70 B dense
Q4, A3, OSS, L70 = (32, 8, 128), (32, 4, 128), (64, 8, 64), (64, 8, 128)


def _shared(name, T, prompts, n, steps, heads, sinks=False, win=0):
    return {"name": name, "op": "shared", "T": T, "prompts": prompts, "n": n, "steps": steps, "Hq": heads[0],
            "Hk": heads[1], "D": heads[2], "sinks": sinks, "win": win}  # fmt: skip


def _scored(name, T, n, heads, tree=False, paged=False, sinks=False):
    return {"name": name, "op": "scored", "T": T, "n": n, "Hq": heads[0], "Hk": heads[1], "D": heads[2], "tree": tree,
            "paged": paged, "sinks": sinks}  # fmt: skip


def _evict(name, layers, n, keep, recent, heads, inplace=False):
    return {"name": name, "op": "evict", "layers": layers, "n": n, "keep": keep, "recent": recent, "Hk": heads[1],
            "D": heads[2], "inplace": inplace}  # fmt: skip


def listed():
    return [
        # two continuations of a short prompt, their first step: the smallest call, all latency
        _shared("shared 2 of 128", 2, 1, 128, 0, Q4),
        # eight samples of a 2048-token prompt well into their answers, the lengths of the 4 B model's batch workload
        _shared("shared 8 of 2048", 8, 1, 2048, 255, Q4),
        # four prompts of odd lengths, four samples each, with sinks (the 20 B mixture's attention)
        _shared("shared 4x4 of 1021 sinks", 16, 4, 1021, 60, OSS, sinks=True),
        # thirty-two samples of a 32768-token prompt (the 70 B model's workload): the largest
        _shared("shared 32 of 32768", 32, 1, 32768, 127, L70),
        # a decode step over a short cache
        _scored("scored 1 of 127", 1, 127, Q4),
        # a decode step over a conversation's cache in pages of 64 rows, the last page part full
        _scored("scored 1 of 4001 paged", 1, 4001, Q4, paged=True),
        # a draft tree of nine rows verified over a 613-row cache (the 30 B mixture's workload)
        _scored("scored tree 9 of 613", 9, 613, A3, tree=True),
        # a 32-row prompt chunk with sinks
        _scored("scored 32 of 2015 sinks", 32, 2015, OSS, sinks=True),
        # the decode step at the end of a 32768-token prompt
        _scored("scored 1 of 32768", 1, 32768, L70),
        # one layer of a short cache halved in place
        _evict("evict 1 layer 257 to 128", 1, 257, 128, 32, Q4, inplace=True),
        # the 4 B model's whole cache cut from 4096 rows to 2048, all 36 layers in place
        _evict("evict 36 layers 4096 to 2048", 36, 4096, 2048, 256, Q4, inplace=True),
        # sixteen layers of a 32767-row cache gathered into a cache a quarter the size
        _evict("evict 16 layers 32767 to 8191", 16, 32767, 8191, 512, L70),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(("shared", "shared", "scored", "scored", "evict"))
    heads = rng.choice((Q4, A3, OSS, L70, (8, 8, 128), (16, 8, 64), (4, 1, 128)))
    if op == "shared":
        T = _log(rng, 1, 32)
        prompts = rng.choice((1, 1, 1, 2, min(T, 5)))
        prompts = min(prompts, T)
        n = _log(rng, 3, 32768 // prompts)
        c = _shared("", T, prompts, n, _log(rng, 1, 400) - 1, heads, rng.random() < 0.3, rng.choice((0, 0, 0, 128, 1000)))
    elif op == "scored":
        T = rng.choice((1, 1, 1, _log(rng, 2, 32)))
        c = _scored("", T, _log(rng, 1, 32768), heads, rng.random() < 0.3, rng.random() < 0.4, rng.random() < 0.3)
    else:
        n = _log(rng, 40, 32768)
        keep = max(1, int(n * rng.uniform(0.1, 0.95)))
        layers = max(1, min(_log(rng, 1, 36), 500_000 // n))
        c = _evict("", layers, n, keep, int(keep * rng.uniform(0.0, 0.5)), heads, rng.random() < 0.5)
    del c["name"]
    return c


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _queries_and_cache(g, T, rows, Hq, Hk, D):
    """rotated queries and a cache's keys and values: keys lean by differing amounts on a direction that their head's
    queries share, so that a few rows take much of the weight and most take little"""
    dev = "cuda"
    u = torch.randn(Hk, D, generator=g, device=dev)
    q = torch.randn(T, Hk, Hq // Hk, D, generator=g, device=dev) + 0.5 * u[None, :, None]
    lean = torch.randn(rows, Hk, 1, generator=g, device=dev)
    k = torch.randn(rows, Hk, D, generator=g, device=dev) + 0.35 * lean * u
    v = torch.randn(rows, Hk, D, generator=g, device=dev)
    return q.reshape(T, Hq, D).bfloat16(), k.bfloat16(), v.bfloat16()


def _layout(c):
    """the rows layout's integers: [base, step, W, (col, off, len) a row] - prompts end to end, each with its forks"""
    T, P, n = c["T"], c["prompts"], c["n"]
    W = next(m for m in (1, 2, 4, 8, 16, 32) if T <= m)
    lens = [max(1, n - 37 * p) for p in range(P)]
    offs = [sum(lens[:p]) for p in range(P)]
    base = sum(lens)
    lay = [base, c["steps"], W]
    for t in range(T):
        p = t * P // T
        lay += [t, offs[p], lens[p]]
    return lay + [0, 0, -1] * (W - T), W, base + (c["steps"] + 1) * W


def _parents(c):
    # a chain, or a tree of drafts: the root, then three branches that grow in turn
    return [t - 1 if not c["tree"] else (-1 if t == 0 else 0 if t <= 3 else t - 3) for t in range(c["T"])]


def prepare(case, seed):
    c, g, dev = case, _gen(seed), "cuda"
    s = {"case": c}
    if c["op"] == "shared":
        lay, W, rows = _layout(c)
        q, k, v = _queries_and_cache(g, W, rows, c["Hq"], c["Hk"], c["D"])
        s.update(q=q, K=k, V=v, rw=torch.tensor(lay, dtype=torch.int32, device=dev), cap=rows, W=W,
                 out=torch.zeros(W, c["Hq"] * c["D"], dtype=torch.bfloat16, device=dev))  # fmt: skip
    elif c["op"] == "scored":
        T, n = c["T"], c["n"]
        cap = -(-(n + T) // 64) * 64 + 64
        q, k, v = _queries_and_cache(g, T, cap, c["Hq"], c["Hk"], c["D"])
        tbl = None
        if c["paged"]:
            pages = torch.randperm(cap // 64, generator=g, device=dev).int()
            tbl = (pages[:, None] * 64 + torch.arange(64, device=dev, dtype=torch.int32)).reshape(-1).contiguous()
        few = 8.0 * T * (c["Hq"] // c["Hk"]) / (n + T)  # what some steps have given the rows: a step's own share still tells
        s.update(q=q, K=k, V=v, tbl=tbl, cap=cap, n0=torch.full((1,), n, dtype=torch.int32, device=dev),
                 par=torch.tensor(_parents(c), dtype=torch.int32, device=dev),
                 totals=torch.rand(c["Hk"], cap, generator=g, device=dev) * few,
                 out=torch.zeros(T, c["Hq"] * c["D"], dtype=torch.bfloat16, device=dev))  # fmt: skip
    else:
        L, n, Hk, D = c["layers"], c["n"], c["Hk"], c["D"]
        cap, capd = n + 3, (n + 3 if c["inplace"] else c["keep"] + 5)
        make = lambda: torch.randn(L, cap, Hk, D, generator=g, device=dev, dtype=torch.bfloat16)  # noqa: E731
        # totals as a decode leaves them: most rows little, a few much, the rows no query looked at equal (zero)
        tot = torch.rand(L, Hk, cap, generator=g, device=dev).pow(8) * 50
        tot[tot < 0.01] = 0
        s.update(K=make(), V=make(), totals=tot, cap=cap, capd=capd, n0=torch.full((1,), n, dtype=torch.int32, device=dev),
                 n_out=torch.zeros(1, dtype=torch.int32, device=dev),
                 idx=torch.full((L, Hk, c["keep"]), -1, dtype=torch.int32, device=dev))  # fmt: skip
        if c["inplace"]:
            s.update(Kd=s["K"], Vd=s["V"], totals_d=s["totals"])
        else:
            s.update(Kd=torch.zeros(L, capd, Hk, D, dtype=torch.bfloat16, device=dev),
                     Vd=torch.zeros(L, capd, Hk, D, dtype=torch.bfloat16, device=dev),
                     totals_d=torch.zeros(L, Hk, capd, device=dev))  # fmt: skip
    if c["op"] != "evict":
        s["sinks"] = torch.randn(c["Hq"], generator=g, device=dev) if c["sinks"] else None
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _weights(q, k, see, sinks, Hk, scale):
    """softmax weights [Hk, G, T, rows] in f32 of queries [T, Hq, D] over keys [rows, Hk, D]; `see` [T, rows]"""
    T, Hq, D = q.shape
    qf = q.float().reshape(T, Hk, Hq // Hk, D).permute(1, 2, 0, 3)
    s = torch.matmul(qf, k.float().permute(1, 2, 0).unsqueeze(1)) * scale
    s = s.masked_fill(~see, float("-inf"))
    m = s.amax(-1, keepdim=True)
    if sinks is not None:
        sk = sinks.reshape(Hk, Hq // Hk, 1, 1)
        m = torch.maximum(m, sk)
    m = torch.where(m == float("-inf"), 0.0, m)
    w = torch.exp(s - m)
    z = w.sum(-1, keepdim=True)
    if sinks is not None:
        z = z + torch.exp(sk - m)
    return w / z


def _mix(w, v):
    """[Hk, G, T, rows] weights over [rows, Hk, D] values -> [T, Hq * D]"""
    o = torch.matmul(w, v.float().permute(1, 0, 2).unsqueeze(1))
    return o.permute(2, 0, 1, 3).reshape(w.shape[2], -1)


def _plain_shared(s):
    c = s["case"]
    rw = s["rw"].long()
    base, step, W = rw[0], rw[1], rw[2]
    col, off, ln = rw[3:].reshape(-1, 3).T.unsqueeze(-1)
    j = torch.arange(s["cap"], device="cuda")
    first = (ln + step + 1 - c["win"]).clamp(min=0) if c["win"] else torch.zeros_like(ln)
    i = torch.div(j - base, W, rounding_mode="floor")
    see = ((j >= off + first) & (j < off + ln) & (j < base)) | ((j >= base) & ((j - base) % W == col) & (i <= step) & (ln + i >= first))
    T = c["T"]  # (padding rows past T are not computed: their output stays as it is)
    w = _weights(s["q"][:T], s["K"], see[:T], s["sinks"], c["Hk"], c["D"] ** -0.5)
    s["out"][:T] = _mix(w, s["V"]).bfloat16()
    return s["out"]


def _plain_scored(s):
    c = s["case"]
    T, n = c["T"], c["n"]
    rows = torch.arange(n + T, device="cuda")
    if s["tbl"] is not None:
        rows = s["tbl"][rows].long()
    # row t sees the n standing rows, itself and its ancestors: paths by doubling the one-step relation
    step = (s["par"].long()[:, None] == torch.arange(T, device="cuda")).float() + torch.eye(T, device="cuda")
    path = torch.linalg.matrix_power(step, T) > 0
    see = torch.cat([torch.ones(T, n, dtype=torch.bool, device="cuda"), path], 1)
    w = _weights(s["q"], s["K"][rows], see, s["sinks"], c["Hk"], c["D"] ** -0.5)
    s["out"].copy_(_mix(w, s["V"][rows]))
    given = w.sum((1, 2))
    s["totals"][:, :n] += given[:, :n]
    s["totals"][:, n : n + T] = given[:, n:]
    return s["out"], s["totals"]


def _plain_evict(s):
    c = s["case"]
    L, n, keep, recent, Hk = c["layers"], c["n"], c["keep"], c["recent"], c["Hk"]
    order = torch.sort(s["totals"][:, :, : n - recent], dim=-1, descending=True, stable=True).indices
    best = torch.sort(order[:, :, : keep - recent], dim=-1).values
    idx = torch.cat([best, torch.arange(n - recent, n, device="cuda").expand(L, Hk, recent)], -1)
    la, ha = torch.arange(L, device="cuda")[:, None, None], torch.arange(Hk, device="cuda")[:, None]
    for src, dst in ((s["K"], s["Kd"]), (s["V"], s["Vd"])):
        dst[:, :keep] = src[la, idx, ha].transpose(1, 2)
    s["totals_d"][:, :, :keep] = torch.gather(s["totals"], -1, idx)
    s["idx"].copy_(idx)
    s["n_out"].fill_(keep)
    return s["Kd"], s["Vd"], s["totals_d"], s["idx"], s["n_out"]


# ---- the library's calls ---------------------------------------------------------------------------------------------
def _own_workspace(s, name, *dims):
    from btb_b200 import capi

    if "ws" not in s:
        s["ws"] = torch.empty(int(getattr(capi.lib(), name)(*dims)), dtype=torch.uint8, device="cuda")
    return s["ws"]


def _own_shared(s):
    from btb_b200.capi import call, ptr, stream_ptr

    c, W = s["case"], s["W"]
    Hq, Hk, D = c["Hq"], c["Hk"], c["D"]
    ws = _own_workspace(s, "btb_b200_attn_shared_workspace_bytes", W, Hq, Hk, D)
    call("btb_b200_attn_shared", ptr(s["q"]), ptr(s["K"]), ptr(s["V"]), ptr(s["out"]), ptr(s["rw"]), W, Hq, Hk, D, D,
         Hk * D, D**-0.5, ptr(ws), c["win"], ptr(s["sinks"]), s["cap"], stream_ptr())  # fmt: skip
    return s["out"]


def _own_scored(s):
    from btb_b200.capi import call, ptr, stream_ptr

    c = s["case"]
    T, Hq, Hk, D = c["T"], c["Hq"], c["Hk"], c["D"]
    ws = _own_workspace(s, "btb_b200_attn_scored_workspace_bytes", T, Hq, Hk, D, s["cap"])
    call("btb_b200_attn_scored", ptr(s["q"]), ptr(s["K"]), ptr(s["V"]), ptr(s["out"]), ptr(s["n0"]), ptr(s["par"]), T, Hq,
         Hk, D, D, Hk * D, D**-0.5, ptr(s["totals"]), s["cap"], ptr(ws), ptr(s["tbl"]), ptr(s["sinks"]), s["cap"],
         stream_ptr())  # fmt: skip
    return s["out"], s["totals"]


def _own_evict(s):
    from btb_b200.capi import call, ptr, stream_ptr

    c = s["case"]
    L, Hk, D = c["layers"], c["Hk"], c["D"]
    row = Hk * D
    ws = _own_workspace(s, "btb_b200_kv_evict_workspace_bytes", L, Hk, s["cap"])
    call("btb_b200_kv_evict", ptr(s["K"]), ptr(s["V"]), ptr(s["totals"]), ptr(s["n0"]), ptr(s["Kd"]), ptr(s["Vd"]),
         ptr(s["totals_d"]), ptr(s["n_out"]), ptr(s["idx"]), L, s["cap"] * row, s["capd"] * row, Hk, D, D, row, s["cap"],
         s["capd"], c["keep"], c["recent"], 0, 0, ptr(ws), stream_ptr())  # fmt: skip
    return s["Kd"], s["Vd"], s["totals_d"], s["idx"], s["n_out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_shared(state) if op == "shared" else _own_scored(state) if op == "scored" else _own_evict(state)
    return _plain_shared(state) if op == "shared" else _plain_scored(state) if op == "scored" else _plain_evict(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "shared":
        lay, W, _ = _layout(c)
        rows, keys, seen = 0, 0, set()
        for t in range(c["T"]):
            off, ln = lay[4 + 3 * t], lay[5 + 3 * t]
            first = max(0, ln + c["steps"] + 1 - c["win"]) if c["win"] else 0
            prefix, steps = max(0, ln - first), min(c["steps"] + 1, ln + c["steps"] + 1 - first)
            rows += steps + (0 if off in seen else prefix)
            keys += prefix + steps
            seen.add(off)
        return {"bytes": rows * 4 * c["Hk"] * c["D"] + 4 * c["T"] * c["Hq"] * c["D"], "flops": 4 * c["D"] * c["Hq"] * keys}
    if c["op"] == "scored":
        T, n = c["T"], c["n"]
        return {"bytes": (n + T) * 4 * c["Hk"] * c["D"] + 4 * T * c["Hq"] * c["D"] + c["Hk"] * (8 * n + 4 * T),
                "flops": 4 * c["D"] * c["Hq"] * T * (n + T / 2)}  # fmt: skip
    heads = c["layers"] * c["Hk"]
    return {"bytes": heads * (4 * c["n"] + c["keep"] * (8 * c["D"] + 8)), "flops": 0}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------
def _one_row(q, k, v, sinks, Hk, D):
    """one row's output [Hq, D] and weights [Hq, rows] over its own keys [rows, Hk, D], f64"""
    Hq = q.shape[0]
    out, wts = [], []
    for h in range(Hq):
        kh, vh = k[:, h * Hk // Hq].double(), v[:, h * Hk // Hq].double()
        s = (kh @ q[h].double()) / math.sqrt(D)
        if sinks is not None:
            s = torch.cat([s, sinks[h].double().reshape(1)])
        w = torch.softmax(s, 0)[: kh.shape[0]]
        out.append(w @ vh)
        wts.append(w)
    return torch.stack(out), torch.stack(wts)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "shared":
        lay = s["rw"].tolist()
        base, step, W = lay[:3]
        out = torch.zeros(s["W"], c["Hq"] * c["D"], dtype=torch.float64, device="cuda")
        for t in range(c["T"]):
            col, off, ln = lay[3 + 3 * t : 6 + 3 * t]
            keys = list(range(off, off + ln)) + [base + i * W + col for i in range(step + 1)]
            keys = torch.tensor(keys[-c["win"] :] if c["win"] else keys, device="cuda")
            out[t] = _one_row(s["q"][t], s["K"][keys], s["V"][keys], s["sinks"], c["Hk"], c["D"])[0].reshape(-1)
        return out
    if c["op"] == "scored":
        T, n, Hk = c["T"], c["n"], c["Hk"]
        par, tot = _parents(c), s["totals"].double()
        tot[:, n : n + T] = 0
        out = torch.zeros(T, c["Hq"] * c["D"], dtype=torch.float64, device="cuda")
        for t in range(T):
            path, p = [], t
            while p >= 0:
                path.append(n + p)
                p = par[p]
            j = torch.tensor(list(range(n)) + path[::-1], device="cuda")
            r = j if s["tbl"] is None else s["tbl"][j].long()
            o, w = _one_row(s["q"][t], s["K"][r], s["V"][r], s["sinks"], Hk, c["D"])
            out[t] = o.reshape(-1)
            tot[:, j] += w.reshape(Hk, -1, w.shape[1]).sum(1)
        return out, tot
    # (moved values have no other value in 64 bits; which rows they are is held by the indices, which have to be equal)
    tot, keep, recent, n = s["totals"].double(), c["keep"], c["recent"], c["n"]
    got = s["totals_d"].double().clone()
    for a in range(c["layers"]):
        for h in range(c["Hk"]):
            x = tot[a, h, : n - recent]
            m = keep - recent
            cut = torch.topk(x, m).values[-1] if m else math.inf
            above = x > cut
            tied = (x == cut) & (torch.cumsum((x == cut).int(), 0) <= m - int(above.sum()))
            rows = torch.cat([torch.nonzero(above | tied).flatten(), torch.arange(n - recent, n, device="cuda")])
            got[a, h, :keep] = tot[a, h, rows]
    return None, None, got, None, None
