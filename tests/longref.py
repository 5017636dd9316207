"""The long-cache operators from their definitions in 64 bits, and how far a kernel may be from them."""

import math

import torch

EPS_BF16 = torch.finfo(torch.bfloat16).eps / 2  # half a step, relative
EPS_F32 = torch.finfo(torch.float32).eps / 2


def attend(q, K, V, rows, sinks=None):
    """one pass row over the cache rows `rows` of each kv head: output [Hq, D], weights [Hq, n], and the bound on the
    output's error. q [Hq, D], K and V [Hk, cap, D], rows [n] (the same for every head)."""
    Hq, D = q.shape
    Hk = K.shape[0]
    k, v = K[:, rows].double(), V[:, rows].double()
    qg = q.double().reshape(Hk, Hq // Hk, D)
    s = torch.einsum("ghd,gnd->ghn", qg, k) / math.sqrt(D)
    if sinks is not None:
        s = torch.cat([s, sinks.double().reshape(Hk, -1, 1)], -1)
    w = torch.softmax(s, -1)[..., : len(rows)]
    out = torch.einsum("ghn,gnd->ghd", w, v)
    # scores: D products added in f32 (each addition off by at most a step), the scaling, the difference to the maximum
    # and the power of two each a few units in the last place of a score; so a weight's relative error
    big = torch.einsum("ghd,gnd->ghn", qg.abs(), k.abs()).amax() / math.sqrt(D) if len(rows) else torch.zeros((), device=q.device)
    rel = 2 * (D + 16) * EPS_F32 * (float(big) + 1) + 8 * EPS_F32
    # the output: rounded to bf16 once, its weights rounded to bf16 once before they multiply the values (half a step
    # each), both sums' own error rel + n EPS_F32
    spread = torch.einsum("ghn,gnd->ghd", w, v.abs())
    tol = EPS_BF16 * (out.abs() + spread) * (1 + 2 * EPS_BF16) + (2 * rel + 2 * len(rows) * EPS_F32) * spread
    return out.reshape(Hq, D), w.reshape(Hq, -1), tol.reshape(Hq, D), rel


def rows_keys(lay, t, win=0):
    """the cache rows of row t of a rows layout, in logical order"""
    base, step, W = lay[:3]
    col, off, ln = lay[3 + 3 * t : 6 + 3 * t]
    keys = list(range(off, off + ln)) + [base + i * W + col for i in range(step + 1)]
    return keys[-win:] if win else keys


def path_keys(par, t, n0):
    """the logical rows of row t of a chain or tree pass after n0 rows"""
    path, p = [], t
    while p >= 0:
        path.append(n0 + p)
        p = par[p]
    return list(range(n0)) + path[::-1]


def rank(v):
    """a total's place in the order evictions go by: NaN above all, -0 as 0"""
    return math.inf if v != v else v + 0.0, v != v


def kept_rows(totals, keep, recent):
    """the rows one kv head keeps of its `totals` (a list of floats), ascending"""
    n = len(totals)
    if n <= keep:
        return list(range(n))
    order = sorted(range(n - recent), key=lambda j: (not totals[j] != totals[j], -rank(totals[j])[0], j))
    return sorted(order[: keep - recent]) + list(range(n - recent, n))
