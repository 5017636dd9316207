// Attention over long caches for sm_100a. Two entry points: btb_b200_attn_shared, a pass in the rows layout whose rows
// share prefixes, and btb_b200_attn_scored, a chain or tree pass that also adds up what each cache row is given.
#include "common.cuh"
#include "btb_b200_internal.h"
#include "attn_core.cuh"

B2_DEFINE_STATUS(attnl)

#include "../../include/btb_b200.h"

namespace {

struct LongArgs {
    const bf16* q;       // [T, Hq, D]
    const bf16* K;       // kv head g, cache row r at g * hs + r * rs
    const bf16* V;
    bf16* out;           // [T, Hq * D]
    const int* n0p;      // rows standing before the pass ...
    const int* par;      // ... [T] parents, -1 the root ...
    const int* tbl;      // ... and logical row -> cache row, or null
    const int* rw;       // the rows layout (RowSeq), or null; with it n0p, par and tbl are not read
    const float* sinks;  // [Hq] a logit joined to the denominator, or null
    float* totals;       // [Hk, ts] what each logical row has been given, or null
    float* lse;          // [T, Hq] log2 of a row's denominator
    float* own;          // [T, Hq, 32] the scores of the pass's own rows in log2 units, -inf where not seen
    float scale;
    int T, Hq, Hk, win, cap;
    long long hs, rs, ts;
};

// the logical keys of pass row t: [first, last], and the cache row of each
struct Keys {
    int first, last, n0;
    RowSeq seq;
    const int* anc;  // the pass's ancestors of t, root first (chain or tree pass)
    const LongArgs& A;
    __device__ __forceinline__ Keys(const LongArgs& a, int t, int n0_, const int* anc_, int len)
        : n0(n0_), seq(a.rw, t, a.rw != nullptr), anc(anc_), A(a) {
        last = a.rw != nullptr ? seq.position() : n0_ + len - 1;
        first = a.win > 0 ? max(last + 1 - a.win, 0) : 0;
    }
    // -1, and the status word, for a row outside the cache: such a key is not read
    __device__ __forceinline__ int row(int j) const {
        int r;
        if (A.rw != nullptr) {
            r = seq.slot(j);
        } else {
            r = j < n0 ? j : n0 + anc[j - n0];
            if (A.tbl != nullptr) r = A.tbl[r];
        }
        if (r >= 0 && r < A.cap) return r;
        b2_fail(B2_ERR_DOMAIN);
        return -1;
    }
};

constexpr int JW = 8;  // warps of a row's block

// One block a (row, kv head): its warps walk the keys 32 at a time with a running maximum and sum, a lane a key for the
// scores and D / 32 dims for the output; the warps' states are folded at the end.
template <int D, int G>
__global__ void __launch_bounds__(JW * 32) long_rows(const LongArgs A) {
    constexpr int E = D / 32;
    __shared__ __align__(16) uint32_t qs[G][D / 2];
    __shared__ float ps[JW][G][32];
    __shared__ float wm[JW][G], wl[JW][G];
    __shared__ float wo[JW][G][D];
    __shared__ int anc[TMAX];
    __shared__ int s_len;
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, g = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = A.rw != nullptr ? 0 : *A.n0p;
    if (A.rw != nullptr) {
        if (A.rw[5 + 3 * t] < 0) return;  // padding
    } else if (n0 < 0 || n0 > A.cap - A.T) {
        if (threadIdx.x == 0) b2_fail(B2_ERR_DOMAIN);
        return;
    }
    if (threadIdx.x == 0) {
        int len = 0;
        if (A.rw == nullptr) {
            for (int p = t; p >= 0 && p < A.T && len < TMAX; p = A.par[p]) ++len;
            int k = len;
            for (int p = t; k > 0; p = A.par[p]) anc[--k] = p;
        }
        s_len = len;
    }
    for (int i = threadIdx.x; i < G * D / 2; i += JW * 32) {
        const int hh = i / (D / 2), d = i - hh * (D / 2);
        qs[hh][d] = reinterpret_cast<const uint32_t*>(A.q + ((size_t)t * A.Hq + g * G + hh) * D)[d];
    }
    if (A.own != nullptr)
        for (int i = threadIdx.x; i < G * 32; i += JW * 32) A.own[((size_t)t * A.Hq + g * G) * 32 + i] = NEG_INF;
    __syncthreads();
    const Keys keys(A, t, n0, anc, s_len);
    const float scale2 = __fmul_rn(A.scale, LOG2E);
    const bf16* Kg = A.K + (size_t)g * A.hs;
    const bf16* Vg = A.V + (size_t)g * A.hs;
    float m[G], l[G], o[G][E];
#pragma unroll
    for (int hh = 0; hh < G; ++hh) {
        m[hh] = NEG_INF, l[hh] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[hh][e] = 0.f;
    }
    for (int j0 = keys.first + warp * 32; j0 <= keys.last; j0 += JW * 32) {
        const int j = j0 + lane;
        const int row = j <= keys.last ? keys.row(j) : -1;
        float s[G];
#pragma unroll
        for (int hh = 0; hh < G; ++hh) s[hh] = 0.f;
        if (row >= 0) {
            const uint4* kr = reinterpret_cast<const uint4*>(Kg + (size_t)row * A.rs);
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
                const uint4 kv = __ldg(kr + c);
#pragma unroll
                for (int hh = 0; hh < G; ++hh) {
                    const uint4 q4 = *reinterpret_cast<const uint4*>(&qs[hh][c * 4]);
                    s[hh] = fma2_bf16(kv.w, q4.w, fma2_bf16(kv.z, q4.z, fma2_bf16(kv.y, q4.y, fma2_bf16(kv.x, q4.x, s[hh]))));
                }
            }
        }
#pragma unroll
        for (int hh = 0; hh < G; ++hh) {
            s[hh] = row >= 0 ? __fmul_rn(s[hh], scale2) : NEG_INF;
            if (A.own != nullptr && j >= n0 && j <= keys.last)
                A.own[((size_t)t * A.Hq + g * G + hh) * 32 + anc[j - n0]] = s[hh];
            float mx = s[hh];
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
            const float mn = fmaxf(m[hh], mx);
            const float c = m[hh] == NEG_INF ? 0.f : ex2(m[hh] - mn);
            const float p = s[hh] == NEG_INF ? 0.f : ex2(s[hh] - mn);
            l[hh] = l[hh] * c + warp_sum(p);
            m[hh] = mn;
            ps[warp][hh][lane] = p;
#pragma unroll
            for (int e = 0; e < E; ++e) o[hh][e] *= c;
        }
        __syncwarp();
        for (int i = 0; i < 32; ++i) {
            const int r = __shfl_sync(0xffffffffu, row, i);
            if (r < 0) continue;
            __align__(8) bf16 v[E];
            ld_run<E, false>(Vg + (size_t)r * A.rs + lane * E, v);
#pragma unroll
            for (int hh = 0; hh < G; ++hh)
#pragma unroll
                for (int e = 0; e < E; ++e) o[hh][e] = fmaf(ps[warp][hh][i], bf2f(v[e]), o[hh][e]);
        }
        __syncwarp();
    }
#pragma unroll
    for (int hh = 0; hh < G; ++hh) {
        if (lane == 0) wm[warp][hh] = m[hh], wl[warp][hh] = l[hh];
#pragma unroll
        for (int e = 0; e < E; ++e) wo[warp][hh][lane * E + e] = o[hh][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G * D; i += JW * 32) {
        const int hh = i / D, d = i - hh * D, head = g * G + hh;
        float M = NEG_INF, L = 0.f, O = 0.f, cO, co;
        for (int w = 0; w < JW; ++w) {
            fold_ml(M, L, wm[w][hh], wl[w][hh], cO, co);
            O = fold_e(O, wo[w][hh][d], cO, co);
        }
        if (A.sinks != nullptr) {
            fold_ml(M, L, __fmul_rn(A.sinks[head], LOG2E), 1.f, cO, co);
            O = __fmul_rn(O, cO);
        }
        A.out[((size_t)t * A.Hq + head) * D + d] = f2bf(__fdiv_rn(O, L));
        if (d == 0 && A.lse != nullptr) A.lse[(size_t)t * A.Hq + head] = M + log2f(L);
    }
}

constexpr int WK = 128;  // keys of a weights block

// What the pass gives each cache row: a thread a key, its score against every row's query again and the weights
// 2^(score - lse) added in row order, so that a total is one sum in one order. The pass's own rows are set, not added to.
template <int D, int G>
__global__ void __launch_bounds__(WK) long_weights(const LongArgs A) {
    extern __shared__ __align__(16) uint32_t dyn[];  // the kv head's queries, [T * G][D / 2]
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.y, n0 = *A.n0p, j = blockIdx.x * WK + threadIdx.x;
    if (n0 < 0 || n0 > A.cap - A.T) return;
    float* tot = A.totals + (size_t)g * A.ts;
    if (blockIdx.x == 0 && threadIdx.x < A.T) {
        float a = 0.f;
        for (int t = 0; t < A.T; ++t)
            for (int hh = 0; hh < G; ++hh) {
                const size_t r = (size_t)t * A.Hq + g * G + hh;
                a += ex2(A.own[r * 32 + threadIdx.x] - A.lse[r]);
            }
        tot[n0 + threadIdx.x] = a;
    }
    if ((int)blockIdx.x * WK >= n0) return;
    for (int i = threadIdx.x; i < A.T * G * (D / 2); i += WK) {
        const int r = i / (D / 2), d = i - r * (D / 2);
        dyn[i] = reinterpret_cast<const uint32_t*>(A.q + ((size_t)(r / G) * A.Hq + g * G + r % G) * D)[d];
    }
    __syncthreads();
    if (j >= n0) return;
    const int row = A.tbl != nullptr ? A.tbl[j] : j;
    if (row < 0 || row >= A.cap) return;  // refused by the pass over the rows
    uint4 kv[D / 8];
    const uint4* kr = reinterpret_cast<const uint4*>(A.K + (size_t)g * A.hs + (size_t)row * A.rs);
#pragma unroll
    for (int c = 0; c < D / 8; ++c) kv[c] = __ldg(kr + c);
    const float scale2 = __fmul_rn(A.scale, LOG2E);
    float a = 0.f;
    for (int r = 0; r < A.T * G; ++r) {
        const uint4* q4 = reinterpret_cast<const uint4*>(dyn + r * (D / 2));
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
            const uint4 w = q4[c];
            s = fma2_bf16(kv[c].w, w.w, fma2_bf16(kv[c].z, w.z, fma2_bf16(kv[c].y, w.y, fma2_bf16(kv[c].x, w.x, s))));
        }
        a += ex2(__fmul_rn(s, scale2) - A.lse[(size_t)(r / G) * A.Hq + g * G + r % G]);
    }
    tot[j] += a;
}

template <int D, int G>
int launch_long(const LongArgs& a, cudaStream_t s) {
    if (const int rc = b2_launch(reinterpret_cast<const void*>(long_rows<D, G>), dim3(a.T, a.Hk), dim3(JW * 32), 0, s, a)) return rc;
    if (a.totals == nullptr) return B2_OK;
    auto kern = long_weights<D, G>;
    static bool allowed[64];
    if (const int rc = b2_allow_smem(reinterpret_cast<const void*>(kern), allowed)) return rc;
    return b2_launch(reinterpret_cast<const void*>(kern), dim3((a.cap + WK - 1) / WK, a.Hk), dim3(WK), (size_t)a.T * G * D * 2, s, a);
}
template <int D>
int launch_long_g(const LongArgs& a, cudaStream_t s) {
    switch (a.Hq / a.Hk) {
        case 1: return launch_long<D, 1>(a, s);
        case 2: return launch_long<D, 2>(a, s);
        case 4: return launch_long<D, 4>(a, s);
        case 8: return launch_long<D, 8>(a, s);
        default: return B2_ERR_DOMAIN;
    }
}

bool shape_ok(int T, int Hq, int Hk, int D) {
    return T > 0 && T <= TMAX && Hk > 0 && Hk <= 65535 && Hq > 0 && Hq % Hk == 0 &&
           (Hq / Hk == 1 || Hq / Hk == 2 || Hq / Hk == 4 || Hq / Hk == 8) && (D == 64 || D == 128);
}
bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// what both entry points refuse: a shape no kernel serves, and a cache that does not lie in 16-byte pieces - kv heads
// inside a cache row (hs < rs) or each head's rows on their own (hs a multiple of rs)
int check_cache(const void* q, const void* K, const void* V, const void* out, int T, int Hq, int Hk, int D, long long hs,
                long long rs, float scale, const void* workspace, int cap) {
    if (!shape_ok(T, Hq, Hk, D) || cap <= 0 || !(scale == scale) || hs < D || rs < D || (hs & 7) || (rs & 7)) return B2_ERR_DOMAIN;
    if (Hk > 1 && !((Hk - 1) * hs + D <= rs || (hs % rs == 0 && hs / rs >= cap))) return B2_ERR_DOMAIN;
    if (misaligned(q) || misaligned(K) || misaligned(V) || misaligned(out) || misaligned(workspace)) return B2_ERR_DOMAIN;
    return B2_OK;
}

}  // namespace

extern "C" size_t btb_b200_attn_shared_workspace_bytes(int T, int Hq, int Hk, int D) {
    return shape_ok(T, Hq, Hk, D) ? 16 : 0;
}

extern "C" int btb_b200_attn_shared(const void* q, const void* K, const void* V, void* out, const void* rw, int T, int Hq,
                                    int Hk, int D, long long hs, long long rs, float scale, void* workspace, int win,
                                    const void* sinks, int cap, void* stream) {
    if (!q || !K || !V || !out || !rw || !workspace) return B2_ERR_NULL;
    if (const int rc = check_cache(q, K, V, out, T, Hq, Hk, D, hs, rs, scale, workspace, cap)) return rc;
    LongArgs a{};
    a.q = static_cast<const bf16*>(q), a.K = static_cast<const bf16*>(K), a.V = static_cast<const bf16*>(V);
    a.out = static_cast<bf16*>(out), a.rw = static_cast<const int*>(rw), a.sinks = static_cast<const float*>(sinks);
    a.scale = scale, a.T = T, a.Hq = Hq, a.Hk = Hk, a.win = win, a.cap = cap, a.hs = hs, a.rs = rs;
    return D == 64 ? launch_long_g<64>(a, static_cast<cudaStream_t>(stream)) : launch_long_g<128>(a, static_cast<cudaStream_t>(stream));
}

extern "C" size_t btb_b200_attn_scored_workspace_bytes(int T, int Hq, int Hk, int D, int cap) {
    if (!shape_ok(T, Hq, Hk, D) || cap <= 0) return 0;
    return (size_t)T * Hq * 33 * 4;
}

extern "C" int btb_b200_attn_scored(const void* q, const void* K, const void* V, void* out, const void* n0p, const void* par,
                                    int T, int Hq, int Hk, int D, long long hs, long long rs, float scale, void* totals,
                                    long long ts, void* workspace, const void* tbl, const void* sinks, int cap, void* stream) {
    if (!q || !K || !V || !out || !n0p || !par || !totals || !workspace) return B2_ERR_NULL;
    if (const int rc = check_cache(q, K, V, out, T, Hq, Hk, D, hs, rs, scale, workspace, cap)) return rc;
    if (ts < cap) return B2_ERR_DOMAIN;
    LongArgs a{};
    a.q = static_cast<const bf16*>(q), a.K = static_cast<const bf16*>(K), a.V = static_cast<const bf16*>(V);
    a.out = static_cast<bf16*>(out), a.n0p = static_cast<const int*>(n0p), a.par = static_cast<const int*>(par);
    a.tbl = static_cast<const int*>(tbl), a.sinks = static_cast<const float*>(sinks);
    a.totals = static_cast<float*>(totals), a.ts = ts;
    a.lse = static_cast<float*>(workspace), a.own = a.lse + (size_t)T * Hq;
    a.scale = scale, a.T = T, a.Hq = Hq, a.Hk = Hk, a.cap = cap, a.hs = hs, a.rs = rs;
    return D == 64 ? launch_long_g<64>(a, static_cast<cudaStream_t>(stream)) : launch_long_g<128>(a, static_cast<cudaStream_t>(stream));
}
