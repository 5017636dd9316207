// Eviction from a cache by accumulated attention weight, for sm_100a: per (layer, kv head) the `recent` last rows stay,
// and of the others the keep - recent with the largest totals, the lower row first among equals. The kept rows move
// down in order, their keys, values and totals with them, in place or into another cache.
//
// Two launches. evict_pick: a block a (layer, kv head) finds the rows from its totals and moves those. evict_move: the keys
// and values, bound by memory - every kept row read and written once.
#include "common.cuh"
#include "btb_b200_internal.h"

B2_DEFINE_STATUS(evict)

#include "../../include/btb_b200.h"

namespace {

struct EvictArgs {
    const bf16* K;        // layer a, kv head g, cache row r at a * ls + g * hs + r * rs
    const bf16* V;
    const float* totals;  // [layers, Hk, cap]
    const int* n0p;       // rows standing
    bf16* Kd;             // the same with ld in ls's place
    bf16* Vd;
    float* totals_d;      // [layers, Hk, cap_d]
    int* n_out;           // rows kept
    int* idx;             // [layers, Hk, keep] the kept rows in order, -1 past the count
    const int* tbl;       // logical row -> cache row of the source and of the destination, or null
    const int* tbl_d;
    int* n_seen;          // n0 as the selection read it (n_out may be n0p's word)
    long long ls, ld, hs, rs;
    int layers, Hk, D, cap, cap_d, keep, recent;
    int held;             // the ranks of a head fit a block's shared memory
    int parts;            // evict_move: blocks that share a (layer, kv head, K or V): pieces of a row in place, else ranges of rows
    int in_place;
};

// a total's rank as an unsigned word: larger totals rank higher, -0 as 0, every NaN above all else
__device__ __forceinline__ uint32_t rank_of(uint32_t bits) {
    const float v = __uint_as_float(bits);
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int ST = 1024, SW = ST / 32;  // threads and warps of a selection block
constexpr int BINS = 2048;              // eleven bits of the rank at a time: 11, 11, 10

// The rank of the last kept total, eleven bits at a time from histograms of the totals that share the bits above; then the rows above it and, from the lowest on, as many
// equal to it as there is room for - each warp counts a stretch of rows, and writes it behind the stretches before it.
// The ranks are held in shared memory where they fit (48 K rows), else made again in each of the five passes.
__global__ void __launch_bounds__(ST) evict_pick(const EvictArgs A) {
    extern __shared__ uint32_t held[];
    __shared__ int hist[BINS];
    __shared__ int sums[2][SW];
    __shared__ int s_bin, s_left;
    pdl_wait();
    pdl_launch_dependents();
    const int g = blockIdx.x, a = blockIdx.y, n = *A.n0p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool bad = n < 0 || n > A.cap;
    if (threadIdx.x == 0 && g == 0 && a == 0) {
        *A.n_seen = bad ? -1 : n;
        if (bad) b2_fail(B2_ERR_DOMAIN);
    }
    if (bad) return;
    const size_t head = (size_t)a * A.Hk + g;
    const uint32_t* tot = reinterpret_cast<const uint32_t*>(A.totals) + head * A.cap;
    uint32_t* tot_d = reinterpret_cast<uint32_t*>(A.totals_d) + head * A.cap_d;
    int* idx = A.idx + head * A.keep;
    const int want = A.keep - A.recent, from = n - A.recent;  // rows to be found, among rows 0 .. from - 1
    if (n <= A.keep) {
        for (int i = threadIdx.x; i < A.keep; i += ST) {
            idx[i] = i < n ? i : -1;
            if (i < n && !A.in_place) tot_d[i] = tot[i];
        }
        return;
    }
    if (A.held) {
#pragma unroll 8
        for (int j = threadIdx.x; j < from; j += ST) held[j] = rank_of(tot[j]);
        __syncthreads();
    }
    auto rank = [&](int j) { return A.held ? held[j] : rank_of(__ldcg(tot + j)); };
    if (want > 0) {
        uint32_t prefix = 0, mask = 0;
        int left = want;  // rows still to be found among those that share `prefix`
#pragma unroll 1
        for (int step = 0; step < 3; ++step) {
            const int shift = step == 0 ? 21 : step == 1 ? 10 : 0;
            const uint32_t field = step == 2 ? 1023u : 2047u;
            for (int i = threadIdx.x; i < BINS; i += ST) hist[i] = 0;
            __syncthreads();
#pragma unroll 4
            for (int j = threadIdx.x; j < from; j += ST) {
                const uint32_t k = rank(j);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & field], 1);
            }
            __syncthreads();
            // thread i: bins 2047 - 2 i and the one below; how many rows lie in them and above
            const int hi = hist[BINS - 1 - 2 * threadIdx.x], lo = hist[BINS - 2 - 2 * threadIdx.x];
            int v = hi + lo;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (lane == 31) sums[0][warp] = v;
            __syncthreads();
            int before = warp > 0 && lane < warp ? sums[0][lane] : 0;
            before = __reduce_add_sync(0xffffffffu, before) + v - hi - lo;
            if (before < left && left <= before + hi) s_bin = BINS - 1 - 2 * threadIdx.x, s_left = left - before;
            else if (before + hi < left && left <= before + hi + lo) s_bin = BINS - 2 - 2 * threadIdx.x, s_left = left - before - hi;
            __syncthreads();
            prefix |= (uint32_t)s_bin << shift, mask |= field << shift;
            left = s_left;
        }
        // each warp's stretch: rows above the last kept rank, rows equal to it
        const int per = ((from + SW - 1) / SW + 31) & ~31, j_lo = min(warp * per, from), j_hi = min(j_lo + per, from);
        int above = 0, equal = 0;
#pragma unroll 4
        for (int j0 = j_lo; j0 < j_hi; j0 += 32) {
            const uint32_t k = j0 + lane < j_hi ? rank(j0 + lane) : 0u;
            above += __popc(__ballot_sync(0xffffffffu, j0 + lane < j_hi && k > prefix));
            equal += __popc(__ballot_sync(0xffffffffu, j0 + lane < j_hi && k == prefix));
        }
        __syncthreads();
        if (lane == 0) sums[0][warp] = above, sums[1][warp] = equal;
        __syncthreads();
        int ties = __reduce_add_sync(0xffffffffu, lane < warp ? sums[1][lane] : 0);  // equal rows before the stretch
        int at = __reduce_add_sync(0xffffffffu, lane < warp ? sums[0][lane] : 0) + min(ties, left);
#pragma unroll 4
        for (int j0 = j_lo; j0 < j_hi; j0 += 32) {
            const int j = j0 + lane;
            const uint32_t k = j < j_hi ? rank(j) : 0u;
            const unsigned eq = __ballot_sync(0xffffffffu, j < j_hi && k == prefix), below = (1u << lane) - 1u;
            const bool in = j < j_hi && (k > prefix || (k == prefix && ties + __popc(eq & below) < left));
            const unsigned kept = __ballot_sync(0xffffffffu, in);
            if (in) idx[at + __popc(kept & below)] = j;
            at += __popc(kept), ties += __popc(eq);
        }
    }
    for (int i = want + threadIdx.x; i < A.keep; i += ST) idx[i] = n - A.keep + i;
    __syncthreads();
    // the totals, down in order: a run is read whole before it is written (in place no later run reads what it writes)
    for (int i0 = 0; i0 < A.keep; i0 += ST) {
        const int i = i0 + threadIdx.x;
        const uint32_t v = i < A.keep ? __ldcg(tot + idx[i]) : 0u;
        __syncthreads();
        if (i < A.keep) tot_d[i] = v;
    }
}

constexpr int MT = 256;  // threads of a moving block
constexpr int MC = 4;    // 16-byte pieces a thread holds of a run of rows

// The kept rows of one (layer, kv head) of K or V in order, a run of rows at a time: the next run's pieces are asked for, then
// this run is written, in place behind a barrier that every thread's reads of it come before. In place a row's destination is
// never past its source, so a run that is written hits no row of a later run. More blocks share the work where heads and layers are few: in place
// each takes a slice of every row's columns, else a range of the rows.
__global__ void __launch_bounds__(MT) evict_move(const EvictArgs A) {
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.x, a = blockIdx.y, kv = blockIdx.z & 1, part = blockIdx.z >> 1;
    const int kept = min(*A.n_seen, A.keep);
    if (kept < 0) return;  // refused
    if (g == 0 && a == 0 && blockIdx.z == 0 && threadIdx.x == 0) *A.n_out = kept;
    const int slices = A.in_place ? A.parts : 1, per = A.D / 8 / slices;  // pieces of a row's slice
    const int span = A.in_place ? kept : (kept + A.parts - 1) / A.parts;
    const int lo = A.in_place ? 0 : part * span, hi = min(kept, lo + span);
    const int row = threadIdx.x / per, col = threadIdx.x - row * per, rows = MT / per;  // rows of a pass over the block's threads
    const bool on = row < rows;
    const int* idx = A.idx + ((size_t)a * A.Hk + g) * A.keep;
    const size_t cols = (size_t)(A.in_place ? part * per : 0) + col;
    const uint4* src = reinterpret_cast<const uint4*>((kv == 0 ? A.K : A.V) + (size_t)a * A.ls + (size_t)g * A.hs) + cols;
    uint4* dst = reinterpret_cast<uint4*>((kv == 0 ? A.Kd : A.Vd) + (size_t)a * A.ld + (size_t)g * A.hs) + cols;
    const size_t rs = (size_t)(A.rs / 8);
    const int run = rows * MC;
    auto from = [&](int i) {  // the cache row of kept row i, -1 past the end or outside the cache
        if (!on || i >= hi) return -1;
        int r = idx[i];
        if (A.tbl != nullptr) r = A.tbl[r];
        if (r >= 0 && r < A.cap) return r;
        b2_fail(B2_ERR_DOMAIN);
        return -1;
    };
    int ahead[MC];
    uint4 next[MC];
    unsigned has = 0;  // bit c: piece c of the next run has a source (a row past the end or outside the cache has none, and is not written)
#pragma unroll
    for (int c = 0; c < MC; ++c) ahead[c] = from(lo + c * rows + row);
#pragma unroll
    for (int c = 0; c < MC; ++c) {
        next[c] = ahead[c] >= 0 ? src[ahead[c] * rs] : make_uint4(0u, 0u, 0u, 0u);
        has |= (unsigned)(ahead[c] >= 0) << c;
    }
#pragma unroll
    for (int c = 0; c < MC; ++c) ahead[c] = from(lo + run + c * rows + row);
#pragma unroll 1
    for (int i0 = lo; i0 < hi; i0 += run) {
        uint4 v[MC];
        const unsigned here = has;
        has = 0;
#pragma unroll
        for (int c = 0; c < MC; ++c) v[c] = next[c];
#pragma unroll
        for (int c = 0; c < MC; ++c) {
            next[c] = ahead[c] >= 0 ? src[ahead[c] * rs] : make_uint4(0u, 0u, 0u, 0u);
            has |= (unsigned)(ahead[c] >= 0) << c;
        }
#pragma unroll
        for (int c = 0; c < MC; ++c) ahead[c] = from(i0 + 2 * run + c * rows + row);
        if (A.in_place) __syncthreads();  // orders every thread's reads of this run before any write of it
#pragma unroll
        for (int c = 0; c < MC; ++c) {
            const int i = i0 + c * rows + row;
            if (!(here >> c & 1u)) continue;
            const int r = A.tbl_d != nullptr ? A.tbl_d[i] : i;
            if (r < 0 || r >= A.cap_d) b2_fail(B2_ERR_DOMAIN);
            else dst[r * rs] = v[c];
        }
    }
}

// a launch that may start while the one before it drains (bit 3 of the `pdl` tunable)
constexpr int KIND = 8;

}  // namespace

extern "C" size_t btb_b200_kv_evict_workspace_bytes(int layers, int Hk, int cap) {
    return layers > 0 && Hk > 0 && cap > 0 ? 16 : 0;
}

extern "C" int btb_b200_kv_evict(const void* K, const void* V, const void* totals, const void* n0p, void* Kd, void* Vd,
                                 void* totals_d, void* n_out, void* idx, int layers, long long ls, long long ld, int Hk, int D,
                                 long long hs, long long rs, int cap, int cap_d, int keep, int recent, const void* tbl,
                                 const void* tbl_d, void* workspace, void* stream) {
    if (!K || !V || !totals || !n0p || !Kd || !Vd || !totals_d || !n_out || !idx || !workspace) return B2_ERR_NULL;
    if (layers <= 0 || layers > 65535 || Hk <= 0 || D <= 0 || D > 8 * MT || (D & 7) || cap <= 0 || cap_d <= 0 || keep <= 0 ||
        keep > cap_d || recent < 0 || recent > keep || hs < D || rs < D || (hs & 7) || (rs & 7) || (ls & 7) || (ld & 7))
        return B2_ERR_DOMAIN;
    if ((reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) | reinterpret_cast<uintptr_t>(Kd) |
         reinterpret_cast<uintptr_t>(Vd) | reinterpret_cast<uintptr_t>(workspace)) & 15)
        return B2_ERR_DOMAIN;
    // the same cache in place: every part of it, laid out alike and read and written through one map
    const bool in_k = K == Kd, in_v = V == Vd, in_t = totals == totals_d;
    if (in_k != in_v || in_k != in_t || (in_k && (ls != ld || cap != cap_d || tbl != tbl_d))) return B2_ERR_DOMAIN;
    EvictArgs a{static_cast<const bf16*>(K), static_cast<const bf16*>(V), static_cast<const float*>(totals),
                static_cast<const int*>(n0p), static_cast<bf16*>(Kd), static_cast<bf16*>(Vd), static_cast<float*>(totals_d),
                static_cast<int*>(n_out), static_cast<int*>(idx), static_cast<const int*>(tbl), static_cast<const int*>(tbl_d),
                static_cast<int*>(workspace), ls, ld, hs, rs, layers, Hk, D, cap, cap_d, keep, recent, 0, 1, in_k};
    a.held = cap <= 48 * 1024;
    // in place a block for every SM, by slices of at least 64 bytes of the rows (whole rows are faster once there are enough:
    // 36 layers of 4096 rows cut to 2048 take 122 us whole, 152 in halves, 232 in quarters); else ranges of at least
    // two runs of rows
    const long long heads = 2LL * layers * Hk, fill = 8LL * b2_sm_count();
    if (a.in_place) {
        while (a.parts < 4 && heads * a.parts < fill / 8 && D % (a.parts * 2 * 32) == 0) a.parts *= 2;
    } else {
        const int run = MT / (D / 8) * MC;
        while (a.parts < 256 && heads * a.parts < fill && (long long)a.parts * 4 * run <= keep) a.parts *= 2;
    }
    static bool allowed[64];
    if (const int rc = b2_allow_smem(reinterpret_cast<const void*>(evict_pick), allowed)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (const int rc = b2_launch(reinterpret_cast<const void*>(evict_pick), dim3(Hk, layers), dim3(ST), a.held ? (size_t)cap * 4 : 0, s, a, KIND))
        return rc;
    return b2_launch(reinterpret_cast<const void*>(evict_move), dim3(Hk, layers, 2 * a.parts), dim3(MT), 0, s, a, KIND);
}
