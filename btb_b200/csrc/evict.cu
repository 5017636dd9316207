// Eviction from a cache by accumulated attention weight, for sm_100a: per (layer, kv head) the `recent` last rows stay,
// and of the others the keep - recent with the largest totals, the lower row first among equals. The kept rows move
// down in order, their keys, values and totals with them, in place or into another cache.
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
};

// a total's rank as an unsigned word: larger totals rank higher, -0 as 0, every NaN above all else
__device__ __forceinline__ uint32_t rank_of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

constexpr int ST = 1024;  // threads of a selection block

// inclusive sums over a block's threads; every thread gets its own and the block's
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    total = warp_sums[31];
    const int before = warp > 0 ? warp_sums[warp - 1] : 0;
    __syncthreads();
    return v + before;
}

// the kept rows of one (layer, kv head): the rank of the last kept total found a byte at a time from histograms, then one
// ordered pass that writes the rows above it and as many equal to it, from the lowest on, as there is room for
__global__ void __launch_bounds__(ST) evict_pick(const EvictArgs A) {
    __shared__ unsigned hist[256];
    __shared__ int warp_sums[32];
    __shared__ unsigned s_digit;
    __shared__ int s_left;
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.x, a = blockIdx.y, n = *A.n0p;
    const bool bad = n < 0 || n > A.cap;
    if (threadIdx.x == 0 && g == 0 && a == 0) {
        *A.n_seen = bad ? 0 : n;
        if (bad) b2_fail(B2_ERR_DOMAIN);
    }
    if (bad) return;
    const float* tot = A.totals + ((size_t)a * A.Hk + g) * A.cap;
    int* idx = A.idx + ((size_t)a * A.Hk + g) * A.keep;
    for (int i = threadIdx.x; i < A.keep; i += ST) {
        if (n <= A.keep) idx[i] = i < n ? i : -1;
        else if (i >= A.keep - A.recent) idx[i] = n - A.keep + i;
    }
    const int want = A.keep - A.recent, from = n - A.recent;
    if (n <= A.keep || want == 0) return;
    unsigned prefix = 0, mask = 0;
    int left = want;  // rows still to be found among those that share `prefix`
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += ST) hist[i] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < from; j += ST) {
            const uint32_t k = rank_of(tot[j]);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = 255, l = left;
            while (d > 0 && (int)hist[d] < l) l -= hist[d--];
            s_digit = d, s_left = l;
        }
        __syncthreads();
        prefix |= s_digit << shift, mask |= 255u << shift;
        left = s_left;
        __syncthreads();
    }
    int done = 0, ties = 0;  // rows written, rows equal to the last kept total seen
    for (int j0 = 0; j0 < from; j0 += ST) {
        const int j = j0 + threadIdx.x;
        const uint32_t k = j < from ? rank_of(tot[j]) : 0u;
        const bool tie = j < from && k == prefix;
        int n_tie, n_kept;
        const int tie_at = block_scan(tie, warp_sums, n_tie);
        const bool in = j < from && (k > prefix || (tie && ties + tie_at <= left));
        const int at = block_scan(in, warp_sums, n_kept);
        if (in) idx[done + at - 1] = j;
        done += n_kept, ties += n_tie;
    }
}

constexpr int MT = 256;  // threads of a moving block
constexpr int MC = 8;    // 16-byte pieces a thread holds

// The kept rows of one (layer, kv head) of K (z = 0) or V (z = 1) moved in order. In place a row's destination is never
// past its source, so a block that walks the rows in order, reads a run of them whole and writes it before it reads
// the next never writes a row that it has still to read.
__global__ void __launch_bounds__(MT) evict_move(const EvictArgs A) {
    pdl_launch_dependents();
    pdl_wait();
    const int g = blockIdx.x, a = blockIdx.y, n = *A.n_seen;
    const int kept = min(n, A.keep), per = A.D / 8;  // pieces of a row
    const size_t at = (size_t)a * A.Hk + g;
    const int* idx = A.idx + at * A.keep;
    if (blockIdx.z == 2) {  // the totals
        const float* src = A.totals + at * A.cap;
        float* dst = A.totals_d + at * A.cap_d;
        for (int j0 = 0; j0 < kept; j0 += MT) {
            const int j = j0 + threadIdx.x;
            const float v = j < kept ? src[idx[j]] : 0.f;
            __syncthreads();
            if (j < kept) dst[j] = v;
            __syncthreads();
        }
        if (g == 0 && a == 0 && threadIdx.x == 0) *A.n_out = kept;
        return;
    }
    const bf16* src = (blockIdx.z == 0 ? A.K : A.V) + (size_t)a * A.ls + (size_t)g * A.hs;
    bf16* dst = (blockIdx.z == 0 ? A.Kd : A.Vd) + (size_t)a * A.ld + (size_t)g * A.hs;
    const long long pieces = (long long)kept * per;
    for (long long p0 = 0; p0 < pieces; p0 += MT * MC) {
        uint4 v[MC];
#pragma unroll
        for (int c = 0; c < MC; ++c) {
            const long long p = p0 + c * MT + threadIdx.x;
            if (p >= pieces) continue;
            int r = idx[p / per];
            if (A.tbl != nullptr) r = A.tbl[r];
            if (r < 0 || r >= A.cap) {
                b2_fail(B2_ERR_DOMAIN);
                r = -1;
            }
            v[c] = r >= 0 ? reinterpret_cast<const uint4*>(src + (size_t)r * A.rs)[p % per] : make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < MC; ++c) {
            const long long p = p0 + c * MT + threadIdx.x;
            if (p >= pieces) continue;
            int r = (int)(p / per);
            if (A.tbl_d != nullptr) r = A.tbl_d[r];
            if (r < 0 || r >= A.cap_d) b2_fail(B2_ERR_DOMAIN);
            else reinterpret_cast<uint4*>(dst + (size_t)r * A.rs)[p % per] = v[c];
        }
        __syncthreads();
    }
}

}  // namespace

extern "C" size_t btb_b200_kv_evict_workspace_bytes(int layers, int Hk, int cap) {
    return layers > 0 && Hk > 0 && cap > 0 ? 16 : 0;
}

extern "C" int btb_b200_kv_evict(const void* K, const void* V, const void* totals, const void* n0p, void* Kd, void* Vd,
                                 void* totals_d, void* n_out, void* idx, int layers, long long ls, long long ld, int Hk, int D,
                                 long long hs, long long rs, int cap, int cap_d, int keep, int recent, const void* tbl,
                                 const void* tbl_d, void* workspace, void* stream) {
    if (!K || !V || !totals || !n0p || !Kd || !Vd || !totals_d || !n_out || !idx || !workspace) return B2_ERR_NULL;
    if (layers <= 0 || layers > 65535 || Hk <= 0 || D <= 0 || (D & 7) || cap <= 0 || cap_d <= 0 || keep <= 0 || keep > cap_d ||
        recent < 0 || recent > keep || hs < D || rs < D || (hs & 7) || (rs & 7) || (ls & 7) || (ld & 7))
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
                static_cast<int*>(workspace), ls, ld, hs, rs, layers, Hk, D, cap, cap_d, keep, recent};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (const int rc = b2_launch(reinterpret_cast<const void*>(evict_pick), dim3(Hk, layers), dim3(ST), 0, s, a)) return rc;
    return b2_launch(reinterpret_cast<const void*>(evict_move), dim3(Hk, layers, 3), dim3(MT), 0, s, a);
}
