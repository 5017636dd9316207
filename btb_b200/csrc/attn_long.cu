// Attention over long caches for sm_100a. Two entry points: btb_b200_attn_shared, a pass in the rows layout whose rows
// share prefixes, and btb_b200_attn_scored, a chain or tree pass that also adds up what each cache row is given.
//
// For a row's query head q over its keys j: s_j = scale q . k_j, out = sum_j e^(s_j) v_j / (sum_j e^(s_j) + e^sink), in one pass
// over the keys with a running maximum m and sum l of 2^(s_j log2 e - m) in f32; the weights are rounded to bf16 once, for
// their product with the values, the sums are of the unrounded ones. A state (m, l, sum of w_j v_j) of any set of keys joins
// another's by scaling both to the larger maximum, so the keys are cut wherever it suits the card. The totals need the
// denominators first: w_j = 2^(s_j log2 e - m - log2 l) is made after the join, from kept scores or from the scores again.
//
// Launches: long_tiles (the shared prefixes on the tensor cores, the rows' own keys beside them), long_join (the states of a row
// folded; for passes of few rows also the totals), long_weights (the totals of passes of more rows). Bound, at the largest
// shapes, by the cache's bytes and what surrounds them: one row of 64 heads over 32768 rows of 8 kv heads (134 MB) takes 38 us a
// call, 0.55 of the measured copy rate; by stamps in the kernels its CTAs end their tiles 25 to 33 us after they began, half of
// them by 31, and all wait for the last. 32 rows over it with 128 steps of their own take 47.7 us, the CTAs' tiles 32 to 43,
// half by 39.5, the states of 256 queries a CTA (19 MB) written and folded most of the rest - in a burst at 1965 MHz; run on, the
// power cap holds the clock near 1675 MHz and a call takes 55, its time following the clock. Short passes (9 to 18 us) are two
// or three launches' latencies. btb_b200_attn_decode_rows takes 98 us and 1981 for those rows (63 steps of their own); it is
// the faster one below a few hundred keys (eight rows of 8 heads over 8 kv heads, 128 keys: 6.1 us against 10.5).
#include <cuda.h>

#include <atomic>

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
    float* scores;       // [Hq, T, score_n] the scores of all keys in log2 units (passes of few rows), or null
    int4* info;          // [T] two words a row: where its states lie
    float2* part_ml;     // a part's rows, then the units': maximum and sum ...
    float* part_o;       // ... and output [., D], not yet divided
    long long unit_row;  // the units' first row: unit u of kv head g at unit_row + (g * units + u) * G
    long long score_n;
    float scale;
    int T, Hq, Hk, win, cap, ctas;
    int own_share;  // warps that take a kv head's units, about
    long long hs, rs, ts;
};

// ---- the pass's work, from what stands on the card ------------------------------------------------------------------
// The prefixes: per kv head an item for each prefix that rows share, its queries all of those rows', its keys cut into
// tiles of 64. The tiles of all heads lie in one line, with a gap of GAP tiles' worth of time behind each item (what it costs
// a CTA to end one and begin the next), which is cut evenly over the CTAs; a CTA's stretch of an item is a part, whose state
// (maximum, sum, output row) the joining kernel folds with the others'. Part (CTA c, item i) keeps its rows at
// c * T G + the rows of all items before i, which no two parts share.
// A row's own keys (its steps in the rows layout, its path in a chain or tree pass) are no one else's: units of up to
// `chunk` keys of one (row, kv head), a warp each, beside the tiles. A one-row pass's own key joins its prefix.
constexpr int KT = 64;         // keys a tile
constexpr int GAP = 8;         // tiles (4: 52.6 us where 8 takes 49.1, for 32 rows over 32768; shorter ones within 3 %)
constexpr int CTAS_MAX = 160;  // CTAs of the tile kernel at most
constexpr int OWN_WARPS = 2;   // warps of a CTA that take units (two more would leave all of them 128 registers)

struct Plan {
    int mask[32];                             // item of lane l's prefix: its rows (0: no item)
    int p_start[32], p_count[32];             // ... its first key (cache row, or logical row of a chain or tree pass) and keys
    int p_tiles[32], p_at[32], p_row0[32];    // ... tiles, its first one's place in a kv head's line, partial rows before it
    int order[32];                            // ... its rows, from p_row0 / G on
    int lead[32];                             // row t's prefix item, -1: padding or refused
    int own[32], own_n[32], unit0[32];        // its own keys: the first's cache row (rows layout), how many; units before it
    int W, line, rows, units, chunk, n0;      // ... and a kv head's length of line, partial rows and units
};

__device__ __forceinline__ int warp_excl(int v, int lane, int& total) {
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
    }
    total = __shfl_sync(0xffffffffu, x, 31);
    return x - v;
}

// units of a (row, kv head) at most: enough for every warp where rows and heads are few
__host__ __device__ __forceinline__ int units_max(int T, int Hk) { return max(16, min(64, 1024 / (T * Hk))); }

// one warp fills `P`; `tell`: this block records a refused layout
template <int G>
__device__ __forceinline__ void make_plan(const LongArgs& A, Plan& P, bool tell) {
    const int t = threadIdx.x & 31;
    int mask = 0, start = 0, count = 0, lead = -1, own = 0, own_n = 0, W = 0, n0 = 0;
    if (A.rw == nullptr) {
        n0 = *A.n0p;
        const int par = t < A.T ? A.par[t] : -1;
        if (n0 < 0 || n0 > A.cap - A.T) {
            if (tell && t == 0) b2_fail(B2_ERR_DOMAIN);
        } else {
            lead = t < A.T ? 0 : -1;
            if (t == 0) mask = A.T == 32 ? -1 : (1 << A.T) - 1, count = n0 + (A.T == 1);
            if (A.T > 1) {  // the row's path as a set of the pass's rows
                unsigned path = 0;
                int q = t < A.T ? t : -1;
                for (int k = 0; k < A.T; ++k) {
                    const bool on = q >= 0 && q < A.T;
                    if (on) path |= 1u << q;
                    const int up = __shfl_sync(0xffffffffu, par, on ? q : 0);
                    q = on ? up : -1;
                }
                own = (int)path, own_n = t < A.T ? __popc(path) : 0;
            }
        }
    } else {
        const int base = A.rw[0], step = A.rw[1];
        W = A.rw[2];
        bool live = t < A.T;
        const int col = live ? A.rw[3 + 3 * t] : 0, off = live ? A.rw[4 + 3 * t] : 0, len = live ? A.rw[5 + 3 * t] : -1;
        live = live && len >= 0;
        if (live) {
            const long long lo = (long long)base + col, hi = lo + (long long)step * W;
            if (step < 0 || W < 0 || off < 0 || len > A.cap || off > A.cap - len || lo < 0 || hi >= A.cap || step > A.cap) {
                if (tell) b2_fail(B2_ERR_DOMAIN);
                live = false;
            }
        }
        const int first = A.win > 0 ? (int)max((long long)len + step + 1 - A.win, 0LL) : 0;
        const unsigned alive = __ballot_sync(0xffffffffu, live);
        const unsigned same = __match_any_sync(0xffffffffu, off) & __match_any_sync(0xffffffffu, len) & alive;
        if (live) {
            lead = __ffs(same) - 1;
            if (lead == t) mask = same, start = off + first, count = max(0, len - first);
            const int i0 = max(0, first - len);
            own = base + i0 * W + col, own_n = step + 1 - i0;
        }
    }
    const int p_tiles = mask ? (count + KT - 1) / KT : 0;
    int line, pr, units;
    const int p_at = warp_excl(p_tiles ? p_tiles + GAP : 0, t, line), p_row0 = warp_excl(p_tiles ? __popc(mask) * G : 0, t, pr);
    // units of about a warp's fair share of the own keys, a multiple of 32, no row in more of them than its room allows
    const int keys = __reduce_add_sync(0xffffffffu, min(own_n, 1 << 20));
    const int most = __reduce_max_sync(0xffffffffu, own_n), room = units_max(A.T, A.Hk);
    const int chunk = (max((keys + A.own_share - 1) / A.own_share, (most + room - 1) / room) + 31) & ~31;
    const int unit0 = warp_excl(own_n > 0 ? (own_n + chunk - 1) / chunk : 0, t, units);
    P.mask[t] = mask, P.p_start[t] = start, P.p_count[t] = count, P.p_tiles[t] = p_tiles, P.p_at[t] = p_at, P.p_row0[t] = p_row0;
    P.lead[t] = lead, P.own[t] = own, P.own_n[t] = own_n, P.unit0[t] = unit0;
    const int src = lead < 0 ? 0 : lead;
    const int its = __shfl_sync(0xffffffffu, mask, src), before = __shfl_sync(0xffffffffu, p_row0, src);
    const int some = __shfl_sync(0xffffffffu, p_tiles, src);
    const int below = __popc(its & ((1u << t) - 1u));  // the row's place among its prefix's
    if (lead >= 0 && some > 0) P.order[before / G + below] = t;
    if (t == 0) P.W = W, P.line = line, P.rows = pr, P.units = units, P.chunk = chunk, P.n0 = n0;
    __syncwarp();
}
// one warp writes for the joining kernel where each row's states lie (none: padding, or refused)
template <int G>
__device__ __forceinline__ void tell_plan(const LongArgs& A, const Plan& P) {
    const int t = threadIdx.x & 31, lead = P.lead[t], l = max(lead, 0);
    if (t >= A.T) return;
    const int below = __popc(P.mask[l] & ((1u << t) - 1u));  // the row's place among its prefix's
    const int units = P.own_n[t] > 0 ? (P.own_n[t] + P.chunk - 1) / P.chunk : 0;
    A.info[2 * t] = make_int4(P.p_at[l], lead < 0 ? 0 : P.p_tiles[l], P.p_row0[l] + below * G, units);
    A.info[2 * t + 1] = make_int4(P.unit0[t], P.line, P.rows, P.units);
}

// the even cut of the heads' line over the CTAs; no more of them than it is long, so that no stretch between two others is
// empty
struct Cut {
    int per, more;  // the first `more` CTAs' stretches are per + 1 long
    __device__ __forceinline__ Cut(int line, int ctas) : per(line / ctas), more(line - line / ctas * ctas) {}
    __device__ __forceinline__ int first(int c) const { return c * per + min(c, more); }
    __device__ __forceinline__ int cta_of(int place) const {
        const int big = more * (per + 1);
        return place < big ? place / (per + 1) : more + (place - big) / per;
    }
};

// a CTA's stretch of one item
struct Part {
    int head, start, keys, tiles, rows, order;  // `keys`: of these tiles (the last may be partly filled)
    int end;                                    // the place behind it
    long long row0;                             // its first partial row
};
// the first part at or behind place `at` of a CTA whose stretch ends at `stop`; tiles 0: none (a warp's lanes ask alike)
template <int G>
__device__ __noinline__ Part part_at(const Plan& P, int span, int at, int stop, int cta) {
    const int lane = threadIdx.x & 31;
    Part p;
    p.head = at / P.line;
    int in = at - p.head * P.line;
    const int first = P.p_at[lane], tiles = P.p_tiles[lane];
    const unsigned here = __ballot_sync(0xffffffffu, tiles > 0 && first + tiles > in);  // items not yet behind
    if (here == 0) ++p.head, in = 0;                                                     // (in the head's last gap)
    const unsigned any = here != 0 ? here : __ballot_sync(0xffffffffu, tiles > 0);
    const int l = __ffs(any) - 1, skip = max(in - P.p_at[l], 0), place = p.head * P.line + P.p_at[l] + skip;
    p.tiles = max(min(P.p_tiles[l] - skip, stop - place), 0);
    p.start = P.p_start[l] + skip * KT;
    p.keys = min(p.tiles * KT, P.p_count[l] - skip * KT);
    p.rows = __popc(P.mask[l]) * G;
    p.order = P.p_row0[l] / G;
    p.row0 = (long long)cta * span + (long long)p.head * P.rows + P.p_row0[l];
    p.end = place + p.tiles;
    return p;
}

// ---- the tiles on the tensor cores -------------------------------------------------------------------------------------
// S = Q K^T and O += P V with tcgen05.mma: up to 128 of an item's query rows (row-of-the-pass major, then the kv head's query
// heads) are the MMA's M, so a shared key is read once for all of them. Two warpgroups turn scores into weights, a thread a
// query row, on alternate key tiles with an output accumulator each (items of up to 128 rows; the two are folded at the
// part's end) or on the two halves of an item's up to 256 rows. Tensor memory, 512 columns: two score tiles of 64 columns a
// warpgroup, so that the next one is there when a warpgroup comes from the last, then the two outputs; weights (bf16) lie over
// their scores.
// the low word of a shared-memory operand's descriptor: where it begins and, for the values, the step to their next 64 dims
__device__ __forceinline__ uint32_t desc_sw128(uint32_t saddr, uint32_t lbo) { return ((saddr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16); }
// (a descriptor's upper word is the same for every operand here: 1024 bytes between 8-row groups, version 1, 128-byte swizzle)
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
// The MMAs are issued by one elected lane (`lead` nonzero in it) of a warp whose lanes all walk the same code: the operands
// then are warp-uniform values, which the instruction wants (by one lane in a branch of its own the longest pass took 67 us
// against 58).
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t on;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(on));
    return on;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 da, db;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\nmov.b64 da, {%1, %6};\nmov.b64 db, {%2, %6};\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "n"(DESC_HI)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 db;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\nmov.b64 db, {%2, %6};\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(lead), "n"(DESC_HI)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t lead, uint32_t bar) {
    asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// two f32 side by side: one instruction for both
__device__ __forceinline__ uint64_t pair2(float x, float y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void split2(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
        "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// the loads so far have arrived; the registers pass through, so that nothing reads them before
__device__ __forceinline__ void tm_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
          "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
          "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
          "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
        :
        : "memory");
}
__device__ __forceinline__ void tm_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
          "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
        :
        : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(tm), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// four rows of 64 columns, wherever they lie
__device__ __forceinline__ void tma_rows4(uint32_t dst, const CUtensorMap* tm, int x, const int* y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
        "[%7];" ::"r"(dst),
        "l"(tm), "r"(x), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(bar)
        : "memory");
}

constexpr int TW = 10 + OWN_WARPS;  // warps: two warpgroups for the weights, the loads' warp, the MMAs' warp, the units' warps
constexpr int STAGES_MAX = 12;      // stages of a ring

struct alignas(8) TileSync {
    uint64_t kfull[STAGES_MAX], kempty[STAGES_MAX], vfull[STAGES_MAX], vempty[STAGES_MAX];
    uint64_t sfull[2][2];   // a warpgroup's scores are there, a buffer each
    uint64_t pready[2][2];  // ... its weights are
    uint64_t pv[2][2];      // ... their product with the values is added
    uint64_t qfull;         // the part's queries are in shared memory
    uint64_t stats;         // the second warpgroup's maxima and sums are in shared memory
    uint64_t next;          // both warpgroups are through with the part
    uint64_t drain;         // every MMA has run
    uint32_t tmem;
    int fail;
};

struct TileArgs {
    LongArgs a;
    int row_mul, col_mul;  // a kv head's rows begin at head * row_mul, its columns at head * col_mul
    int stages;            // of either ring
};

// a warp's bounded wait that also ends once any other role has given up; its lanes get one answer
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, TileSync& sy) {
    for (uint32_t it = 0; it < B2_WAIT_LIMIT; ++it) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *(volatile int*)&sy.fail)) return false;
    }
    *(volatile int*)&sy.fail = 1;
    return false;
}
__device__ __forceinline__ bool wait_or_fail(uint64_t* bar, uint32_t parity, TileSync& sy) {
    const uint32_t b = smem_u32(bar);
    return __all_sync(0xffffffffu, mbar_try_wait(b, parity)) || wait_long(b, parity, sy);
}

// the place of the n-th (from 0) set bit
__device__ __forceinline__ int bit_place(unsigned set, int n) {
    int at = 0;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1)
        if (__popc(set & ((1u << (at + s)) - 1u)) <= n) at += s;
    return at;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t v) {  // an 8 x 8 matrix of 16-bit values, two of a row a lane, transposed
    uint32_t w;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(w) : "r"(v));
    return w;
}

// a warp's units: every `stride`-th from `first` on, 32 keys at a time with a running maximum and sum. So few queries (a kv
// head's of one row) on keys nobody shares want few instructions and early loads, not tiles: the products are warp MMAs
// straight from registers. S (16 keys x 8 heads) takes 16 bytes of a key's row a lane: the lane's eight dims stand for the
// products' k in an order of our own, the same for keys and queries. O (heads x dims) takes the weights and the values each
// turned by movmatrix, 16 bytes of a value's row a lane. (As f32 chains, a lane a key, the units ended 4 us after the tiles of
// 8 rows of 256 steps over a 2048-row prefix and 20 us after those of 32 rows of 128 steps over 32768: 21 and 83 us a call
// where these took 17 and 62.) Lane 4 y + x: keys y, y + 8, ..; heads 2 x, 2 x + 1 of the
// scores; head y and dims 32 c + 8 x .. + 7 of the output. Keys outside are never read.
template <int D, int G>
__device__ __forceinline__ void own_units(const LongArgs& A, const Plan& P, int first, int stride) {
    constexpr int C = D / 32;
    const int lane = threadIdx.x & 31, x = lane & 3, y = lane >> 2;
    const float scale2 = __fmul_rn(A.scale, LOG2E);
    const long long all = (long long)P.units * A.Hk;
    for (long long u = first; u < all; u += stride) {
        const int g = (int)(u / P.units), in = (int)(u - (long long)g * P.units);
        const int t = 31 - __clz(__ballot_sync(0xffffffffu, P.own_n[lane] > 0 && P.unit0[lane] <= in));
        const int i0 = (in - P.unit0[t]) * P.chunk, n = min(P.chunk, P.own_n[t] - i0), own = P.own[t];
        const bf16* Kg = A.K + (size_t)g * A.hs + x * 8;
        const bf16* Vg = A.V + (size_t)g * A.hs + x * 8;
        float* scores = A.own != nullptr ? A.own + ((size_t)t * A.Hq + g * G) * 32 : nullptr;
        uint4 q[C];
#pragma unroll
        for (int c = 0; c < C; ++c)
            q[c] = y < G ? __ldg(reinterpret_cast<const uint4*>(A.q + ((size_t)t * A.Hq + g * G + y) * D + c * 32 + x * 8)) : make_uint4(0u, 0u, 0u, 0u);
        if (scores != nullptr) {
            for (int h = 0; h < G; ++h) scores[h * 32 + lane] = NEG_INF;
            __syncwarp();
        }
        float m[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f}, o[C][4][2];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[c][i][0] = o[c][i][1] = 0.f;
#pragma unroll 1
        for (int j0 = 0; j0 < n; j0 += 32) {
            int row[4], place[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j0 + y + 8 * k;
                row[k] = -1, place[k] = 0;
                if (j < n) {
                    if (A.rw != nullptr) {
                        row[k] = own + (i0 + j) * P.W;
                    } else {
                        place[k] = bit_place((unsigned)own, j);
                        row[k] = P.n0 + place[k];
                        if (A.tbl != nullptr) row[k] = A.tbl[row[k]];
                        if (row[k] < 0 || row[k] >= A.cap) {
                            b2_fail(B2_ERR_DOMAIN);
                            row[k] = -1;
                        }
                    }
                }
            }
            uint4 kv[4][C], vv[2][C];
            auto load = [&](const bf16* from, int k, int c) {
                return row[k] >= 0 ? __ldg(reinterpret_cast<const uint4*>(from + (size_t)row[k] * A.rs + c * 32)) : make_uint4(0u, 0u, 0u, 0u);
            };
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int c = 0; c < C; ++c) kv[k][c] = load(Kg, k, c);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int c = 0; c < C; ++c) vv[k][c] = load(Vg, k, c);
            float s[2][4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint4 k0 = kv[2 * b][c], k1 = kv[2 * b + 1][c];
                    mma16816(s[b], k0.x, k1.x, k0.y, k1.y, q[c].x, q[c].y);
                    mma16816(s[b], k0.z, k1.z, k0.w, k1.w, q[c].z, q[c].w);
                }
            }
            float f[2], p[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // head 2 x + e: key y + 8 k's score in s[k / 2][2 (k % 2) + e]
                float mx = m[e];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float& v = s[k >> 1][2 * (k & 1) + e];
                    v = row[k] >= 0 ? __fmul_rn(v, scale2) : NEG_INF;
                    mx = fmaxf(mx, v);
                    if (scores != nullptr && 2 * x + e < G && row[k] >= 0) scores[(2 * x + e) * 32 + place[k]] = v;
                }
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
                const float sub = mx == NEG_INF ? 0.f : mx;
                f[e] = m[e] == NEG_INF ? 0.f : ex2(m[e] - sub);
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float w = ex2(s[k >> 1][2 * (k & 1) + e] - sub);
                    p[k >> 1][2 * (k & 1) + e] = w, sum += w;
                }
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                l[e] = l[e] * f[e] + sum;
                m[e] = mx;
            }
            const float f0 = __shfl_sync(0xffffffffu, f[0], y >> 1), f1 = __shfl_sync(0xffffffffu, f[1], y >> 1), fy = y & 1 ? f1 : f0;  // head y's
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][i][0] *= fy, o[c][i][1] *= fy;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t w0, w1;
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w0) : "f"(p[b][1]), "f"(p[b][0]));
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w1) : "f"(p[b][3]), "f"(p[b][2]));
                const uint32_t a0 = turned(w0), a2 = turned(w1);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint32_t u0[4] = {vv[0][c].x, vv[0][c].y, vv[0][c].z, vv[0][c].w}, u1[4] = {vv[1][c].x, vv[1][c].y, vv[1][c].z, vv[1][c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float d[4] = {o[c][i][0], o[c][i][1], 0.f, 0.f};
                        mma16816(d, a0, 0u, a2, 0u, turned(u0[i]), turned(u1[i]));
                        o[c][i][0] = d[0], o[c][i][1] = d[1];
                    }
                }
                if (b == 0) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int c = 0; c < C; ++c) vv[k][c] = load(Vg, k + 2, c);
                }
            }
        }
        const size_t at = (size_t)(A.unit_row + u * G);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (y == 0 && 2 * x + e < G) A.part_ml[at + 2 * x + e] = make_float2(m[e], l[e]);
        if (y < G) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float4* to = reinterpret_cast<float4*>(A.part_o + (at + y) * D + c * 32 + x * 8);
                to[0] = make_float4(o[c][0][0], o[c][0][1], o[c][1][0], o[c][1][1]);
                to[1] = make_float4(o[c][2][0], o[c][2][1], o[c][3][0], o[c][3][1]);
            }
        }
    }
}

// where the issuing warp stands: the stages' descriptors and numbers, and the phases - of either ring, and of the weights'
// and the products' buffers, a bit each (2 w + b)
struct Issuer {
    uint32_t k, v;
    int ks, vs;
    uint32_t kph, vph, pph;
};

// The MMAs of one part: job j is tile j for warpgroup j & 1 (NRT 1), or its half of tile j / 2's query rows (NRT 2);
// scores run four jobs ahead of the products with the values, over the weights of the warpgroup's last tile but one.
// D f32, A and B bf16; S: both K-major, N = 64 keys; O: the values' dims are B's N and lie contiguous, N = D.
template <int D, int NRT>
__device__ __forceinline__ bool issue_part(Issuer& is, TileSync& sy, uint32_t lead, uint32_t tmem, uint32_t q0, uint32_t k0, uint32_t v0, int stages, int jobs) {
    constexpr int TILE = KT * D * 2, HALF = KT * 128, QTILE = 128 * D * 2, QHALF = 128 * 128;
    constexpr uint32_t base_desc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 4) << 24);
    constexpr uint32_t desc_s = base_desc | ((uint32_t)(KT >> 3) << 17), desc_o = base_desc | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    uint32_t k = is.k, v = is.v, kph = is.kph, vph = is.vph, pph = is.pph;
    int ks = is.ks, vs = is.vs;
#pragma unroll 1
    for (int j0 = -4; j0 < jobs; j0 += 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int w = u & 1, b = u >> 1, j = j0 + u;
            constexpr bool one = NRT == 1;
            if (j0 >= 0 && j < jobs) {  // job j's share of the output
                if ((one || w == 0) && !wait_or_fail(&sy.vfull[vs], vph, sy)) return false;
                if (!wait_or_fail(&sy.pready[w][b], (pph >> u) & 1, sy)) return false;
                pph ^= 1u << u;
                tm_after();
#pragma unroll
                for (int i = 0; i < KT / 16; ++i)
                    mma_ts(lead, tmem + 256 + w * 128, tmem + w * 128 + b * KT + i * 8, v + i * (2048 >> 4), desc_o, i > 0 || j >= 2);
                mma_commit(lead, smem_u32(&sy.pv[w][b]));
                if (one || w == 1) {
                    mma_commit(lead, smem_u32(&sy.vempty[vs]));
                    v += TILE >> 4;
                    if (++vs == stages) vs = 0, vph ^= 1, v = v0;
                }
            }
            if (j + 4 < jobs) {  // the scores of job j + 4
                if ((one || w == 0) && !wait_or_fail(&sy.kfull[ks], kph, sy)) return false;
                tm_after();
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    mma_ss(lead, tmem + w * 128 + b * KT, q0 + (uint32_t)(((one ? 0 : w * QTILE) + (i >> 2) * QHALF + (i & 3) * 32) >> 4),
                           k + (uint32_t)(((i >> 2) * HALF + (i & 3) * 32) >> 4), desc_s, i > 0);
                mma_commit(lead, smem_u32(&sy.sfull[w][b]));
                if (one || w == 1) {
                    mma_commit(lead, smem_u32(&sy.kempty[ks]));
                    k += TILE >> 4;
                    if (++ks == stages) ks = 0, kph ^= 1, k = k0;
                }
            }
        }
    }
    is.k = k, is.v = v, is.kph = kph, is.vph = vph, is.pph = pph, is.ks = ks, is.vs = vs;
    return true;
}

template <int D, int G>
__global__ void __launch_bounds__(TW * 32, 1)
    long_tiles(const __grid_constant__ CUtensorMap kbox, const __grid_constant__ CUtensorMap krows,
               const __grid_constant__ CUtensorMap vbox, const __grid_constant__ CUtensorMap vrows, const TileArgs X) {
    constexpr int TILE = KT * D * 2, QTILE = 128 * D * 2;  // bytes of a tile of keys or values, and of queries:
    constexpr int HALF = KT * 128, QHALF = 128 * 128;      // D / 64 blocks of rows of 128 bytes
    const LongArgs& A = X.a;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ TileSync sy;
    __shared__ Plan plan;
    __shared__ float s_m[128], s_l[128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nq = A.T * G > 128 ? 2 : 1;
    const uint32_t sq = smem_u32(smem), sk = sq + nq * QTILE, sv = sk + X.stages * TILE;

    if (threadIdx.x == 32) {
        for (int s = 0; s < X.stages; ++s) {
            mbar_init(smem_u32(&sy.kfull[s]), 1), mbar_init(smem_u32(&sy.kempty[s]), 1);
            mbar_init(smem_u32(&sy.vfull[s]), 1), mbar_init(smem_u32(&sy.vempty[s]), 1);
        }
        for (int w = 0; w < 2; ++w) {
            for (int b = 0; b < 2; ++b)
                mbar_init(smem_u32(&sy.sfull[w][b]), 1), mbar_init(smem_u32(&sy.pready[w][b]), 4), mbar_init(smem_u32(&sy.pv[w][b]), 1);
        }
        mbar_init(smem_u32(&sy.qfull), 8), mbar_init(smem_u32(&sy.stats), 4), mbar_init(smem_u32(&sy.next), 8);
        mbar_init(smem_u32(&sy.drain), 1);
        sy.fail = 0;
        mbar_fence_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sy.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tm_before();
    }
    // The kernels before are through; only now may the joining kernel start, which reads what they left before it waits. The warp
    // that took the tensor memory says so: no kernel that starts on it can take tensor memory ahead of this CTA, and then wait
    // for this CTA while this CTA waits for it.
    pdl_wait();
    if (warp == 9) pdl_launch_dependents();
    if (warp == 0) make_plan<G>(A, plan, blockIdx.x == 0);
    __syncthreads();
    const Cut cut(plan.line * A.Hk, gridDim.x);
    const int begin = cut.first(blockIdx.x);
    const int stop = sq & 1023 ? begin : cut.first(blockIdx.x + 1);  // (the tiles leave no room to align them here)
    tm_after();
    const uint32_t tmem = sy.tmem;

    if (warp < 8) {
        // ---- the weights: thread = query row of the tile ------------------------------------------------------------------
        const int wg = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + wg * 128, to = tmem + lanes + 256 + wg * 128;
        // a negative scale's sign is the queries', and a zero one's zero (a masked score stays -inf times what remains)
        const float size2 = fabsf(__fmul_rn(A.scale, LOG2E)), scale2 = size2 == 0.f ? 1.f : size2;
        uint32_t turn = 0;  // bit b: score buffer b's phase
        uint32_t stph = 0, nph = 0;
        bool ok = true;
        for (int at = begin; at < stop && ok;) {
            const Part p = part_at<G>(plan, A.T * G, at, stop, blockIdx.x);
            if (p.tiles == 0) break;
            at = p.end;
            const bool two = p.rows > 128;
            {   // the part's queries into shared memory as the MMA reads them: 16-byte piece c of row r at c ^ (r & 7)
                const uint32_t flip = A.scale < 0.f ? 0x80008000u : 0u;
                // eight lanes a row's 128 bytes, four rows a warp at a time (a row a lane took 5500 cycles for 256 rows: every
                // lane's piece another line)
                const int x = lane & 7, n = two ? 8 : 4;  // the warp's runs of four rows of each of the D / 64 column blocks
#pragma unroll 1
                for (int i0 = 0; i0 < n; i0 += 4) {
                    uint4 v[4][D / 64];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = (i0 + i) * 32 + warp * 4 + (lane >> 3);
                        const int t = r < p.rows ? plan.order[p.order + r / G] : 0;
                        const uint4* src = reinterpret_cast<const uint4*>(A.q + ((size_t)t * A.Hq + p.head * G + r % G) * D) + x;
#pragma unroll
                        for (int c = 0; c < D / 64; ++c) v[i][c] = r < p.rows && size2 != 0.f ? src[c * 8] : make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = (i0 + i) * 32 + warp * 4 + (lane >> 3), rr = r & 127;
#pragma unroll
                        for (int c = 0; c < D / 64; ++c) {
                            uint4 w = v[i][c];
                            w.x ^= flip, w.y ^= flip, w.z ^= flip, w.w ^= flip;
                            *reinterpret_cast<uint4*>(smem + (r >> 7) * QTILE + c * QHALF + rr * 128 + ((x ^ (rr & 7)) << 4)) = w;
                        }
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sy.qfull));
            }
            const int mine = two ? p.tiles : (p.tiles + 1 - wg) >> 1;  // this warpgroup's tiles
            const int valid = two ? p.rows - wg * 128 : p.rows;        // ... and query rows
            const bool idle = (warp & 3) * 32 >= valid;
            float* keep = nullptr;  // where this row's scores go
            if (A.scores != nullptr && row < valid)
                keep = A.scores + ((size_t)p.head * p.rows + row) * A.score_n + p.start + wg * KT;
            float m = NEG_INF, l = 0.f;
#pragma unroll 1
            for (int i = 0; i < mine; ++i) {
                const int b = i & 1;
                if (!(ok = wait_or_fail(&sy.sfull[wg][b], (turn >> b) & 1, sy))) break;
                turn ^= 1u << b;
                tm_after();
                if (!idle) {
                    const int left = p.keys - (two ? i : 2 * i + wg) * KT;  // keys from this tile's first on
                    uint32_t s[2][32];
                    tm_ld32(ts + b * KT, s[0]);
                    tm_ld32(ts + b * KT + 32, s[1]);
                    tm_wait_ld(s[0]);
                    tm_wait_ld(s[1]);
                    if (left < KT) {
#pragma unroll
                        for (int c = 0; c < KT; ++c) s[c >> 5][c & 31] = c < left ? s[c >> 5][c & 31] : 0xff800000u;
                    }
                    float mx[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
                    for (int c = 0; c < KT; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c >> 5][c & 31]));
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                    // The weights are taken relative to a reference that follows the maximum only when that has risen by more
                    // than 8 (a factor of 256, which sums and bf16 weights hold without loss): most tiles leave the output alone.
                    const float ref = i == 0 ? top : (top > m + 8.f ? top : m);
                    if (i > 0 && __any_sync(0xffffffffu, ref != m)) {
                        // (the product before must be in: the one before that is, these scores were asked for after it)
                        if (!(ok = wait_or_fail(&sy.pv[wg][b ^ 1], ~(turn >> (b ^ 1)) & 1, sy))) break;
                        tm_after();
                        const float f = m == NEG_INF ? 0.f : ex2(m - ref);
                        l *= f;
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tm_ld16(to + c, o);
                            tm_wait_ld(o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tm_st16(to + c, o);
                        }
                    }
                    m = ref;
                    const float sub = m == NEG_INF ? 0.f : m;
                    if (keep != nullptr) {
                        float* to_row = keep + (size_t)i * (two ? KT : 2 * KT);
#pragma unroll
                        for (int c = 0; c < KT; c += 4)
                            *reinterpret_cast<float4*>(to_row + c) =
                                make_float4(__uint_as_float(s[c >> 5][c & 31]) * scale2, __uint_as_float(s[c >> 5][(c & 31) + 1]) * scale2,
                                            __uint_as_float(s[c >> 5][(c & 31) + 2]) * scale2, __uint_as_float(s[c >> 5][(c & 31) + 3]) * scale2);
                    }
                    const uint64_t mul = pair2(scale2, scale2), add = pair2(-sub, -sub);
                    uint64_t sum[2] = {0ull, 0ull};  // (two sums each)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            float x, y;
                            split2(fma2(pair2(__uint_as_float(s[h][2 * c]), __uint_as_float(s[h][2 * c + 1])), mul, add), x, y);
                            x = ex2(x), y = ex2(y);
                            sum[c & 1] = add2(sum[c & 1], pair2(x, y));
                            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[c]) : "f"(y), "f"(x));
                        }
                        tm_st16(ts + b * KT + h * 16, w);
                    }
                    float x, y;
                    split2(add2(sum[0], sum[1]), x, y);
                    l += x + y;
                    tm_wait_st();
                }
                tm_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sy.pready[wg][b]));
            }
            // ---- the part's state ----------------------------------------------------------------------------------------
            if (ok && mine > 0) ok = wait_or_fail(&sy.pv[wg][(mine - 1) & 1], ~(turn >> ((mine - 1) & 1)) & 1, sy);
            tm_after();
            if (!two && wg == 1) {
                s_m[row] = m, s_l[row] = l;
                tm_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sy.stats));
            }
            if (!two && wg == 0 && ok) {
                ok = wait_or_fail(&sy.stats, stph, sy);
                tm_after();
            }
            if (!two) stph ^= 1;
            if (ok && !idle && (two || wg == 0)) {
                const bool other = !two && p.tiles > 1;
                float f0 = 1.f, f1 = 0.f, M = m, L = l;
                if (other) fold_ml(M, L, s_m[row], s_l[row], f0, f1);
                const size_t row0 = (size_t)(p.row0 + warp * 32);  // the warp's first row (two: the second warpgroup's from 128 on)
                const int rows = min(32, valid - (warp & 3) * 32);
                // by way of the queries' place (all scores are made), so that a row's 32 columns are stored by eight lanes side by
                // side: row r, piece c of 16 bytes at c ^ (r & 7)
                uint8_t* mid = smem + warp * 4096;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    tm_ld32(to + c, o);
                    tm_wait_ld(o);
                    if (other) {
                        uint32_t o2[32];
                        tm_ld32(to + 128 + c, o2);
                        tm_wait_ld(o2);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(fold_e(__uint_as_float(o[k]), __uint_as_float(o2[k]), f0, f1));
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        *reinterpret_cast<uint4*>(mid + lane * 128 + ((k ^ (lane & 7)) << 4)) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int r = k * 4 + (lane >> 3), piece = lane & 7;
                        const uint4 v = *reinterpret_cast<const uint4*>(mid + r * 128 + ((piece ^ (r & 7)) << 4));
                        if (r < rows) *reinterpret_cast<uint4*>(A.part_o + (row0 + r) * D + c + piece * 4) = v;
                    }
                    __syncwarp();
                }
                if (lane < rows) A.part_ml[row0 + lane] = make_float2(M, L);
            }
            tm_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sy.next));
            if (ok) ok = wait_or_fail(&sy.next, nph, sy);
            nph ^= 1;
            tm_after();
        }
    } else if (warp == 8) {
        // ---- the loads --------------------------------------------------------------------------------------------------------
        int st = 0, asked[2] = {0, 0};  // copies of keys and of values begun
        uint32_t ph = 1;                // (the first round finds the stages empty)
        bool ok = true;
        for (int at = begin; at < stop && ok;) {
            const Part p = part_at<G>(plan, A.T * G, at, stop, blockIdx.x);
            if (p.tiles == 0) break;
            at = p.end;
            const int x = p.head * X.col_mul, y0 = p.head * X.row_mul;
            // sixteen lanes four rows each (each half of the lanes 64 columns); past the tile's keys the last one again (its
            // weight there is 0: the values multiplied by it must be ones that the rows see)
            auto rows_of = [&](int i, int* r) {
                const int keys = min(KT, p.keys - i * KT);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = p.start + i * KT + min((lane & 15) * 4 + k, keys - 1);
                    r[k] = A.tbl != nullptr ? A.tbl[j] : j;
                }
            };
            int ahead[4];
            if (A.tbl != nullptr) rows_of(0, ahead);
#pragma unroll 1
            for (int i = 0; i < p.tiles && ok; ++i) {
                int y[4], r0 = p.start + i * KT;
                bool box = p.keys - i * KT >= KT;  // 64 rows one after the other: one copy
                if (A.tbl != nullptr || !box) {    // (else nothing to look up: a tile's cost here is what this warp spends on it)
                    if (A.tbl == nullptr) rows_of(i, ahead);
                    r0 = __shfl_sync(0xffffffffu, ahead[0], 0);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        int r = ahead[k];
                        box = box && r == r0 + (lane & 15) * 4 + k;
                        if (r < 0 || r >= A.cap) {
                            b2_fail(B2_ERR_DOMAIN);
                            r = 0, box = false;
                        }
                        y[k] = y0 + r;
                    }
                    box = __all_sync(0xffffffffu, box);
                    if (A.tbl != nullptr && i + 1 < p.tiles) rows_of(i + 1, ahead);
                }
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (asked[kv] >= X.stages && !(ok = wait_or_fail(kv == 0 ? &sy.kempty[st] : &sy.vempty[st], ph, sy))) break;
                    const uint32_t bar = smem_u32(kv == 0 ? &sy.kfull[st] : &sy.vfull[st]), dst = (kv == 0 ? sk : sv) + st * TILE;
                    if (lane == 0) mbar_expect_tx(bar, TILE);
                    __syncwarp();
                    if (box) {
                        if (lane < D / 64) tma_box(dst + lane * HALF, kv == 0 ? &kbox : &vbox, x + lane * 64, y0 + r0, bar);
                    } else if (lane < D / 4) {
                        tma_rows4(dst + (lane >> 4) * HALF + (lane & 15) * 512, kv == 0 ? &krows : &vrows, x + (lane >> 4) * 64, y, bar);
                    }
                    ++asked[kv];
                }
                if (++st == X.stages) st = 0, ph ^= 1;
            }
        }
        // its copies have landed before the CTA ends (they have, unless some role gave up)
        for (int s = 0; s < X.stages; ++s)
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const int uses = (asked[kv] + X.stages - 1 - s) / X.stages;
                if (uses > 0) (void)mbar_wait_bounded(smem_u32(kv == 0 ? &sy.kfull[s] : &sy.vfull[s]), (uint32_t)(uses - 1) & 1);
            }
    } else if (warp >= 10) {
        if (warp == 10 && blockIdx.x == 0) tell_plan<G>(A, plan);
        own_units<D, G>(A, plan, (warp - 10) * gridDim.x + blockIdx.x, OWN_WARPS * gridDim.x);
    } else {
        // ---- the MMAs -----------------------------------------------------------------------------------------------------------
        // What a job costs this warp is its instructions, one after the other beside the weights' warps, so a buffer's and a
        // warpgroup's numbers are constants of an unrolled turn of four jobs and addresses advance by additions.
        const uint32_t lead = elect_lane(), q0 = desc_sw128(sq, 0), k0 = desc_sw128(sk, 0), v0 = desc_sw128(sv, HALF);
        Issuer is{k0, v0, 0, 0, 0u, 0u, 0u};
        uint32_t qph = 0;
        bool ok = true;
        for (int at = begin; at < stop && ok;) {
            const Part p = part_at<G>(plan, A.T * G, at, stop, blockIdx.x);
            const int tiles = __shfl_sync(0xffffffffu, p.tiles, 0), rows = __shfl_sync(0xffffffffu, p.rows, 0);
            if (tiles == 0) break;
            at = __shfl_sync(0xffffffffu, p.end, 0);
            if (!(ok = wait_or_fail(&sy.qfull, qph, sy))) break;
            qph ^= 1;
            ok = rows > 128 ? issue_part<D, 2>(is, sy, lead, tmem, q0, k0, v0, X.stages, 2 * tiles)
                            : issue_part<D, 1>(is, sy, lead, tmem, q0, k0, v0, X.stages, tiles);
        }
        mma_commit(lead, smem_u32(&sy.drain));
        (void)mbar_wait_bounded(smem_u32(&sy.drain), 0);
        __syncwarp();
    }
    tm_before();
    __syncthreads();
    if (threadIdx.x == 0 && (sy.fail || (sq & 1023))) b2_fail(sy.fail ? B2_ERR_TIMEOUT : B2_ERR_CUDA);
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---- a row's parts joined ------------------------------------------------------------------------------------------------
constexpr int JT = 256, JW = JT / 32;      // threads and warps of a block
constexpr int STATES_MAX = CTAS_MAX + 64;  // a row's parts and units
constexpr int WEIGHT_KEYS = 4 * JT;         // keys of a block that adds up weights
// a kv head's queries (T G) up to which a pass keeps its scores for the weights instead of making them again. Over 32768 rows
// of 8 heads by 8 queries, us a call kept and made again: 8 queries 37 and 54, 16 41.5 and 56, 32 51 and 59, 64 77 and 59.6. (That
// length alone was measured: shorter caches, whose scores are fewer bytes, go by the same number.)
constexpr int KEEP_ROWS = 32;

// where the states of (row t, kv head g) lie: state k of query head hh in row at(k) + hh
struct States {
    long long p_row, u_row;
    int np, n, step, G;
    // a: place, tiles, row, units; b: unit, line, rows, units
    __device__ __forceinline__ States(const LongArgs& A, const int4 a, const int4 b, int g, int G_) : G(G_) {
        const int place = g * b.y + a.x;
        int c = 0;
        np = 0, step = A.T * G;
        if (a.y > 0) {
            const Cut cut(b.y * A.Hk, A.ctas);
            c = cut.cta_of(place);
            np = cut.cta_of(place + a.y - 1) - c + 1;
        }
        p_row = (long long)c * step + (long long)g * b.z + a.z;
        u_row = A.unit_row + ((long long)g * b.w + b.x) * G;
        n = np + a.w;
    }
    __device__ __forceinline__ long long at(int k) const { return k < np ? p_row + (long long)k * step : u_row + (long long)(k - np) * G; }
};
// a warp's look at a query head's states: the largest maximum M and the sum L relative to it, the sink in both; the states'
// factors into `fac` where given
__device__ __forceinline__ void row_stats(const LongArgs& A, const States& S, int head, int hh, float& M, float& L, float* fac) {
    const int lane = threadIdx.x & 31;
    const float sink = A.sinks != nullptr ? __fmul_rn(A.sinks[head], LOG2E) : NEG_INF;
    M = sink;
    const float2 first = lane < S.n ? __ldcg(A.part_ml + S.at(lane) + hh) : make_float2(NEG_INF, 0.f);
    M = fmaxf(M, first.x);
    for (int k = lane + 32; k < S.n; k += 32) M = fmaxf(M, __ldcg(A.part_ml + S.at(k) + hh).x);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
    const float sub = M == NEG_INF ? 0.f : M;
    L = 0.f;
    for (int k = lane; k < S.n; k += 32) {
        const float2 ml = k == lane ? first : __ldcg(A.part_ml + S.at(k) + hh);
        const float f = ml.x == NEG_INF ? 0.f : ex2(ml.x - sub);
        L += f * ml.y;
        if (fac != nullptr) fac[k] = f;
    }
    L = warp_sum(L);
    if (A.sinks != nullptr) L += ex2(sink - sub);
}

// The first T Hk blocks join one (row, kv head) each: JW / G warps a query head, each every so many-th state, a lane D / 32
// dims, their sums added in order. The blocks after them, where a pass of few rows kept its scores, add up what it gives each
// cache row: a thread four keys, 2^(score - log2 of the row's denominator) over the kv head's queries in order - one sum in one
// order.
template <int D, int G>
__global__ void __launch_bounds__(JT) long_join(const LongArgs A, int weight_blocks) {
    constexpr int E = D / 32, WH = JW / G;  // warps a query head
    __shared__ float fac[JW][STATES_MAX];
    __shared__ __align__(16) float part[JW][D];
    __shared__ float s_lse[KEEP_ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    if ((int)blockIdx.x < A.T * A.Hk) {
        const int t = blockIdx.x / A.Hk, g = blockIdx.x - t * A.Hk, hh = warp / WH, sub = warp - hh * WH, head = g * G + hh;
        float M, L, o[E];
        // Twice: first, while the tiles are still at work, over places of the workspace whose contents are of no interest, so
        // that the instructions are on the SM when the states are (two rows over 128 take 9.3 us a call so, else 9.7; one over 32768
        // 37.4, else 38.5).
#pragma unroll 1
        for (int real = 0; real < 2; ++real) {
            int4 a = make_int4(0, 1, 0, 1), b = make_int4(0, 1, 1, 1);
            if (real) {
                pdl_wait();
                a = __ldcg(A.info + 2 * t), b = __ldcg(A.info + 2 * t + 1);
            }
            const States S(A, a, b, g, G);
            if (S.n == 0) return;  // padding, or refused
            constexpr int B = 8;  // states in flight; the first ones are asked for before their factors are known
            float v[B][E];
            auto load = [&](int k0) {
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const float* src = A.part_o + (size_t)(S.at(min(k0 + j * WH, S.n - 1)) + hh) * D + lane * E;
                    if (E == 4) {
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
                        v[j][0] = x.x, v[j][1] = x.y, v[j][E - 2] = x.z, v[j][E - 1] = x.w;
                    } else {
                        const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
                        v[j][0] = x.x, v[j][E - 1] = x.y;
                    }
                }
            };
            load(sub);
            row_stats(A, S, head, hh, M, L, fac[warp]);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 1
            for (int k0 = sub; k0 < S.n; k0 += B * WH) {
                if (k0 != sub) load(k0);
#pragma unroll
                for (int j = 0; j < B; ++j) {  // (no branch: the loads would sink below it, one after the other)
                    const bool on = k0 + j * WH < S.n;
                    const float f = on ? fac[warp][on ? k0 + j * WH : 0] : 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = fmaf(f, on ? v[j][e] : 0.f, o[e]);
                }
            }
            if (WH > 1) {
#pragma unroll
                for (int e = 0; e < E; ++e) part[warp][lane * E + e] = o[e];
                __syncthreads();
                if (sub == 0)
                    for (int w = 1; w < min(WH, S.n); ++w)
#pragma unroll
                        for (int e = 0; e < E; ++e) o[e] += part[warp + w][lane * E + e];
                __syncthreads();
            }
        }
        if (sub != 0) return;
        if (lane == 0 && A.lse != nullptr) A.lse[(size_t)t * A.Hq + head] = M + log2f(L);
        bf16* out = A.out + ((size_t)t * A.Hq + head) * D + lane * E;
        const float inv = __fdiv_rn(1.f, L);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            __nv_bfloat162 v;
            v.x = f2bf(o[e] * inv), v.y = f2bf(o[e + 1] * inv);
            *reinterpret_cast<__nv_bfloat162*>(out + e) = v;
        }
        return;
    }
    // ---- the weights ------------------------------------------------------------------------------------------------------
    pdl_wait();
    const int b = blockIdx.x - A.T * A.Hk, g = b / weight_blocks, n0 = __ldcg(A.n0p);
    const int n = n0 < 0 || n0 > A.cap - A.T ? -1 : n0 + (A.T == 1);  // keys whose scores were kept; -1: refused
    const int j0 = (b - g * weight_blocks) * WEIGHT_KEYS;
    if (n < 0 || (j0 >= n && j0 > 0)) return;
    const int rows = A.T * G;
    const float* from = A.scores + (size_t)g * rows * A.score_n + threadIdx.x * 4;
    float4 s[8];  // (the first scores asked for before the denominators are made)
    auto load = [&](int j, int r0) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            s[r] = r0 + r < rows && j + (int)threadIdx.x * 4 < n ? __ldcg(reinterpret_cast<const float4*>(from + (size_t)(r0 + r) * A.score_n + j))
                                                                  : make_float4(NEG_INF, NEG_INF, NEG_INF, NEG_INF);
    };
    load(j0, 0);
    for (int r = warp; r < rows; r += JW) {
        const int t = r / G, hh = r - t * G;
        const States S(A, __ldcg(A.info + 2 * t), __ldcg(A.info + 2 * t + 1), g, G);
        float M, L;
        row_stats(A, S, g * G + hh, hh, M, L, nullptr);
        if (lane == 0) s_lse[r] = M + log2f(L);
    }
    __syncthreads();
    float* tot = A.totals + (size_t)g * A.ts;
    if (A.T > 1 && j0 == 0 && (int)threadIdx.x < A.T) {  // the pass's own rows: set
        float a = 0.f;
#pragma unroll 8
        for (int r = 0; r < rows; ++r) a += ex2(__ldcg(A.own + ((size_t)(r / G) * A.Hq + g * G + r % G) * 32 + threadIdx.x) - s_lse[r]);
        tot[n0 + threadIdx.x] = a;
    }
    for (int j = j0; j < n; j += weight_blocks * WEIGHT_KEYS) {
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < rows; r0 += 8) {
            if (j != j0 || r0 != 0) load(j, r0);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r0 + r >= rows) break;
                const float d = s_lse[r0 + r];
                a[0] += ex2(s[r].x - d), a[1] += ex2(s[r].y - d), a[2] += ex2(s[r].z - d), a[3] += ex2(s[r].w - d);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = j + threadIdx.x * 4 + k;
            if (at < n) tot[at] = at < n0 ? tot[at] + a[k] : a[k];
        }
    }
}

// ---- what a pass of many rows gives each cache row -------------------------------------------------------------------------
// The scores once more, turned round: S^T = K Q^T with 128 keys as the MMA's M and the kv head's T G queries as its N, so that
// a thread has a key and adds the weights 2^(score - log2 of the row's denominator) of its row of tensor memory one after the
// other - one sum in one order, no exchange. Bound by the powers (a tile of 128 keys and 256 queries: 32768, 16 a clock) once
// there are tiles for every SM; the queries, the first tile and its product are ready before the joining kernel is waited for.
constexpr int WT = 128;  // keys of a tile, threads of a block
template <int D>
__global__ void __launch_bounds__(WT) long_weights(const __grid_constant__ CUtensorMap kbox, const __grid_constant__ CUtensorMap krows,
                                                   const TileArgs X) {
    constexpr int TILE = WT * D * 2, HALF = WT * 128;
    const LongArgs& A = X.a;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t full, done;
    __shared__ uint32_t tmem_slot;
    __shared__ float s_lse[256], s_own[4][32];
    const int G = A.Hq / A.Hk, rows = A.T * G, N = (rows + 31) & ~31, g = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sk = smem_u32(smem), sq = sk + TILE, cols = N > 128 ? 256u : N > 64 ? 128u : N > 32 ? 64u : 32u;
    const int n0 = *A.n0p;
    const bool fits = n0 >= 0 && n0 <= A.cap - A.T && !(sk & 1023);
    const int tiles = fits ? (n0 + WT - 1) / WT : 0;
    if ((sk & 1023) && threadIdx.x == 0) b2_fail(B2_ERR_CUDA);
    if (!fits || ((int)blockIdx.x >= tiles && blockIdx.x > 0)) {
        pdl_launch_dependents();
        pdl_wait();
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&full), 1), mbar_init(smem_u32(&done), 1);
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tm_before();
    __syncthreads();
    tm_after();
    pdl_launch_dependents();
    const uint32_t tmem = tmem_slot;
    const int x = g * X.col_mul, y0 = g * X.row_mul;
    auto load = [&](int tile) {  // (warp 0)
        const int keys = min(WT, n0 - tile * WT);
        const uint32_t bar = smem_u32(&full);
        if (lane == 0) mbar_expect_tx(bar, TILE);
        __syncwarp();
        if (keys == WT && A.tbl == nullptr) {
            if (lane < D / 32) tma_box(sk + lane * (KT * 128), &kbox, x + (lane >> 1) * 64, y0 + tile * WT + (lane & 1) * KT, bar);
            return;
        }
        int y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = tile * WT + min(lane * 4 + k, keys - 1);
            const int r = A.tbl != nullptr ? A.tbl[j] : j;
            y[k] = y0 + (r < 0 || r >= A.cap ? 0 : r);  // (refused by the tiles' kernel)
        }
        for (int c = 0; c < D / 64; ++c) tma_rows4(sk + c * HALF + lane * 512, &krows, x + c * 64, y, bar);
    };
    if (warp == 0 && tiles > 0) load(blockIdx.x);
    for (int i = threadIdx.x; i < rows * (D / 8); i += WT) {
        const int r = i / (D / 8), piece = i - r * (D / 8), t = r / G;
        const uint4 v = reinterpret_cast<const uint4*>(A.q + ((size_t)t * A.Hq + g * G + r - t * G) * D)[piece];
        *reinterpret_cast<uint4*>(smem + TILE + (piece >> 3) * (N * 128) + r * 128 + (((piece & 7) ^ (r & 7)) << 4)) = v;
    }
    fence_proxy_async();
    __syncthreads();
    const float scale2 = __fmul_rn(A.scale, LOG2E);
    float* tot = A.totals + (size_t)g * A.ts;
    bool ok = true, first = true;
    uint32_t ph = 0;
    for (int tile = blockIdx.x; first || tile < tiles; tile += gridDim.x, ph ^= 1) {
        if (warp == 0 && tile < tiles) {
            ok = mbar_wait_bounded(smem_u32(&full), ph);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(WT >> 4) << 24);
                const uint32_t ka = desc_sw128(sk, 0), qb = desc_sw128(sq, 0);
                tm_after();
                const uint32_t lead = elect_lane();
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_ss(lead, tmem, ka + (uint32_t)(((k >> 2) * HALF + (k & 3) * 32) >> 4),
                           qb + (uint32_t)(((k >> 2) * (N * 128) + (k & 3) * 32) >> 4), idesc, k > 0);
                mma_commit(lead, smem_u32(&done));
            }
        }
        if (first) {  // everything so far was there before the tiles; the denominators are the joining kernel's
            pdl_wait();
            for (int r = threadIdx.x; r < rows; r += WT) s_lse[r] = A.lse[(size_t)(r / G) * A.Hq + g * G + r % G];
            __syncthreads();
            if (blockIdx.x == 0) {  // the pass's own rows: set; a lane a row, each warp a quarter of the queries
                const int each = (rows + 3) / 4, lo = warp * each, hi = min(lo + each, rows);
                float a = 0.f;
#pragma unroll 16
                for (int r = lo; r < hi; ++r) {
                    const int t = r / G;
                    a += ex2(__ldcg(A.own + ((size_t)t * A.Hq + g * G + r - t * G) * 32 + lane) - s_lse[r]);
                }
                s_own[warp][lane] = a;
                __syncthreads();
                if ((int)threadIdx.x < A.T) tot[n0 + lane] = (s_own[0][lane] + s_own[1][lane]) + (s_own[2][lane] + s_own[3][lane]);
            }
            first = false;
        }
        if (tile >= tiles) break;
        if (ok) ok = mbar_wait_bounded(smem_u32(&done), ph);
        if (!__syncthreads_and(ok)) break;
        tm_after();
        if (warp == 0 && tile + (int)gridDim.x < tiles) load(tile + gridDim.x);  // (the product has read this one)
        float a = 0.f;
        const uint32_t at = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll 1
        for (int c0 = 0; c0 < N; c0 += 32) {
            uint32_t s[32];
            tm_ld32(at + c0, s);
            tm_wait_ld(s);
            const int n = min(32, rows - c0);
            if (n == 32) {
                float e[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) e[c] = ex2(fmaf(__uint_as_float(s[c]), scale2, -s_lse[c0 + c]));
#pragma unroll
                for (int c = 0; c < 32; ++c) a += e[c];
            } else {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (c < n) a += ex2(fmaf(__uint_as_float(s[c]), scale2, -s_lse[c0 + c]));
            }
        }
        const int j = tile * WT + threadIdx.x;
        if (j < n0) tot[j] += a;
        tm_before();
        __syncthreads();
        tm_after();
    }
    if (!ok) b2_fail(B2_ERR_TIMEOUT);
    tm_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
// a cache of `rows` rows of `cols` elements, `stride` elements apart, in boxes of box_rows x 64 under the 128-byte swizzle
int make_map(CUtensorMap* tm, const void* base, long long rows, long long cols, long long stride, int box_rows) {
    static std::atomic<EncodeFn> known{nullptr};
    EncodeFn fn = known.load(std::memory_order_acquire);
    if (fn == nullptr) {
        cudaDriverEntryPointQueryResult q;
        void* p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || p == nullptr) {
            (void)cudaGetLastError();
            return B2_ERR_CUDA;
        }
        fn = reinterpret_cast<EncodeFn>(p);
        known.store(fn, std::memory_order_release);
    }
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, es[2] = {1, 1};
    return fn(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? B2_OK
               : B2_ERR_DOMAIN;
}

// the kernels of a call start under programmatic dependent launch (bit 3 of the `pdl` tunable): each sets up while the one
// before it drains
template <typename... P, typename... A>
int launch(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute at[1];
    if (b2_tuning().pdl & 8) {
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at, cfg.numAttrs = 1;
    }
    if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) {
        (void)cudaGetLastError();
        return B2_ERR_CUDA;
    }
    return B2_OK;
}

int long_ctas() { return min(b2_sm_count(), CTAS_MAX); }
// rows of the parts at most: a CTA's stretch moves on by the rows of a kv head's items, T G at most, and a kv head by as many
// (32 rows of 64 heads over 8 kv heads of 128: 38 MB with the units' rows)
size_t part_rows(int T, int Hq, int Hk) { return (size_t)long_ctas() * T * (Hq / Hk) + (size_t)T * Hq; }
size_t state_rows(int T, int Hq, int Hk) { return part_rows(T, Hq, Hk) + (size_t)T * Hq * units_max(T, Hk); }
constexpr size_t INFO_BYTES = TMAX * 2 * sizeof(int4);
long long score_stride(int cap) { return ((long long)cap + KT - 1) / KT * KT; }
bool keeps_scores(int T, int Hq, int Hk) { return T * (Hq / Hk) <= KEEP_ROWS; }

template <int D, int G>
int launch_long(const LongArgs& a, cudaStream_t s) {
    TileArgs x{};
    x.a = a;
    const bool by_row = a.Hk == 1 || (a.Hk - 1) * a.hs + D <= a.rs;  // kv heads inside a cache row
    const long long rows = by_row ? a.cap : (a.Hk - 1) * (a.hs / a.rs) + a.cap, cols = by_row ? (a.Hk - 1) * (a.Hk > 1 ? a.hs : 0) + D : D;
    if (rows > 0x7fffffffLL || cols > 0x7fffffffLL) return B2_ERR_DOMAIN;
    x.row_mul = by_row ? 0 : (int)(a.hs / a.rs), x.col_mul = by_row && a.Hk > 1 ? (int)a.hs : 0;
    CUtensorMap tm[4];
    for (int k = 0; k < 4; ++k)
        if (const int rc = make_map(&tm[k], k < 2 ? a.K : a.V, rows, cols, a.rs, k & 1 ? 1 : KT)) return rc;
    const int tile = KT * D * 2, queries = (a.T * G > 128 ? 2 : 1) * 128 * D * 2;
    // (16 KB short of what a block may have: the joining kernel's blocks then find room a little earlier. 8 rows over 2048 take
    // 15.6 us so, else 16.5, 32 over 32768 47.4 and 49.1; one row over 32768, with a stage fewer, 38.1 and 37.5)
    x.stages = min((208 * 1024 - queries) / (2 * tile), STAGES_MAX);
    auto tiles = long_tiles<D, G>;
    static bool tiles_allowed[64], weights_allowed[64];
    if (const int rc = b2_allow_smem(reinterpret_cast<const void*>(tiles), tiles_allowed)) return rc;
    if (const int rc = launch(tiles, dim3(a.ctas), dim3(TW * 32), (size_t)queries + (size_t)2 * x.stages * tile, s, tm[0], tm[1], tm[2], tm[3], x))
        return rc;
    // (blocks enough for the whole cache, or for the card)
    const int wb = a.scores != nullptr ? min((a.cap + WEIGHT_KEYS - 1) / WEIGHT_KEYS, max(1, 4 * a.ctas / a.Hk)) : 0;
    if (const int rc = launch(long_join<D, G>, dim3(a.T * a.Hk + wb * a.Hk), dim3(JT), 0, s, a, wb)) return rc;
    if (a.totals == nullptr || a.scores != nullptr) return B2_OK;
    auto weights = long_weights<D>;
    if (const int rc = b2_allow_smem(reinterpret_cast<const void*>(weights), weights_allowed)) return rc;
    // a grid of two blocks an SM. (Nothing holds an SM to two: at head dim 64 its shared memory has room for four, and of more
    // than 512 columns of tensor memory the later blocks wait until the earlier ones have ended)
    const int N = (a.T * G + 31) & ~31;
    return launch(weights, dim3(min((a.cap + WT - 1) / WT, max(1, 2 * a.ctas / a.Hk)), a.Hk), dim3(WT), (size_t)(WT + N) * D * 2, s, tm[0], tm[1], x);
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
    if ((long long)cap * Hk > 0x7fffffffLL) return B2_ERR_DOMAIN;  // (tiles are counted in 32 bits)
    if (Hk > 1 && !((Hk - 1) * hs + D <= rs || (hs % rs == 0 && hs / rs >= cap))) return B2_ERR_DOMAIN;
    if (misaligned(q) || misaligned(K) || misaligned(V) || misaligned(out) || misaligned(workspace)) return B2_ERR_DOMAIN;
    return B2_OK;
}

}  // namespace

extern "C" size_t btb_b200_attn_shared_workspace_bytes(int T, int Hq, int Hk, int D) {
    return shape_ok(T, Hq, Hk, D) ? state_rows(T, Hq, Hk) * (D * 4 + 8) + INFO_BYTES : 0;
}

// the states' place in a workspace; returns what lies behind it
static float* take_states(LongArgs& a, void* workspace, int D) {
    const size_t rows = state_rows(a.T, a.Hq, a.Hk);
    a.info = static_cast<int4*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + INFO_BYTES);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * D);
    a.unit_row = (long long)part_rows(a.T, a.Hq, a.Hk);
    return reinterpret_cast<float*>(a.part_ml + rows);
}

extern "C" int btb_b200_attn_shared(const void* q, const void* K, const void* V, void* out, const void* rw, int T, int Hq,
                                    int Hk, int D, long long hs, long long rs, float scale, void* workspace, int win,
                                    const void* sinks, int cap, void* stream) {
    if (!q || !K || !V || !out || !rw || !workspace) return B2_ERR_NULL;
    if (const int rc = check_cache(q, K, V, out, T, Hq, Hk, D, hs, rs, scale, workspace, cap)) return rc;
    LongArgs a{};
    a.q = static_cast<const bf16*>(q), a.K = static_cast<const bf16*>(K), a.V = static_cast<const bf16*>(V);
    a.out = static_cast<bf16*>(out), a.rw = static_cast<const int*>(rw), a.sinks = static_cast<const float*>(sinks);
    a.scale = scale, a.T = T, a.Hq = Hq, a.Hk = Hk, a.win = win, a.cap = cap, a.ctas = long_ctas(), a.hs = hs, a.rs = rs;
    a.own_share = max(1, a.ctas * OWN_WARPS / Hk);
    (void)take_states(a, workspace, D);
    return D == 64 ? launch_long_g<64>(a, static_cast<cudaStream_t>(stream)) : launch_long_g<128>(a, static_cast<cudaStream_t>(stream));
}

extern "C" size_t btb_b200_attn_scored_workspace_bytes(int T, int Hq, int Hk, int D, int cap) {
    if (!shape_ok(T, Hq, Hk, D) || cap <= 0) return 0;
    size_t n = INFO_BYTES + state_rows(T, Hq, Hk) * (D * 4 + 8) + (size_t)T * Hq * 33 * 4;
    if (keeps_scores(T, Hq, Hk)) n = ((n + 15) & ~(size_t)15) + (size_t)T * Hq * score_stride(cap) * 4;
    return n;
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
    a.scale = scale, a.T = T, a.Hq = Hq, a.Hk = Hk, a.cap = cap, a.ctas = long_ctas(), a.hs = hs, a.rs = rs;
    a.own_share = max(1, a.ctas * OWN_WARPS / Hk);
    a.lse = take_states(a, workspace, D), a.own = a.lse + (size_t)T * Hq;
    if (keeps_scores(T, Hq, Hk)) {
        const uintptr_t past = reinterpret_cast<uintptr_t>(a.own + (size_t)T * Hq * 32);
        a.scores = reinterpret_cast<float*>((past + 15) & ~(uintptr_t)15), a.score_n = score_stride(cap);
    }
    return D == 64 ? launch_long_g<64>(a, static_cast<cudaStream_t>(stream)) : launch_long_g<128>(a, static_cast<cudaStream_t>(stream));
}
