// sjk_kv16_tree.cu - attention of several new tokens of every sequence, drafted as a tree or in a row, over a paged 16-bit
// cache: out_j = sum over V(j) of softmax(scale q_j . k_t) v_t, V(j) = the last `window` of the committed positions [0, len)
// and the drafted ones len + k whose bit k token j's mask has.
//
// All query heads of a KV head's group, of all the tokens of a sequence, are rows of one product: a key read once serves
// (tokens x heads of a group) rows, up to NMAX = 64 or 128 in one pass, more in tiles of rows that CTAs side by side work on at
// the same time, so that the second one's keys come from L2 (100,000 tokens, 256 rows: 411 MB of DRAM reads for 410 MB of live
// rows). Bound: HBM up to 64 rows a KV head; above that waits between the steps of a tile's chain (rows, products, maximum, weights,
// products: some 4,000 to 5,000 cycles, in which the warps issue 0.47 instructions a cycle), and for short sequences that chain
// alone; for hundreds of them the walk over the sequences, a warp's in every CTA and then each role's. Measured (us a pass from
// Python, of a program that keeps the GPU busy, which in the second case then runs at 1.2 GHz under its power cap, box by box):
// one chat of 611 tokens with 8 drafts 12.9; 32 sequences of 8K-64K, 4 KV heads of 256 bf16 channels, 16 drafts x 4 heads 870-910 (84 to
// 88 % of a plain copy's rate); 100,000 tokens, 8 heads of 128 f16 channels, 64 drafts x 4 heads 244-251 (420-430 TFLOP/s); 64 pieces of
// up to 33 tokens over windows of 512, 24 heads of 64 channels 103. 1,024 sequences of 100 tokens with 4 drafts, 2 KV heads of 128
// channels, on the GPU: 90, and 106 with `first`; 4,096 of 20: 329 and 382.
//  - S^T = K Q^T with 128 positions as the M rows of tcgen05.mma and the query rows as its N columns (16 to 128), and
//    O^T += V^T P with 128 channels as M: what a tile costs the softmax goes with the number of query rows, where query rows
//    as M would make 8 of them as dear as 128. K, V and P lie in shared memory as they come: K rows are K-major for the
//    first product, the same layout of V is MN-major for the second, and a thread, which has a position of all columns,
//    writes its weights as whole 16-byte words of an MN-major P. S (two buffers) and O live in TMEM.
//  - Warps: 16 for the softmax (a quarter of the columns each four, 16 columns at a time: 260 us at 100,000 tokens, where 8 with 32
//    columns took 269 and 16 with 32 spilled registers, 299), one each that loads K, loads V (rings of their own, so that neither
//    waits for the other's slots), issues the products (a whole warp, so that descriptors are uniform: 32 sequences 1,355 -> 930
//    with it and the boxes), and loads the queries. Linked by mbarriers only; every wait is bounded.
//  - Pages of a multiple of 8 tokens come as TMA boxes of up to 128 tokens of a page and 64 channels, into the swizzled layout;
//    others row by row with 16-byte cp.async. Rows of a box that are not live are zeroed on their way, and the second product
//    takes groups of 16 positions with a live one alone.
//  - The maximum of a row is looked for when a score is more than SLACK above the one in use (at a pair's start, seldom
//    afterwards); then O is rescaled in TMEM. Weights reach 2^SLACK, which f16 and 32-bit sums have room for.
//  - Weights enter as the sum of two 16-bit terms, as in sjk_kv16_attend: 2^-16 (bf16) or 2^-22 (f16) of a weight, and for
//    f16, whose weights are held 2^10 larger, at most 2^-35 of the row's largest. Sums and statistics are 32-bit.
//  - V may hold infinities or NaNs in positions that only some of the rows see (drafted ones, a window's edge), and 0 times those is no
//    zero, nor is it one in a weight's second term. Pairs of which a sum comes out as no number are gone through once more behind
//    all others, with V's infinities and NaNs as zeros (noted on the way, per channel or, where rows see different positions, per
//    position) and then put into the sums of the rows that see them. So a bad value costs its CTA's pairs a second time in the same
//    pipeline, however long they are, and no role waits longer than for a tile (rows summed anew where they occur, a position
//    at a time, would hold the others up beyond what they wait). Looking for them in every V tile instead slows all calls. A NaN in
//    every sequence (us, a call without and with): 1 x 611 13.5 and 32, 1 x 100,000 217 and 971, 32 x 36,000 746 and 4,450.
// A list of (sequence, KV head) pairs in steps of 128 positions is cut into equal runs, one per CTA, for each tile of rows;
// lengths are read from device memory. Split pairs leave (m, l, o) in the scratch and a second kernel joins them in order.
#include "sjk_kv16.cuh"
#include "sjk_internal.h"
#include "sjk_tc.cuh"

#include <cuda.h>

#include <math.h>

namespace {

using namespace sjk16;

constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int TS = 128;                     // positions of a step
constexpr int CTAS = 148;                   // one per SM
constexpr int OV = 1;                       // what a pair costs beside its steps, in steps
constexpr int GROUPS = 4;                   // of softmax warps, which divide the columns
constexpr int N_SOFT = 4 * GROUPS, N_LOAD = 2;       // warps; then one that issues products, and one that loads queries
constexpr int W_MMA = N_SOFT + N_LOAD, W_Q = W_MMA + 1, NT = 32 * (W_Q + 1);
constexpr int INFO = 4, TILES = 16;         // rings of what a pair's rows and a tile's positions are
constexpr int SEG = 1024;                   // pairs that are gone through before those of them that come again
constexpr int EDGES = 4;                    // tiles of a pair of which rows see different positions: up to 64 positions from two places on
__device__ unsigned int g_tree_status;

SJK_DEV void flag() { atomicOr(&g_tree_status, (unsigned) SJK_DEVICE_PAGE); }

struct Params {
    sjk_kv16 c;
    sjk_rows q, out;
    const int32_t * first, * len, * rows;
    const uint64_t * masks;
    int n_seq, n_tok, nodes, grp;
    int window, page_shift;
    float scale;
    bool over;                              // outputs may lie over the queries
    float * part;                           // [CTA][2][NMAX][D]
    float * ml;                             // [CTA][2][NMAX][2]
    int4 * split;                           // by CTA: sequence (-1: none), KV head, first and last run; behind them: tiles
    int box;                                // tokens of a box (WHOLE)
    CUtensorMap maps[2];                    // K, V (WHOLE)
};

// What a sequence is to a tile of rows: its committed length, tokens, positions [lo, hi) that some token sees, rows.
struct Seq {
    int len, count, first, row0, nr, step0, steps;
    uint32_t hi;
};
// its first token and their number (0: none, or more than there may be)
SJK_DEV int2 tokens_of(const Params & p, int i) {
    if (!p.first) return make_int2(i * p.nodes, p.nodes);
    const int64_t f0 = p.first[i], f1 = p.first[i + 1];
    if (f0 < 0 || f1 < f0 || f1 > p.n_tok || f1 - f0 > p.nodes) { flag(); return make_int2(0, 0); }
    return make_int2((int) f0, (int) (f1 - f0));
}
SJK_DEV int tiles_of(const Params & p, int i, int nmax) { return (tokens_of(p, i).y * p.grp + nmax - 1) / nmax; }
SJK_DEV Seq seq_of(const Params & p, int i, int tile, int nmax) {
    Seq s = {0, 0, 0, 0, 0, 0, 0, 0u};
    const int len = p.len[i];
    const int2 tok = tokens_of(p, i);
    s.first = tok.x;
    s.count = tok.y;
    const int rows = s.count * p.grp, tiles = (rows + nmax - 1) / nmax;
    if (tile >= tiles) return s;
    s.nr = rows;
    if (tiles > 1) {                        // (rows are at most CTAS NMAX: the products fit)
        s.row0 = (int) ((unsigned) rows * (unsigned) tile / (unsigned) tiles);
        s.nr = (int) ((unsigned) rows * (unsigned) (tile + 1) / (unsigned) tiles) - s.row0;
    }
    s.len = max(len, 0);
    int64_t hi = (int64_t) s.len + s.count;
    const int64_t cap = (int64_t) p.c.table_stride * p.c.page_tokens, most = cap < 0x7FFFFFFF ? cap : 0x7FFFFFFF;
    if (hi > most) { flag(); hi = most; }
    s.hi = (uint32_t) hi;
    const int lo = p.window && s.len > p.window ? s.len - p.window : 0;
    s.step0 = (int) ((uint32_t) min((int64_t) lo, hi - 1) / TS);
    s.steps = (int) ((s.hi - 1u) / TS) + 1 - s.step0;
    return s;
}
SJK_DEV uint32_t units_of(const Params & p, const Seq & s) { return s.steps > 0 ? (uint32_t) p.c.n_head_kv * (uint32_t) (s.steps + OV) : 0u; }

// First committed position that some token of the pair may see, and whether some of its rows see a position of a tile (from
// t0 on) that others do not: a drafted one, or one at the window's edge.
SJK_DEV uint32_t low_of(const Params & p, const Seq & s) { return p.window && s.len > p.window ? (uint32_t) (s.len - p.window) : 0u; }
SJK_DEV bool partly(const Params & p, const Seq & s, uint32_t t0) { return t0 + TS > (uint32_t) s.len || (p.window && t0 < low_of(p, s) + (uint32_t) s.count); }
// Groups of 16 positions of a tile that lie in the pair's span (one at least): the second product takes these alone.
SJK_DEV int end16(const Seq & s, uint32_t t0) { const uint32_t n = s.hi - t0; return n < TS ? (int) ((n + 15u) >> 4) : TS / 16; }
SJK_DEV int first16(const Params & p, const Seq & s, uint32_t t0) {
    const uint32_t lo = low_of(p, s);
    return lo > t0 ? min((int) ((lo - t0) >> 4), end16(s, t0) - 1) : 0;
}

// A run's place: pair (sequence, KV head), step, units left, unit of the list at which the pair begins.
struct Cursor {
    int seq, h, st, rem;
    uint32_t base;
    Seq s;
    // the pair's steps of this run
    SJK_DEV int take() const { const int left = s.steps - st; return left < rem ? left : rem; }
    SJK_DEV void next(const Params & p, int tile, int nmax, int taken) {
        rem -= taken;
        st += taken;
        if (st < s.steps) return;
        st = 0;
        rem -= OV;
        base += (uint32_t) (s.steps + OV);
        if (rem <= 0) return;
        if (++h < p.c.n_head_kv) return;
        h = 0;
        do { s = seq_of(p, ++seq, tile, nmax); } while (s.steps <= 0);
    }
};

template <int N>
struct Int { static constexpr int value = N; };

// What row n of a pair is.
template <int NMAX>
struct Info {
    uint64_t mask[NMAX];                    // drafted tokens that it sees
    int64_t out[NMAX];                      // its place in the output
    int lo[NMAX];                           // first committed position that it sees
};

template <int TYPE_, int D_, int NMAX_>
struct Shape {
    static constexpr int TYPE = TYPE_, D = D_, NMAX = NMAX_;        // NMAX: query rows of a pass
    static constexpr int MINE = NMAX / GROUPS, PASSES = MINE / 16;        // columns of a softmax thread, 16 at a time
    static constexpr int PARTS = (D + 127) / 128, BLOCKS = D == 64 ? 1 : 2;          // M tiles of O; 64-channel blocks of one
    static constexpr int CH = D / 8 < 16 ? D / 8 : 16;                               // words of a row in a part
    static constexpr int PART = BLOCKS * TS * 128, QP = BLOCKS * NMAX * 128, PB = NMAX / 64 * TS * 128;  // bytes: part of a K or V tile, of Q; term of P
    // slots (parts) of K and of V: what 227 KB hold beside Q and P
    static constexpr int KS = D == 64 ? (NMAX > 64 ? 4 : 5) : D == 256 || NMAX > 64 ? 2 : 3, VS = D == 64 ? (NMAX > 64 ? 3 : 4) : NMAX > 64 ? 1 : 2;
    // A weight's two terms as columns side by side (V is read once for both, 64 rows of 256 channels: 881 us sustained -> 846 for
    // 32 sequences of 8K-64K), or one product after the other into the same sums (fewer columns of O: 128 rows of 128 channels,
    // 100,000 tokens 242 against 260, 64 pieces of prompts 103 against 106).
    static constexpr bool SIDE = PARTS > 1;
    static constexpr uint32_t COL_S = 0, COL_O = 2 * NMAX, PART_O = SIDE ? 2 * NMAX : NMAX, COLS = COL_O + PARTS * PART_O > 256 ? 512 : 256;     // of TMEM
    static constexpr float SLACK = TYPE == SJK_F16 ? 5.0f : 8.0f, UP = TYPE == SJK_F16 ? 10.0f : 0.0f;
};

template <typename S>
struct Shared {
    uint8_t k[S::KS * S::PART], v[S::VS * S::PART], q[S::PARTS * S::QP], pt[2 * S::PB];
    Info<S::NMAX> info[INFO];
    uint32_t live[TILES][4];                // positions of a tile that have a row in the cache
    // of a row (in its group's place, which does not depend on how many rows a pair has): its maximum in use, what its scores are
    // shifted by, and a factor for its sums
    float m[S::NMAX], up[S::NMAX], fac[S::NMAX], red[N_SOFT][32];
    uint64_t k_full[S::KS], k_empty[S::KS], v_full[S::VS], v_empty[S::VS], v_land[S::VS];
    uint64_t s_full[2], s_empty[2], q_full[INFO], p_full, pv_done, o_free, q_empty;
    Cursor start, next;                     // of this segment, and of the one behind it
    uint32_t tiles, pairs, landed;          // gone through so far: where the roles are in their rings
    uint32_t per, tmem;
    int tile, run;
    // pairs of the segment that come again (a bit per group of softmax warps), and of the one that is gone through again: the sum of V's
    // infinities and NaNs in places that all rows see, and the places of the others
    uint32_t again[SEG * GROUPS / 32], any_again;
    float bad[S::PARTS * 128];
    uint32_t edge[EDGES][4], edge_t0[EDGES];
    int edges;
};

// ---- products -----------------------------------------------------------------------------------------------------
// rows of 64 16-bit elements in 128 bytes, 16-byte words swizzled by the row (128-byte swizzle), 8 rows in 1,024 bytes;
// lbo: from one 64-element block to the next where the elements side by side are M or N
SJK_DEV uint64_t swizzled(uint32_t addr, uint32_t lbo) {
    return (uint64_t) ((addr >> 4) & 0x3FFFu) | ((uint64_t) ((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t) (1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// f16 or bf16 operands, 32-bit accumulators, M 128; mn: both operands with M or N side by side in memory
template <int TYPE>
SJK_DEV uint32_t idesc(int n, bool mn) {
    const uint32_t t = TYPE == SJK_BF16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (mn ? 3u << 15 : 0u) | ((uint32_t) (n >> 3) << 17) | (8u << 24);
}
SJK_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u));
}
SJK_DEV bool elected() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
    return r != 0;
}
// a box of 64 channels of one head and some tokens of a page
SJK_DEV void box(uint32_t dst, const CUtensorMap * map, int c, int h, int slot, uint32_t page, uint64_t * bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(map), "r"(c), "r"(h), "r"(slot), "r"(page), "r"(tc::smem_addr(bar)) : "memory");
}
SJK_DEV void ld8(uint32_t t, float * v) {
    uint32_t r[8];
    tc::ld_x8_u(t, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
SJK_DEV bool any_of(int id, bool x) {       // over the 128 threads of a group
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
                 : "=r"(r) : "r"((uint32_t) x), "r"(id), "r"(128) : "memory");
    return r != 0;
}
// N columns of a lane over the warp's lanes: lane c gets column c (with fewer than 32, lanes c + N i as well)
template <bool MAX, int N>
SJK_DEV float columns(const float * v, int lane) {
    float a[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const bool up = lane & (N / 2);
        const float send = up ? v[i] : v[i + N / 2], keep = up ? v[i + N / 2] : v[i], r = __shfl_xor_sync(FULL, send, N / 2);
        a[i] = MAX ? fmaxf(keep, r) : keep + r;
    }
#pragma unroll
    for (int o = N / 4; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const bool up = lane & o;
            const float send = up ? a[i] : a[i + o], keep = up ? a[i + o] : a[i], r = __shfl_xor_sync(FULL, send, o);
            a[i] = MAX ? fmaxf(keep, r) : keep + r;
        }
    float x = a[0];
#pragma unroll
    for (int o = N; o < 32; o <<= 1) {
        const float r = __shfl_xor_sync(FULL, x, o);
        x = MAX ? fmaxf(x, r) : x + r;
    }
    return x;
}
// Waits that give up once and for all: after one that ran out (the status word says so) a role goes on without waiting, so
// that everyone meets the same barriers and the CTA ends.
struct Waiter {
    bool dead = false;
    SJK_DEV void operator()(uint64_t * bar, uint32_t parity) {
        if (!dead && !tc::mbar_wait(bar, parity)) dead = true;
    }
    SJK_DEV void warp(uint64_t * bar, uint32_t parity) {    // by a whole warp
        (*this)(bar, parity);
        dead = __any_sync(FULL, dead);
    }
};

// A part of a V tile of a pair that is gone through again, by a warp: infinities and NaNs become zeros and are noted, per channel or (`edge`
// not negative: the tile's place among those of which rows see different positions) per position; rows that are not live: zeros.
template <typename S>
__device__ __noinline__ void clean_tile(Shared<S> & sm, uint8_t * tile, unsigned live0, unsigned live1, unsigned live2, unsigned live3, int part, int edge) {
    constexpr int LR = S::BLOCKS * 8, RI = 32 / LR;         // lanes of a row, rows at a time
    constexpr uint32_t E = S::TYPE == SJK_F16 ? 0x7C00u : 0x7F80u;
    const int lane = threadIdx.x & 31, wd = lane % LR, d = part * 128 + wd * 8;
    for (int r0 = lane / LR; r0 < TS; r0 += 4 * RI) {
        auto place = [&](int b) { const int rt = r0 + b * RI; return reinterpret_cast<uint4 *>(tile + (wd >> 3) * (TS * 128) + rt * 128 + (((wd ^ rt) & 7) << 4)); };
        uint4 x[4];                         // (their loads are out together)
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = *place(b);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int rt = r0 + b * RI;
            const unsigned live = rt < 32 ? live0 : rt < 64 ? live1 : rt < 96 ? live2 : live3;
            if (!((live >> (rt & 31)) & 1u)) { *place(b) = make_uint4(0u, 0u, 0u, 0u); continue; }
            if (d >= S::D) continue;
            uint32_t w[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
            bool found = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) found |= (w[e] & E) == E || (w[e] & (E << 16)) == E << 16;
            if (!found) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t sh = (e & 1) * 16;
                if (((w[e / 2] >> sh) & E) != E) continue;
                const float2 f = widen2<S::TYPE>(w[e / 2]);
                if (edge < 0) atomicAdd(&sm.bad[d + e], e & 1 ? f.y : f.x);  // (infinities and NaNs alone: any order gives the same)
                w[e / 2] &= ~(0xFFFFu << sh);
            }
            if (edge >= 0) atomicOr(&sm.edge[edge][rt >> 5], 1u << (rt & 31));
            *place(b) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __syncwarp();
}

// What V's infinities and NaNs make of a row of a pair that was gone through again: where it sees some, their sum in place of the finite one. A
// warp; to the output, or (not whole) to `part`.
template <typename S>
__device__ __noinline__ void mark_row(const Params & p, const Shared<S> & sm, int seq, int h, int len, uint64_t mask, int lo, bool whole, int64_t out, float * part) {
    constexpr int NC = S::D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t row = p.rows ? (int64_t) p.rows[seq] : (int64_t) seq;
    const uint32_t * table = row >= 0 && row < (int64_t) p.c.n_rows ? p.c.tables + row * p.c.table_stride : nullptr;
    float x[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) x[c] = sm.bad[32 * c + lane];
    for (int k = 0; k < sm.edges * 4 && table; ++k)
        for (uint32_t bits = sm.edge[k >> 2][k & 3]; bits; bits &= bits - 1u) {
            const uint32_t t = sm.edge_t0[k >> 2] + (uint32_t) (32 * (k & 3) + __ffs((int) bits) - 1);
            if (t >= (uint32_t) len ? !((mask >> (t - (uint32_t) len)) & 1ull) : t < (uint32_t) lo) continue;
            const uint32_t g = t / (uint32_t) p.c.page_tokens, page = table[g];
            if (page >= p.c.n_pages) continue;
            const int64_t at = (int64_t) page * p.c.page_stride + (int64_t) (t - g * (uint32_t) p.c.page_tokens) * p.c.slot_stride + (int64_t) h * p.c.head_stride + lane;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float v = load1(p.c.v, at + 32 * c, S::TYPE);
                if (!(fabsf(v) < INFINITY)) x[c] += v;
            }
        }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (fabsf(x[c]) < INFINITY) continue;
        if (whole) store1(p.out.p, out + 32 * c + lane, S::TYPE, x[c]);
        else part[32 * c + lane] = x[c];
    }
}

// Whether one of a thread's sums (nc columns from addr on, n columns apart where a weight's terms lie side by side) is no number. A function, since
// few calls come here and its registers cost the others 1 to 3 % in line.
template <typename S>
__device__ __noinline__ bool odd_sums(uint32_t addr, int n, int nc, int tl) {
    bool odd = false;
    for (int part = 0; part < S::PARTS; ++part)
        for (int c = 0; c < nc; c += 8) {
            float o[8], y[8];
            ld8(addr + part * S::PART_O + (uint32_t) c, o);
            if (S::SIDE) ld8(addr + part * S::PART_O + (uint32_t) (c + n), y);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) odd |= c + e < nc && part * 128 + tl < S::D && !(fabsf(S::SIDE ? o[e] + y[e] : o[e]) < INFINITY);
        }
    return odd;
}

// Every role's way through the pairs of a segment: all of them, or (again) those of which a sum came out as no number. FIRST: the first
// segment's pairs for the first time, which is all that most calls have.
template <typename S, bool WHOLE, bool FIRST>
SJK_DEV void pass(const Params & p, Shared<S> & sm, bool anew) {
    constexpr int D = S::D, KS = S::KS, VS = S::VS, NMAX = S::NMAX;
    const bool again = !FIRST && anew;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t tmem = sm.tmem;
    Cursor at = sm.start;
    Waiter wait;
    int place = -1;                         // of the pair in the segment
    // whether there is one more
    auto more = [&]() {
        for (++place; at.rem > 0 && place < SEG; ++place) {
            if (!again || ((sm.again[place * GROUPS / 32] >> (place * GROUPS % 32)) & ((1u << GROUPS) - 1u))) return true;
            at.next(p, sm.tile, NMAX, at.take());
        }
        return false;
    };
    if (warp < N_SOFT) {
        // ---- softmax: position 32 (warp % 4) + lane of a tile; four groups of four warps have a quarter of the columns each ----
        const int group = warp >> 2, quarter = warp & 3, bar = 1 + group, tl = quarter * 32 + lane, tg = tid & 127, g0 = group * S::MINE;
        const uint32_t lanes = (uint32_t) (quarter * 32) << 16;
        // scores are positive multiples of the products (the queries' signs are turned for a negative scale)
        const float sc = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * 1.4426950408889634f;
        const float2 sc2 = make_float2(sc, sc);
        float2 l[S::MINE / 2];              // sums of the thread's columns, in pairs
        uint32_t jj = FIRST ? 0u : sm.tiles;                 // tiles so far
        for (int item = FIRST ? 0 : (int) sm.pairs; more(); ++item) {
            const Seq s = at.s;
            const int steps = at.take(), h = at.h;
            const int n = (s.nr + 15) & ~15, all8 = n / 8, most8 = (all8 + GROUPS - 1) / GROUPS;     // columns of the products
            const int n8 = max(0, min(most8, all8 - group * most8)), c0 = group * most8 * 8, nc = n8 * 8;    // octets of columns, first column, their number
            const bool begun = at.st == 0, ended = at.st + steps == s.steps;
            const Info<NMAX> & info = sm.info[item % INFO];
            if (tg < nc) {
                sm.m[g0 + tg] = -INFINITY;
                sm.up[g0 + tg] = 3e38f;     // (no score so far: any is above)
            }
#pragma unroll
            for (int c = 0; c < S::MINE / 2; ++c) l[c] = make_float2(0.0f, 0.0f);
            tc::nbar_sync(bar, 128);
            wait.warp(&sm.q_full[item % INFO], (uint32_t) (item / INFO) & 1u);
            // K octets of columns of tile jj, from cp on (from gp on in the group's places): weights into P, sums into lp
            auto octets_of = [&](auto kk, int cp, int gp, float2 * lp, bool fresh, int step, unsigned live, auto && wait_p) {
                constexpr int K = decltype(kk)::value, N = 8 * K;
                const uint32_t from = tmem + lanes + S::COL_S + (jj & 1u) * NMAX + (uint32_t) cp;
                float x[N];
                const bool all = !partly(p, s, (uint32_t) step * TS), plain = live == FULL && all;
                auto load = [&]() {         // products; those of positions that a row does not see: -inf
#pragma unroll
                    for (int q = 0; q < K; ++q) ld8(from + 8 * q, x + 8 * q);
                    tc::wait_ld();
                    if (!plain) {
                        const uint32_t t = (uint32_t) step * TS + (uint32_t) tl;
                        uint32_t seen = (live >> lane) & 1u ? FULL : 0u;
                        if (seen && !all) {
                            if (t >= (uint32_t) s.len) {
                                const uint32_t k = t - (uint32_t) s.len;
                                seen = 0u;
#pragma unroll
                                for (int c = 0; c < N; ++c) seen |= (uint32_t) ((info.mask[cp + c] >> k) & 1ull) << c;
                            } else if (p.window) {
                                seen = 0u;
#pragma unroll
                                for (int c = 0; c < N; ++c) seen |= (t >= (uint32_t) info.lo[cp + c] ? 1u : 0u) << c;
                            }
                        }
#pragma unroll
                        for (int c = 0; c < N; ++c)
                            if (!((seen >> c) & 1u)) x[c] = -INFINITY;
                    }
                };
                auto shift = [&]() {        // to exponents of the weights
#pragma unroll
                    for (int q = 0; q < N / 4; ++q) {
                        const float4 u = *reinterpret_cast<const float4 *>(&sm.up[gp + q * 4]);
                        const float2 a = tc::num::fma2(make_float2(x[4 * q], x[4 * q + 1]), sc2, make_float2(u.x, u.y));
                        const float2 b = tc::num::fma2(make_float2(x[4 * q + 2], x[4 * q + 3]), sc2, make_float2(u.z, u.w));
                        x[4 * q] = a.x; x[4 * q + 1] = a.y; x[4 * q + 2] = b.x; x[4 * q + 3] = b.y;
                    }
                };
                load();
                bool renew = fresh;
                if (!fresh) {
                    shift();
                    float top = x[0];
#pragma unroll
                    for (int c = 1; c + 1 < N; c += 2) top = fmaxf(fmaxf(top, x[c]), x[c + 1]);
                    top = fmaxf(top, x[N - 1]);
                    renew = any_of(bar, top > S::SLACK + S::UP);
                    if (renew) load();
                }
                if (renew) {                // a row's first tile, or a score too far above the maximum in use: a new one
                    const float top = columns<true, N>(x, lane);
                    sm.red[warp][lane] = top;
                    tc::nbar_sync(bar, 128);
                    if (tg < N) {
                        const float old = sm.m[gp + tg];
                        float m = -INFINITY;
#pragma unroll
                        for (int w = 0; w < 4; ++w) m = fmaxf(m, sm.red[group * 4 + w][tg]);
                        m = fmaxf(m * sc, old);
                        sm.fac[gp + tg] = m == old ? 1.0f : tc::num::ex2(old - m);
                        sm.m[gp + tg] = m;
                        sm.up[gp + tg] = m == -INFINITY ? 3e38f : S::UP - m;
                    }
                    tc::nbar_sync(bar, 128);
                    shift();
                    if (!fresh) {
#pragma unroll
                        for (int c = 0; c < N / 2; ++c) {
                            lp[c].x *= sm.fac[gp + 2 * c];
                            lp[c].y *= sm.fac[gp + 2 * c + 1];
                        }
                        wait_p();           // O has tiles of this pair
#pragma unroll 1
                        for (int part = 0; part < S::PARTS; ++part)
#pragma unroll 1
                            for (int q = 0; q < K; ++q) {
                                const uint32_t addr = tmem + lanes + S::COL_O + part * S::PART_O + (uint32_t) (cp + q * 8);
                                float o[8], y[8];
                                ld8(addr, o);
                                if (S::SIDE) ld8(addr + (uint32_t) n, y);
                                tc::wait_ld();
                                uint32_t r[8], z[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const float f = sm.fac[gp + q * 8 + e];
                                    r[e] = __float_as_uint(o[e] * f);
                                    if (S::SIDE) z[e] = __float_as_uint(y[e] * f);
                                }
                                tc::st_x8(addr, r);
                                if (S::SIDE) tc::st_x8(addr + (uint32_t) n, z);
                            }
                        tc::wait_st();
                    }
                }
                uint32_t hi[N / 2], lw[N / 2];
#pragma unroll
                for (int c = 0; c < N / 2; ++c) {
                    const float2 a = make_float2(tc::num::ex2(x[2 * c]), tc::num::ex2(x[2 * c + 1]));
                    lp[c] = tc::num::add2(lp[c], a);
                    hi[c] = pack2<S::TYPE>(a.x, a.y);
                    const float2 r = tc::num::fma2(widen2<S::TYPE>(hi[c]), make_float2(-1.0f, -1.0f), a);
                    lw[c] = pack2<S::TYPE>(r.x, r.y);
                }
                wait_p();
#pragma unroll
                for (int q = 0; q < K; ++q) {
                    const uint32_t h8 = (uint32_t) (cp >> 3) + (uint32_t) q;
                    auto place = [&](uint32_t o8) { return (o8 >> 3) * (TS * 128) + (uint32_t) tl * 128u + (((o8 ^ (uint32_t) tl) & 7u) << 4); };
                    const uint32_t ph = place(h8), pl = S::SIDE ? place(h8 + (uint32_t) (n >> 3)) : ph + S::PB;
                    *reinterpret_cast<uint4 *>(&sm.pt[ph]) = make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
                    *reinterpret_cast<uint4 *>(&sm.pt[pl]) = make_uint4(lw[4 * q], lw[4 * q + 1], lw[4 * q + 2], lw[4 * q + 3]);
                }
            };
            for (int i = 0; i < steps; ++i, ++jj) {
                const int step = s.step0 + at.st + i;
                wait.warp(&sm.s_full[jj & 1u], (jj >> 1) & 1u);
                tc::fence_after_sync();
                const unsigned live = sm.live[jj % TILES][quarter];
                bool free_p = jj == 0;      // the products with the tile before are done
                auto wait_p = [&]() {
                    if (free_p) return;
                    free_p = true;
                    wait.warp(&sm.pv_done, (jj - 1) & 1u);
                    tc::fence_after_sync();
                };
#pragma unroll
                for (int ps = 0; ps < S::PASSES; ++ps) {
                    const int m8 = n8 - 2 * ps;
                    if (m8 == 1) octets_of(Int<1>(), c0 + 16 * ps, g0 + 16 * ps, l + 8 * ps, i == 0, step, live, wait_p);
                    else if (m8 > 1) octets_of(Int<2>(), c0 + 16 * ps, g0 + 16 * ps, l + 8 * ps, i == 0, step, live, wait_p);
                }
                wait_p();                   // (no thread falls behind a phase)
                tc::fence_proxy_async();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&sm.s_empty[jj & 1u]);
                    tc::mbar_arrive(&sm.p_full);
                }
            }
            // the pair's output, or its partial
            wait.warp(&sm.pv_done, (jj - 1) & 1u);
            tc::fence_after_sync();
            const bool whole = begun && ended;
            const int64_t slot = ((int64_t) blockIdx.x * 2 + (begun ? 1 : 0)) * NMAX;
#pragma unroll
            for (int ps = 0; ps < S::PASSES; ++ps) {
                constexpr int N = 16;
                float v[N];
#pragma unroll
                for (int c = 0; c < N / 2; ++c) { v[2 * c] = l[8 * ps + c].x; v[2 * c + 1] = l[8 * ps + c].y; }
                const float sum = columns<false, N>(v, lane);
                if (ps) tc::nbar_sync(bar, 128);
                sm.red[warp][lane] = sum;
                tc::nbar_sync(bar, 128);
                const int c = 16 * ps + tg;
                if (tg < N && c < nc) {
                    const float (* red)[32] = &sm.red[group * 4];
                    const float all = (red[0][tg] + red[1][tg]) + (red[2][tg] + red[3][tg]);
                    sm.fac[g0 + c] = all == 0.0f ? 0.0f : 1.0f / all;
                    if (!whole) *reinterpret_cast<float2 *>(p.ml + (slot + c0 + c) * 2) = make_float2(sm.m[g0 + c], all);
                }
            }
            if (tid == 0 && begun && !ended)
                p.split[blockIdx.x] = make_int4(at.seq, h, sm.run, (int) ((at.base + (uint32_t) (s.steps + OV) - 1u) / sm.per));
            // f(column, sum of the thread's channel of this part) over the group's rows
            auto sums = [&](int part, auto && f) {
#pragma unroll 1
                for (int c = 0; c < nc; c += 8) {
                    float o[8], y[8];
                    const uint32_t addr = tmem + lanes + S::COL_O + part * S::PART_O + (uint32_t) (c0 + c);
                    ld8(addr, o);
                    if (S::SIDE) ld8(addr + (uint32_t) n, y);
                    tc::wait_ld();
                    if (part * 128 + tl < D)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (c0 + c + e < s.nr) f(c + e, S::SIDE ? o[e] + y[e] : o[e]);
                }
            };
            // Rows of a group with a sum that is no number are stored the second time (there: no others); the first time as well, unless
            // outputs lie over the queries, which the second one reads.
            tc::nbar_sync(bar, 128);
            const uint32_t bit = 1u << (place * GROUPS % 32 + group);
            uint32_t & word = sm.again[place * GROUPS / 32];
            const bool mine = again ? (word & bit) != 0u : !p.over || !any_of(bar, odd_sums<S>(tmem + lanes + S::COL_O + (uint32_t) c0, n, min(nc, s.nr - c0), tl));
            float * part0 = p.part + slot * D;
            bool odd = !mine;
            if (mine) {
#pragma unroll 1
                for (int part = 0; part < S::PARTS; ++part) {
                    const int d = part * 128 + tl;
                    sums(part, [&](int c, float x) {
                        odd |= !(fabsf(x) < INFINITY);
                        if (whole) store1(p.out.p, info.out[c0 + c] + d, S::TYPE, x * sm.fac[g0 + c]);
                        else part0[(c0 + c) * D + d] = x;
                    });
                }
            }
            __syncwarp();
            if (!again) {
                if (any_of(bar, odd) && tg == 0) {
                    atomicOr(&word, bit);
                    sm.any_again = 1u;
                }
            } else if (mine) {
                tc::nbar_sync(bar, 128);
                for (int c = quarter; c < nc && c0 + c < s.nr; c += 4)
                    mark_row<S>(p, sm, at.seq, h, s.len, info.mask[c0 + c], info.lo[c0 + c], whole, info.out[c0 + c], part0 + (c0 + c) * D);
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sm.o_free);
            tc::nbar_sync(bar, 128);        // the factors have been read
            at.next(p, sm.tile, NMAX, steps);
        }
    } else if (warp < W_MMA) {
        // ---- K, and V ----
        const bool is_v = warp == N_SOFT + 1;
        const int slots = is_v ? VS : KS;
        uint64_t * full = is_v ? sm.v_full : sm.k_full, * empty = is_v ? sm.v_empty : sm.k_empty;
        uint8_t * ring = is_v ? sm.v : sm.k;
        uint32_t jj = FIRST ? 0u : sm.tiles, pp = jj * S::PARTS, told = pp;     // tiles; parts asked for, and announced (not WHOLE)
        auto tell = [&](uint32_t upto) {    // copies of the parts before `upto` have landed
            tc::fence_proxy_async();
            __syncwarp();
            for (; told < upto; ++told)
                if (lane == 0) tc::mbar_arrive(&full[told % slots]);
        };
        // WHOLE: a part of a V tile whose dead rows (that came with a box, or came not) are to be zeros
        struct Mend { bool on; int slot, part, edge; unsigned dead[4]; } m = {};
        uint32_t landed = FIRST ? 0u : sm.landed;            // parity of every slot's v_land
        int item = FIRST ? 0 : (int) sm.pairs, edges = 0;
        auto mend_box = [&]() {             // once it has landed
            m.on = false;
            wait.warp(&sm.v_land[m.slot], (landed >> m.slot) & 1u);
            landed ^= 1u << m.slot;
            uint8_t * dst = ring + m.slot * S::PART;
            constexpr int LR = S::BLOCKS * 8, RI = 32 / LR;         // lanes of a row, rows at a time
            const int wd = lane % LR;
            if (again) clean_tile<S>(sm, dst, ~m.dead[0], ~m.dead[1], ~m.dead[2], ~m.dead[3], m.part, m.edge);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                for (int r0 = 0; !again && r0 < 32 && m.dead[g] >> r0; r0 += RI) {
                    const int r = r0 + lane / LR, rt = 32 * g + r;
                    if ((m.dead[g] >> r) & 1u) *reinterpret_cast<uint4 *>(dst + (wd >> 3) * (TS * 128) + rt * 128 + (((wd ^ rt) & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&full[m.slot]);
        };
        auto flush = [&] {
            if (WHOLE) {
                if (m.on) mend_box();
            } else {
                tc::cp_async_wait_group<0>();
                tell(pp);
            }
        };
        for (; more(); ++item) {
            const Seq s = at.s;
            const int steps = at.take();
            const bool clean = again && is_v;
            if (clean) {                    // the notes of the pair before have been read
                flush();
                if (item > 0) wait.warp(&sm.o_free, (uint32_t) (item - 1) & 1u);
                for (int d = lane; d < S::PARTS * 128; d += 32) sm.bad[d] = 0.0f;
                if (lane < EDGES * 4) sm.edge[lane >> 2][lane & 3] = 0u;
                edges = 0;
                if (lane == 0) sm.edges = 0;
                __syncwarp();
            }
            const int64_t row = p.rows ? (int64_t) p.rows[at.seq] : (int64_t) at.seq;
            const uint32_t * table = row >= 0 && row < (int64_t) p.c.n_rows ? p.c.tables + row * p.c.table_stride : nullptr;
            if (!table && lane == 0) flag();
            const uint32_t lo0 = low_of(p, s);
            for (int i = 0; i < steps; ++i, ++jj) {
                const uint32_t t0 = (uint32_t) (s.step0 + at.st + i) * TS;
                // the tile's live positions (a lane looks up every 32nd) and their rows, and (WHOLE) the lane's box: all look-ups
                // are out before the first is used
                uint32_t place[5], page[5];
                const uint32_t mine = (uint32_t) (lane / S::BLOCKS) * (uint32_t) p.box;
#pragma unroll
                for (int u = 0; u < 5; ++u) {
                    const uint32_t t = u < 4 ? t0 + (uint32_t) (32 * u + lane) : t0 + mine;
                    const bool on = u < 4 ? t < s.hi && t >= lo0 : WHOLE && mine < TS && t < s.hi && t + (uint32_t) p.box > lo0;
                    const uint32_t g = p.page_shift >= 0 ? t >> p.page_shift : t / (uint32_t) p.c.page_tokens;
                    place[u] = t - g * (uint32_t) p.c.page_tokens;
                    page[u] = on && table ? table[g] : SJKVARN_NO_BLOCK;
                }
                unsigned live[4], dead[4];
                int64_t off[4];             // -1: none
                const int a16 = first16(p, s, t0), b16 = end16(s, t0);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (page[u] >= p.c.n_pages && page[u] != SJKVARN_NO_BLOCK) flag();
                    off[u] = page[u] < p.c.n_pages ? (int64_t) page[u] * p.c.page_stride + (int64_t) place[u] * p.c.slot_stride : -1;
                    const int g16 = (32 * u + lane) >> 4;
                    live[u] = __ballot_sync(FULL, off[u] >= 0);
                    dead[u] = __ballot_sync(FULL, WHOLE && is_v && off[u] < 0 && g16 >= a16 && g16 < b16);     // (copies fill theirs with zeros)
                    if (!is_v && lane == 0) sm.live[jj % TILES][u] = live[u];
                }
                int edge = -1;
                if (clean) {
                    if (partly(p, s, t0)) {
                        edge = edges++;
                        if (lane == 0) { sm.edge_t0[edge] = t0; sm.edges = edges; }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) dead[u] = ~live[u];
                }
                const bool mend = WHOLE && (clean || (dead[0] | dead[1] | dead[2] | dead[3]) != 0u);
                const bool asks = WHOLE && page[4] < p.c.n_pages;
                const uint32_t tx = WHOLE ? (uint32_t) __popc(__ballot_sync(FULL, asks)) * (uint32_t) p.box * 128u : 0u;
#pragma unroll 1
                for (int part = 0; part < S::PARTS; ++part, ++pp) {
                    const int slot = (int) (pp % (uint32_t) slots);
                    if (pp >= (uint32_t) slots) {
                        const uint32_t parity = (pp / (uint32_t) slots - 1u) & 1u;
                        if ((!WHOLE || m.on) && !wait.dead && !__all_sync(FULL, tc::mbar_test(&empty[slot], parity))) {
                            // nothing more to ask for now: hand on what has been
                            if (WHOLE) mend_box();
                            else {
                                tc::cp_async_wait_group<0>();
                                tell(pp);
                            }
                        }
                        if (WHOLE && wait.dead && m.on) mend_box();
                        wait.warp(&empty[slot], parity);
                    }
                    uint8_t * dst = ring + slot * S::PART;
                    if constexpr (WHOLE) {
                        uint64_t * bar = mend ? &sm.v_land[slot] : &full[slot];
                        if (lane == 0) tc::mbar_expect_tx(bar, tx);
                        __syncwarp();
                        if (asks)
                            box(tc::smem_addr(dst) + (uint32_t) (lane % S::BLOCKS) * (TS * 128) + mine * 128u, &p.maps[is_v ? 1 : 0],
                                part * 128 + (lane % S::BLOCKS) * 64, at.h, (int) place[4], page[4], bar);
                        if (m.on) mend_box();           // the one before, while this one is on its way
                    }
                    if (mend) {
                        m.on = true;
                        m.slot = slot;
                        m.part = part;
                        m.edge = edge;
#pragma unroll
                        for (int u = 0; u < 4; ++u) m.dead[u] = dead[u];
                    }
                    if constexpr (!WHOLE) {
                        const uint16_t * base = static_cast<const uint16_t *>(is_v ? p.c.v : p.c.k) + (int64_t) at.h * p.c.head_stride + part * 128;
#pragma unroll
                        for (int u = 0; u < 4; ++u)
#pragma unroll 4
                            for (int k = 0; k < S::CH; ++k) {
                                const int w = k * 32 + lane, r = w / S::CH, c = w - r * S::CH;
                                const int64_t o = __shfl_sync(FULL, off[u], r);
                                tc::cp_async16(dst + (c >> 3) * (TS * 128) + (32 * u + r) * 128 + (((c ^ r) & 7) << 4), base + (o >= 0 ? o : 0) + c * 8, o >= 0 ? 16u : 0u);
                            }
                        tc::cp_async_commit();
                        if (clean) {
                            tc::cp_async_wait_group<0>();
                            __syncwarp();
                            clean_tile<S>(sm, dst, live[0], live[1], live[2], live[3], part, edge);
                            tell(pp + 1);
                            continue;
                        }
                        if (slots == 1) tc::cp_async_wait_group<0>();
                        else if (slots == 2) tc::cp_async_wait_group<1>();
                        else if (slots == 3) tc::cp_async_wait_group<2>();
                        else tc::cp_async_wait_group<3>();
                        const uint32_t flight = slots < 4 ? (uint32_t) slots - 1u : 3u;      // parts still on their way
                        if (pp + 1 > flight) tell(pp + 1 - flight);
                    }
                }
            }
            at.next(p, sm.tile, NMAX, steps);
        }
        flush();
        if (is_v && lane == 0) sm.landed = landed;
    } else if (warp == W_MMA) {
        // ---- products: the warp stays together and one thread issues, so that descriptors are the same for all lanes ----
        const bool leader = elected();
        const uint32_t ka = tc::smem_addr(sm.k), va = tc::smem_addr(sm.v), qa = tc::smem_addr(sm.q), pa = tc::smem_addr(sm.pt);
        const uint32_t tm = __shfl_sync(FULL, tmem, 0);
        uint32_t jj = FIRST ? 0u : sm.tiles, kp = jj * S::PARTS, vp = kp;       // tiles; parts of K and of V
        int pend_n = 0, pend_a = 0, pend_b = 0, items = FIRST ? 0 : (int) sm.pairs;
        bool pend = false, pend_first = false;               // a tile whose second product is to come
        auto second = [&](uint32_t j) {                      // O^T += V^T P of tile j
            if (pend_first && items > 1) wait.warp(&sm.o_free, (uint32_t) (items - 2) & 1u);
            wait.warp(&sm.p_full, j & 1u);
            const uint32_t id = idesc<S::TYPE>(S::SIDE ? 2 * pend_n : pend_n, true);
#pragma unroll 1
            for (int part = 0; part < S::PARTS; ++part, ++vp) {
                const uint32_t slot = vp % VS;
                wait.warp(&sm.v_full[slot], (vp / VS) & 1u);
                tc::fence_after_sync();
                const uint64_t a = swizzled(va + slot * S::PART, D == 64 ? 0u : TS * 128u), b = swizzled(pa, TS * 128u);
                const uint32_t d = tm + S::COL_O + part * S::PART_O;
                if (leader && !wait.dead) {
                    constexpr int TERMS = S::SIDE ? 1 : 2;
                    if (pend_b - pend_a == TS / 16) {
#pragma unroll
                        for (int k = 0; k < TERMS * TS / 16; ++k)
                            mma_ss(d, a + (uint64_t) ((k & 7) * 2048 >> 4), b + (uint64_t) (((k >> 3) * S::PB + (k & 7) * 2048) >> 4), id, pend_first && k == 0 ? 0u : 1u);
                    } else {
#pragma unroll 1
                        for (int k = pend_a; k < pend_b; ++k) {
                            mma_ss(d, a + (uint64_t) (k * 2048 >> 4), b + (uint64_t) (k * 2048 >> 4), id, pend_first && k == pend_a ? 0u : 1u);
                            if (!S::SIDE) mma_ss(d, a + (uint64_t) (k * 2048 >> 4), b + (uint64_t) ((S::PB + k * 2048) >> 4), id, 1u);
                        }
                    }
                    tc::mma_commit(&sm.v_empty[slot]);
                    if (part + 1 == S::PARTS) tc::mma_commit(&sm.pv_done);
                }
                __syncwarp();
            }
        };
        while (more()) {
            const int steps = __shfl_sync(FULL, at.take(), 0), n = __shfl_sync(FULL, (at.s.nr + 15) & ~15, 0);
            const uint32_t id = idesc<S::TYPE>(n, false);
            if (pend) second(jj - 1);       // the pair's end does not wait for the next one's queries
            pend = false;
            wait.warp(&sm.q_full[items % INFO], (uint32_t) (items / INFO) & 1u);
            for (int i = 0; i < steps; ++i, ++jj) {
                const uint32_t b = jj & 1u;
                if (jj >= 2) wait.warp(&sm.s_empty[b], ((jj >> 1) - 1u) & 1u);
#pragma unroll 1
                for (int part = 0; part < S::PARTS; ++part, ++kp) {
                    const uint32_t slot = kp % KS;
                    wait.warp(&sm.k_full[slot], (kp / KS) & 1u);
                    tc::fence_after_sync();
                    const uint64_t ad = swizzled(ka + slot * S::PART, 16u), bd = swizzled(qa + part * S::QP, 16u);
                    const uint32_t d = tm + S::COL_S + b * NMAX;
                    if (leader && !wait.dead) {
#pragma unroll
                        for (int k = 0; k < (D < 128 ? D : 128) / 16; ++k)
                            mma_ss(d, ad + (uint64_t) (((k >> 2) * TS * 128 + (k & 3) * 32) >> 4), bd + (uint64_t) (((k >> 2) * NMAX * 128 + (k & 3) * 32) >> 4), id,
                                   part || k ? 1u : 0u);
                        tc::mma_commit(&sm.k_empty[slot]);
                        if (part + 1 == S::PARTS) {
                            if (i + 1 == steps) tc::mma_commit(&sm.q_empty);
                            tc::mma_commit(&sm.s_full[b]);
                        }
                    }
                    __syncwarp();
                }
                if (pend) second(jj - 1);
                pend = true;
                pend_n = n;
                pend_a = first16(p, at.s, (uint32_t) (at.s.step0 + at.st + i) * TS);
                pend_b = end16(at.s, (uint32_t) (at.s.step0 + at.st + i) * TS);
                pend_first = i == 0;
                if (i == 0) ++items;
            }
            at.next(p, sm.tile, NMAX, steps);
        }
        if (pend) second(jj - 1);
        if (lane == 0) {
            sm.tiles = jj;
            sm.pairs = (uint32_t) items;
            if (!again) sm.next = at;
        }
    } else {
        // ---- queries, and what the rows see ----
        for (int item = FIRST ? 0 : (int) sm.pairs; more(); ++item) {
            const Seq s = at.s;
            const int steps = at.take(), n = (s.nr + 15) & ~15;
            if (item > 0) wait.warp(&sm.q_empty, (uint32_t) (item - 1) & 1u);
            Info<NMAX> & info = sm.info[item % INFO];
            int64_t from[NMAX / 32];
#pragma unroll
            for (int u = 0; u < NMAX / 32; ++u) {
                const int r = 32 * u + lane;
                from[u] = -1;
                if (r >= n) continue;
                uint64_t mask = 0ull;
                int lo = 0x7FFFFFFF;
                if (r < s.nr) {
                    const int j = (s.row0 + r) / p.grp, g = (s.row0 + r) - j * p.grp, head = at.h * p.grp + g;
                    mask = p.masks ? p.masks[s.first + j] : (2ull << j) - 1ull;
                    if (s.count < 64) mask &= (1ull << s.count) - 1ull;
                    lo = 0;
                    if (p.window) {         // the last `window` of the committed and the drafted ones
                        int drop = __popcll(mask) - p.window;
                        for (; drop > 0; --drop) mask &= mask - 1ull;
                        const int keep = p.window - __popcll(mask);
                        lo = s.len > keep ? s.len - keep : 0;
                    }
                    from[u] = (int64_t) (s.first + j) * p.q.row_stride + (int64_t) head * p.q.head_stride;
                    info.out[r] = (int64_t) (s.first + j) * p.out.row_stride + (int64_t) head * p.out.head_stride;
                }
                info.mask[r] = mask;
                info.lo[r] = lo;
            }
#pragma unroll
            for (int u = 0; u < NMAX / 32; ++u)
                if (32 * u < n)
#pragma unroll 4
                    for (int k = 0; k < D / 8; ++k) {
                        const int w = k * 32 + lane, r = w / (D / 8), c = w - r * (D / 8);
                        const int64_t o = __shfl_sync(FULL, from[u], r);
                        tc::cp_async16(sm.q + (c >> 3) * (NMAX * 128) + (32 * u + r) * 128 + (((c ^ r) & 7) << 4),
                                       static_cast<const uint16_t *>(p.q.p) + (o >= 0 ? o : 0) + c * 8, o >= 0 ? 16u : 0u);
                    }
            tc::cp_async_wait_all();
            if (p.scale <= 0.0f) {          // scores of the other sign, or none
                __syncwarp();
                for (int w = lane; w < S::PARTS * S::QP / 16; w += 32) {
                    uint4 & x = reinterpret_cast<uint4 *>(sm.q)[w];
                    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u, keep = p.scale < 0.0f ? FULL : 0u;
                    x = make_uint4((x.x ^ flip) & keep, (x.y ^ flip) & keep, (x.z ^ flip) & keep, (x.w ^ flip) & keep);
                }
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sm.q_full[item % INFO]);
            at.next(p, sm.tile, NMAX, steps);
        }
    }
}
// What follows a segment's first turn: its pairs that come again, and the segments behind it. A function of its own and not inlined: as a second
// turn of the same code it cost the first one 3 to 20 % (registers).
template <typename S, bool WHOLE>
__device__ __noinline__ void rest(const Params & p, Shared<S> & sm) {
    const int tid = threadIdx.x;
    for (bool again = sm.any_again;; again = !again && sm.any_again) {
        if (!again) {
            if (sm.next.rem <= 0) return;
            __syncthreads();                // all have looked at what is made new here
            if (tid == 0) { sm.start = sm.next; sm.any_again = 0u; }
            if (tid < SEG * GROUPS / 32) sm.again[tid] = 0u;
            __syncthreads();
        }
        pass<S, WHOLE, false>(p, sm, again);
        __syncthreads();
    }
}

template <typename S, bool WHOLE>
__global__ void __launch_bounds__(NT, 1) tree_kernel(const __grid_constant__ Params p) {
    constexpr int KS = S::KS, VS = S::VS, NMAX = S::NMAX;
    extern __shared__ uint8_t raw[];
    Shared<S> & sm = *reinterpret_cast<Shared<S> *>(raw + ((1024u - (tc::smem_addr(raw) & 1023u)) & 1023u));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < KS; ++i) { tc::mbar_init(&sm.k_full[i], 1); tc::mbar_init(&sm.k_empty[i], 1); }
        for (int i = 0; i < VS; ++i) { tc::mbar_init(&sm.v_full[i], 1); tc::mbar_init(&sm.v_empty[i], 1); tc::mbar_init(&sm.v_land[i], 1); }
        for (int i = 0; i < 2; ++i) { tc::mbar_init(&sm.s_full[i], 1); tc::mbar_init(&sm.s_empty[i], N_SOFT); }
        tc::mbar_init(&sm.p_full, N_SOFT);
        tc::mbar_init(&sm.pv_done, 1);
        tc::mbar_init(&sm.o_free, N_SOFT);
        for (int i = 0; i < INFO; ++i) tc::mbar_init(&sm.q_full[i], 1);
        tc::mbar_init(&sm.q_empty, 1);
        tc::mbar_fence_init();
        sm.any_again = 0u;
    }
    if (tid < SEG * GROUPS / 32) sm.again[tid] = 0u;
    if (warp == W_MMA) { tc::tmem_alloc(&sm.tmem, S::COLS); tc::tmem_relinquish(); }
    pdl_wait();
    pdl_release();
    // As many lists as the sequence with the most rows has tiles, side by side in the grid, and where the CTA's run begins in
    // its own: units of all sequences, a block of them per lane.
    if (warp == 0) {
        const int block = (p.n_seq + 31) / 32;
        int tiles = 1;
        uint32_t mine = 0;
        for (int i = 0; i < block; ++i)
            if (lane * block + i < p.n_seq) tiles = max(tiles, tiles_of(p, lane * block + i, NMAX));
        tiles = (int) __reduce_max_sync(FULL, (unsigned) tiles);
        const int tile = blockIdx.x % tiles, run = blockIdx.x / tiles, wl = gridDim.x / tiles;
        for (int i = 0; i < block; ++i)
            if (lane * block + i < p.n_seq) mine += units_of(p, seq_of(p, lane * block + i, tile, NMAX));
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(FULL, incl, o);
            if (lane >= o) incl += y;
        }
        const uint32_t list = __shfl_sync(FULL, incl, 31);
        const uint32_t per = (list + (uint32_t) wl - 1u) / (uint32_t) wl;        // (at least a unit, where there is one)
        const int64_t o = (int64_t) run * per;
        Cursor c = {};
        if (o < list && run < wl) {
            const uint32_t off = (uint32_t) o;
            c.rem = (int) (o + per < list ? per : list - off);
            const int g = __ffs(__ballot_sync(FULL, incl > off)) - 1;
            c.base = __shfl_sync(FULL, incl - mine, g);
            c.seq = g * block;
            for (;; ++c.seq) {              // (the block's last sequence at the latest: its sum is above off)
                c.s = seq_of(p, c.seq, tile, NMAX);
                const uint32_t u = units_of(p, c.s);
                if (c.base + u > off) break;
                c.base += u;
            }
            c.h = (int) ((off - c.base) / (uint32_t) (c.s.steps + OV));
            c.base += (uint32_t) c.h * (uint32_t) (c.s.steps + OV);
            const int in = (int) (off - c.base);
            c.st = in > OV ? in - OV : 0;
            if (in < OV) c.rem -= OV - in;  // no steps where the run has only units before a first step
        }
        if (lane == 0) {
            sm.start = c;
            sm.per = per;
            sm.tile = tile;
            sm.run = run;
            p.split[blockIdx.x] = make_int4(-1, 0, 0, 0);
            if (blockIdx.x == 0) p.split[gridDim.x] = make_int4(tiles, 0, 0, 0);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    pass<S, WHOLE, true>(p, sm, false);
    __syncthreads();
    if (sm.any_again || sm.next.rem > 0) rest<S, WHOLE>(p, sm);
    tc::fence_before_sync();
    __syncthreads();
    if (warp == W_MMA) tc::tmem_dealloc(sm.tmem, S::COLS);
}

// Joins the runs of a split pair in order. grid: CTAs of the kernel before, rows in groups of 8, a warp each.
template <int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ Params p, int type, int nmax) {
    constexpr int NV = (D / 4 + 31) / 32;   // 16-byte words of a lane
    pdl_wait();
    pdl_release();
    const int4 e = p.split[blockIdx.x];
    if (e.x < 0) return;
    const int tiles = p.split[gridDim.x].x, tile = blockIdx.x % tiles, lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
    const Seq s = seq_of(p, e.x, tile, nmax);
    if (r >= s.nr) return;
    auto slot_of = [&](int w) { return (((int64_t) w * tiles + tile) * 2 + (w == e.z ? 1 : 0)) * nmax + r; };
    float top = -INFINITY, sum = 0.0f;
    for (int w0 = e.z; w0 <= e.w; w0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (w0 + lane <= e.w) ml = *reinterpret_cast<const float2 *>(p.ml + slot_of(w0 + lane) * 2);
        float t = ml.x;
#pragma unroll
        for (int x = 16; x; x >>= 1) t = fmaxf(t, __shfl_xor_sync(FULL, t, x));
        t = fmaxf(t, top);
        const float use = t == -INFINITY ? 0.0f : t;
        sum = sum * tc::num::ex2(top - use) + ml.y * tc::num::ex2(ml.x - use);
        top = t;
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(FULL, sum, x);
    const float use = top == -INFINITY ? 0.0f : top, inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float4 o[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int w = e.z; w <= e.w; ++w) {
        const int64_t at = slot_of(w);
        const float f = tc::num::ex2(p.ml[at * 2] - use);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (32 * v + lane < D / 4) {
                const float4 x = reinterpret_cast<const float4 *>(p.part + at * D)[32 * v + lane];
                // (an infinity stays one, however small the run's share)
                auto add = [&](float a, float y) { return fabsf(a) < INFINITY ? fmaf(a, f, y) : a + y; };
                o[v].x = add(x.x, o[v].x); o[v].y = add(x.y, o[v].y);
                o[v].z = add(x.z, o[v].z); o[v].w = add(x.w, o[v].w);
            }
    }
    const int j = (s.row0 + r) / p.grp, head = e.y * p.grp + (s.row0 + r) - j * p.grp;
    const int64_t dst = (int64_t) (s.first + j) * p.out.row_stride + (int64_t) head * p.out.head_stride;
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (32 * v + lane < D / 4) {
            const int d = 4 * (32 * v + lane);
            store1(p.out.p, dst + d, type, o[v].x * inv);
            store1(p.out.p, dst + d + 1, type, o[v].y * inv);
            store1(p.out.p, dst + d + 2, type, o[v].z * inv);
            store1(p.out.p, dst + d + 3, type, o[v].w * inv);
        }
}

// Maps of the cache's K and V as boxes of `box` tokens; false where its strides do not allow them.
bool maps_of(Params * p) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void * f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return false;
    const sjk_kv16 & c = p->c;
    const cuuint64_t dims[4] = {(cuuint64_t) c.head_dim, (cuuint64_t) c.n_head_kv, (cuuint64_t) c.page_tokens, (cuuint64_t) c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t) c.head_stride * 2, (cuuint64_t) c.slot_stride * 2, (cuuint64_t) c.page_stride * 2};
    const cuuint32_t sizes[4] = {64u, 1u, (cuuint32_t) p->box, 1u}, ones[4] = {1u, 1u, 1u, 1u};
    for (int i = 0; i < 2; ++i)
        if (encode(&p->maps[i], c.type == SJK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, i ? c.v : c.k, dims, strides, sizes, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

template <typename S, bool WHOLE>
int tree_launch(const Params & p, sjk_stream st) {
    constexpr size_t bytes = sizeof(Shared<S>) + 1024;
    static_assert(bytes <= 227 * 1024, "shared memory of a CTA");
    if (smem_limit<tree_kernel<S, WHOLE>>(bytes)) return SJK_ERR_DEVICE;
    return launch(tree_kernel<S, WHOLE>, dim3(CTAS), dim3(NT), bytes, st, p);
}

template <typename S>
int run(Params & p, sjk_stream st) {
    // pages of a multiple of 8 tokens come as boxes: as many tokens of a page as end where a tile's rows do
    p.box = 128;
    while (p.box > 1 && p.c.page_tokens % p.box) p.box >>= 1;
    const int rc = p.box >= 8 && maps_of(&p) ? tree_launch<S, true>(p, st) : tree_launch<S, false>(p, st);
    if (rc) return rc;
    const int rows = p.nodes * p.grp < S::NMAX ? p.nodes * p.grp : S::NMAX;
    return launch(tree_merge_kernel<S::D>, dim3(CTAS, (unsigned) ((rows + 7) / 8)), dim3(256), 0, st, p, S::TYPE, S::NMAX);
}

template <int TYPE>
int run_dim(Params & p, int nmax, sjk_stream st) {
    switch (p.c.head_dim) {
        case 64: return nmax > 64 ? run<Shape<TYPE, 64, 128>>(p, st) : run<Shape<TYPE, 64, 64>>(p, st);
        case 96: return nmax > 64 ? run<Shape<TYPE, 96, 128>>(p, st) : run<Shape<TYPE, 96, 64>>(p, st);
        case 128: return nmax > 64 ? run<Shape<TYPE, 128, 128>>(p, st) : run<Shape<TYPE, 128, 64>>(p, st);
        default: return run<Shape<TYPE, 256, 64>>(p, st);
    }
}

// Rows of a pass: 128 where a KV head has more than 64 and shared memory holds them beside the tiles.
int rows_of(const sjk_kv16 * c, int64_t rows) { return rows > 64 && c->head_dim <= 128 ? 128 : 64; }

}  // namespace

extern "C" size_t sjk_kv16_attend_tree_scratch_bytes(const sjk_kv16 * c) {
    if (!c || (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256)) return 0;
    return (size_t) CTAS * (2 * (size_t) rows_of(c, 128) * ((size_t) c->head_dim + 2) * sizeof(float) + sizeof(int4)) + sizeof(int4);
}

extern "C" int sjk_kv16_attend_tree(const sjk_kv16 * c, const sjk_rows * q, int n_tok, const int32_t * first, const int32_t * len,
                                    const int32_t * rows, const uint64_t * masks, int n_seq, int nodes, float scale, int window,
                                    const sjk_rows * out, void * scratch, size_t scratch_bytes, sjk_stream st) {
    if (!c || !q || !out || sjk_kv16_check(c) || n_seq < 0 || n_tok < 0 || nodes < 0 || window < 0 || !isfinite(scale)) return SJKVARN_ERR_ARG;
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256) return SJK_ERR_UNSUPPORTED;
    if (nodes > SJK_TREE_MAX) return SJK_ERR_UNSUPPORTED;
    if (q->type != c->type || out->type != c->type || q->n_head < 1 || q->n_head != out->n_head || q->n_head % c->n_head_kv) return SJKVARN_ERR_ARG;
    if (!list_ok(first) || !list_ok(len) || !list_ok(rows) || !aligned(masks, 8) || !rows_ok(*out) || (n_seq && !len)) return SJKVARN_ERR_ARG;
    if (n_tok && (!q->p || !out->p)) return SJKVARN_ERR_ARG;
    const int64_t strides = c->page_stride | c->slot_stride | c->head_stride | q->row_stride | q->head_stride;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(q->p, 16) || (strides & 7)) return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    if (!first && (int64_t) n_seq * nodes != (int64_t) n_tok) return SJKVARN_ERR_ARG;
    const int grp = q->n_head / c->n_head_kv;
    const int nmax = rows_of(c, (int64_t) nodes * grp);
    const int64_t tiles = ((int64_t) nodes * grp + nmax - 1) / nmax;
    if (tiles > CTAS) return SJK_ERR_UNSUPPORTED;
    // a list counts its units in 32 bits
    const double steps = fmin((double) c->table_stride * c->page_tokens, 2147483647.0) / TS + OV + 2;
    if (steps * n_seq * c->n_head_kv > 2e9) return SJK_ERR_UNSUPPORTED;
    if (n_seq == 0 || n_tok == 0 || nodes == 0) return 0;
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < sjk_kv16_attend_tree_scratch_bytes(c)) return SJKVARN_ERR_BUFFER;
    Params p = {};
    p.c = *c; p.q = *q; p.out = *out;
    p.first = first; p.len = len; p.rows = rows; p.masks = masks;
    p.n_seq = n_seq; p.n_tok = n_tok; p.nodes = nodes; p.grp = grp;
    p.window = window; p.scale = scale;
    auto span = [&](const sjk_rows & r) { return ((size_t) (n_tok - 1) * r.row_stride + (size_t) (r.n_head - 1) * r.head_stride + c->head_dim) * 2; };
    p.over = (q->row_stride | q->head_stride | out->row_stride | out->head_stride) < 0 || !apart(q->p, span(*q), out->p, span(*out));
    p.page_shift = -1;
    for (int b = 0; b < 31; ++b)
        if (c->page_tokens == 1 << b) p.page_shift = b;
    p.part = static_cast<float *>(scratch);
    p.ml = p.part + (size_t) CTAS * 2 * nmax * c->head_dim;
    p.split = reinterpret_cast<int4 *>(p.ml + (size_t) CTAS * 2 * nmax * 2);
    return c->type == SJK_F16 ? run_dim<SJK_F16>(p, nmax, st) : run_dim<SJK_BF16>(p, nmax, st);
}

SJK_STATUS_READER(tree_wait_status_take)

int sjk_tree_status_take(void) {
    unsigned v = 0;
    if (sjk_check(cudaMemcpyFromSymbol(&v, g_tree_status, sizeof v))) return -1;
    if (v) {
        const unsigned z = 0;
        if (sjk_check(cudaMemcpyToSymbol(g_tree_status, &z, sizeof z))) return -1;
    }
    const int t = tree_wait_status_take();
    return t < 0 ? -1 : (int) v | t;
}
