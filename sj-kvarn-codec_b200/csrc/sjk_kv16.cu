// sjk_kv16.cu - attention of one new token per sequence over a paged 16-bit cache, split over the cache's length and
// joined: out = sum_t softmax_t(scale q . k_t) v_t over the last min(len, window) positions of each sequence.
//
// Bound: HBM, every live K and V row once (4 D bytes per position and KV head for 4 D grp flops: at most 16 flops per
// byte for 16 query heads, far under the tensor cores' ridge). Measured (us a call on the GPU alone, by CUDA graphs; GB/s
// of live rows): 32 sequences of 8K-64K, 4 KV heads of 256 bf16 channels 790-800 (6,270-6,350: a plain copy's rate is
// 6,539); one of 100,000 tokens with 32-bit queries and outputs 77 (5,320); 48 windows of 4,096, 24 heads of 64 channels 94
// (5,390); 256 short chats of 0 to 2,048 tokens 71 (4,600); one of 611 tokens 9.1. Pages of one token cost 3 to 10 % more
// than those of 16 (88 sequences of up to 19,024 tokens, 2 heads of 128: 59 against 58). What is left above the bytes:
// 4-5 us until the first products (launch, lengths, table, queries, first rows, each behind the other), 3 us for the merge,
// and SMs whose share of the memory is smaller than others' (the slowest end 15 % after the mean).
//  - A warp is a worker of its own. Per KV head, the (sequence, step of TS tokens) pairs of a call form one list, cut
//    into equal runs, one per warp of a grid that fills the GPU; lengths are read from device memory, so every warp
//    finds its run with a scan over them. A sequence weighs OV units beside its steps, for what its start and its
//    output cost. Ragged batches balance by construction, no CTA barrier paces the work, and the workers of all heads
//    are at the same tokens at the same time, whose rows lie side by side in memory.
//  - A warp streams its steps through a ring in shared memory with cp.async, a step ahead and across the ends of
//    sequences; positions that are not live are filled with zeros, not read.
//  - The query heads of a KV head are the N = 8 columns of mma.m16n8k16: S^T = K Q^T with 16 tokens as rows, and
//    O^T = V^T P with 16 channels as rows, so a group of up to 8 heads wastes no rows of the accumulators, P goes from
//    the first product's layout to the second's with one 8x8 transpose (movmatrix), and the rescaling of O needs
//    values of its own lane only. These instructions are bound to registers and issue per warp, which lets every warp
//    run on its own; the tensor pipe is far from its limit here (16 flops per byte at most).
//  - A worker that held all of a sequence and head writes the output; otherwise (m, l, o[D]) per query head goes to
//    the worker's slot in the scratch, and the merge kernel joins the slots in list order (the result does not depend
//    on which worker came first). The worker that begins a split pair leaves word of it, so the merge looks at as many
//    entries as there can be split pairs and scans nothing.
// Softmax statistics, sums and outputs are 32-bit. Queries of the cache's type enter as they are, and P as the sum of
// two 16-bit terms, one product each: to 2^-16 (bf16) or 2^-22 (f16) of a weight, so that a 16-bit output is off by its
// own rounding (one term would be 2^-8 of a weight off; the second one's products cost 1 % where one pass over K and V
// does, 256 short chats 69 us a pass against 68, and 4 % where 20 heads take two). For 32-bit queries or
// outputs (or a type other than the cache's) q and P are the sums of two (f16) or three (bf16) 16-bit terms side by side
// in the columns of the same products (4 or 2 heads in 8 columns), and each step's products are summed apart from what
// came before them, which keeps the result near 32 bits.
// Weights lie in (0, 1], and f16 has its last bit at 2^-24 there: weights of f16 caches are held 2^15 times larger, in l as
// well as in O, so that what is lost of a weight is at most 2^-40 of the largest in the worker's run (without it 2^-25:
// with one token 17 nats above all others, the others were gone from O while l still had them).
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

#include <math.h>

namespace {

using namespace sjk16;

constexpr unsigned FULL = 0xFFFFFFFFu;
// What a (sequence, KV head, row tile) costs beside its steps, in steps. 256 short chats, us on the GPU in two turns: 69
// and 71 with 4; 72 and 80 with 1, 71 and 68 with 2, 76 and 74 with 8 (256 sequences of up to 100 tokens 18.5; 19.4, 18.4, 20.7;
// long ragged batches within 1 %).
constexpr int OV = 4;
// Units of a worker's run, at least: fewer make more partials to join, more leave SMs idle. One sequence of 611 tokens 9.3
// us with 2, 10.6 with 1, 10.5 with 4, 13.1 with 8; seven of up to 300 with 32-bit rows 10.8, 10.0, 12.2, 14.7.
constexpr int MIN_RUN = 2;
constexpr float F16_UP = 32768.0f;          // weights of f16 caches, and so their sums and partials, are this much larger
__device__ unsigned int g_kv16_status;

struct Params {
    sjk_kv16 c;
    sjk_rows q, out;
    const int32_t * len, * rows;
    int n_seq, grp, tiles;                  // tiles: row tiles of a KV head (R query heads each)
    int window, page_shift;                 // page_shift: log2 of the page's tokens, -1 where it is no power of two
    uint32_t slot_stride;
    float scale;
    int n_work, wph;                        // workers; workers of a (KV head, row tile), 0: all share one list
    float * part;                           // [n_work][2][R][D]
    float * ml;                             // [n_work][2][R][2]
    int4 * split;                           // by pair (or, with more pairs than workers, by worker): sequence (-1: not
    int by_pair;                            // split), (KV head, row tile), first and last worker
};

// 16 tokens per m tile; steps of 32 tokens for small heads, whose rows are short
__host__ __device__ constexpr int tok_tiles(int D) { return D <= 64 ? 2 : 1; }
__host__ __device__ constexpr int step_toks(int D) { return 16 * tok_tiles(D); }

// live positions [lo, hi) of a sequence, and the steps that cover them
struct Span { int lo, hi, first, n; };
template <int TS>
SJK_DEV Span span_of(const Params & p, int seq) {
    Span s = {0, 0, 0, 0};
    int len = p.len[seq];
    const int64_t most = (int64_t) p.c.table_stride * p.c.page_tokens;
    if (len > most) { len = (int) most; atomicOr(&g_kv16_status, (unsigned) SJK_DEVICE_PAGE); }
    if (len <= 0) return s;
    s.hi = len;
    s.lo = p.window > 0 && len > p.window ? len - p.window : 0;
    s.first = s.lo / TS;
    s.n = (s.hi - 1) / TS + 1 - s.first;
    return s;
}

// units of a sequence in a (KV head, row tile)'s list: its steps behind OV that stand for its start and end
SJK_DEV uint32_t units_of(const Span & s) { return s.n ? (uint32_t) (s.n + OV) : 0u; }

template <int TS>
struct Cursor {                             // a place in the lists
    int seq, hp, st;                        // sequence, (KV head, row tile), step
    int rem;                                // units of the run from this step on; <= 0: the run is done
    uint32_t base;                          // unit of its list at which the sequence begins
    Span s;
    SJK_DEV bool next(const Params & p) {   // true: to another pair
        --rem;
        if (++st < s.n) return false;
        st = 0;
        rem -= OV;
        base += units_of(s);
        if (rem <= 0) return true;
        do {
            if (++seq == p.n_seq) { seq = 0; ++hp; base = 0u; }
            s = span_of<TS>(p, seq);
        } while (s.n == 0);
        return true;
    }
};

// exclusive prefix sum over the warp's lanes; *total gets the sum
SJK_DEV uint32_t warp_scan(uint32_t x, int lane, uint32_t * total) {
    uint32_t incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(FULL, incl, o);
        if (lane >= o) incl += y;
    }
    *total = __shfl_sync(FULL, incl, 31);
    return incl - x;
}

SJK_DEV uint32_t smem_addr(const void * p) { return (uint32_t) __cvta_generic_to_shared(p); }
SJK_DEV void cp16(uint32_t dst, const void * src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
SJK_DEV void cp16_or_zero(uint32_t dst, const void * src, bool on) {
    const int n = on ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
SJK_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
SJK_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
SJK_DEV void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
SJK_DEV void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
SJK_DEV uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int TYPE>
SJK_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (TYPE == SJK_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
SJK_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Kernel shape: TYPE of the cache, head size, T 16-bit terms of q and P, NT8 tiles of 8 columns; WHOLE: pages are of a
// multiple of 16 tokens, so that 16 tokens lie in one page, their rows a stride apart.
template <int TYPE_, int D_, int T_, int NT8_, bool WHOLE_>
struct Shape {
    static constexpr int TYPE = TYPE_, D = D_, T = T_, NT8 = NT8_;
    static constexpr bool WHOLE = WHOLE_;
    static constexpr int HT = T == 1 ? 8 : T == 2 ? 4 : 2;  // query heads of a tile
    static constexpr int R = HT * NT8;                      // and of a pass
    static constexpr int TM = tok_tiles(D), TS = step_toks(D), KS = D / 16;
    static constexpr int PITCH = 2 * D + 16;                // an odd number of 16-byte words: ldmatrix without conflicts
    static constexpr int ENTRY = TS * PITCH;
    // Eight warps in the one CTA of an SM, and a ring of one step (its K and its V tile, each asked for again as soon as
    // its products are done). More in flight was slower: the SMs' shares of the memory drift apart, and the slowest SM
    // ends last (48 windowed sequences of 64 channels: 90 us, 96 with three tiles, 100 with four; 32 sequences of
    // 8K-64K at 256 channels: 775, 778 with three). Six warps: 256 short chats 76 us against 67; ten and more: 11.2 us
    // against 9.3 for one sequence of 611 tokens, no gain elsewhere.
    static constexpr int W = 8;
    static constexpr int WARP_BYTES = 2 * ENTRY + 16;
    static constexpr int CTA_BYTES = W * WARP_BYTES;
};

// pairs of channels 8 STEP apart, from element `at` on
template <int TYPE, int STEP, int N>
SJK_DEV void load_pairs(float2 (&x)[N], const void * p, int64_t at, bool on) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        x[k] = make_float2(0.0f, 0.0f);
        if (on) x[k] = make_float2(load1(p, at + 8 * STEP * k, TYPE), load1(p, at + 8 * STEP * k + 1, TYPE));
    }
}
// w[i] to place i ^ u
template <int N>
SJK_DEV void swap_by(uint32_t (&w)[N], int u) {
#pragma unroll
    for (int b = 1; b < N; b <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!(i & b)) {
                const uint32_t x = w[i], y = w[i | b];
                w[i] = u & b ? y : x;
                w[i | b] = u & b ? x : y;
            }
}
template <int TYPE, int KS>
SJK_DEV void store_channels(void * p, int64_t at, const float (&o)[KS][4], int i, float f) {
#pragma unroll
    for (int k = 0; k < KS; ++k) store1(p, at + 16 * k, TYPE, o[k][i] * f);
}

template <typename S>
__global__ void __launch_bounds__(32 * S::W, 1) kv16_attend_kernel(const __grid_constant__ Params p) {
    constexpr int D = S::D, TS = S::TS, TM = S::TM, KS = S::KS, NT8 = S::NT8, T = S::T, HT = S::HT, R = S::R, PITCH = S::PITCH, W = S::W;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t * mine = smem + (size_t) warp * S::WARP_BYTES;
    const uint32_t ring = smem_addr(mine);
    uint32_t * s_mask = reinterpret_cast<uint32_t *>(mine + 2 * S::ENTRY);
    pdl_wait();
    pdl_release();

    // The worker's run: units of all sequences (a lane sums a block of them), then the block and the sequence at which
    // the run begins.
    const int HP = p.c.n_head_kv * p.tiles;
    const int block = (p.n_seq + 31) / 32;
    Span s0 = lane < p.n_seq ? span_of<TS>(p, lane) : Span{0, 0, 0, 0};
    uint32_t mine_u = block == 1 ? units_of(s0) : 0u, list;             // list: units of one (KV head, row tile)
    if (block > 1) {
#pragma unroll 8
        for (int i = 0; i < block; ++i) {
            const int q = lane * block + i;
            if (q < p.n_seq) mine_u += units_of(span_of<TS>(p, q));
        }
    }
    const uint32_t mine_0 = warp_scan(mine_u, lane, &list);
    Cursor<TS> at;                          // where the products are; `ld` below: where the loads are
    at.rem = 0;
    int worker = blockIdx.x * W + warp, wph = p.wph, ahead = warp;      // ahead: warps of the CTA in front of this one
    uint32_t off = 0;                       // where the run begins in its list
    int64_t per;
    if (wph) {
        per = (list + (uint32_t) wph - 1u) / (uint32_t) wph;
        if (per < MIN_RUN) {
            // fewer runs than workers: neighbours in the list go to different SMs
            per = MIN_RUN;
            wph = (int) ((list + MIN_RUN - 1u) / MIN_RUN);
            worker = warp * gridDim.x + blockIdx.x;
            ahead = -1;
        }
        at.hp = wph ? worker / wph : HP;
        const int64_t o = (int64_t) (worker - at.hp * wph) * per;
        if (at.hp < HP && o < list) { off = (uint32_t) o; at.rem = (int) (o + per < list ? per : list - o); }
    } else {
        const int64_t total = (int64_t) list * HP;
        per = (total + p.n_work - 1) / p.n_work;
        if (per < MIN_RUN) per = MIN_RUN;
        const int64_t run0 = worker * per;
        if (run0 < total) {
            at.hp = (int) (run0 / list);
            off = (uint32_t) (run0 - (int64_t) at.hp * list);
            at.rem = (int) (run0 + per < total ? per : total - run0);
        }
    }
    if (!p.by_pair && lane == 0) p.split[worker] = make_int4(-1, 0, 0, 0);
    bool joint = false;                     // the CTA's warps all work on one pair: their partials are joined here
    if (at.rem > 0) {
        int g = 31 - __clz(__ballot_sync(FULL, mine_u > 0u && mine_0 <= off));
        at.base = __shfl_sync(FULL, mine_0, g);
        at.seq = g;
        if (block > 1) {
            const int end = (g + 1) * block;
            for (int q0 = g * block;; q0 += 32) {           // (one round for up to 1,024 sequences)
                s0 = q0 + lane < p.n_seq && q0 + lane < end ? span_of<TS>(p, q0 + lane) : Span{0, 0, 0, 0};
                uint32_t all;
                const uint32_t before = at.base + warp_scan(units_of(s0), lane, &all);
                if (at.base + all <= off) { at.base += all; continue; }
                g = 31 - __clz(__ballot_sync(FULL, s0.n > 0 && before <= off));
                at.seq = q0 + g;
                at.base = __shfl_sync(FULL, before, g);
                break;
            }
        }
        at.s.lo = __shfl_sync(FULL, s0.lo, g);
        at.s.hi = __shfl_sync(FULL, s0.hi, g);
        at.s.first = __shfl_sync(FULL, s0.first, g);
        at.s.n = __shfl_sync(FULL, s0.n, g);
        // step j lies at unit OV + j of its sequence; the units before it go with its start
        const int in = (int) (off - at.base);
        const int64_t cta0 = (int64_t) off - ahead * per, j0 = wph ? worker % wph - ahead : 0;
        joint = ahead >= 0 && (wph == 0 || (j0 >= 0 && j0 + W <= wph)) && cta0 >= at.base && cta0 + per > (int64_t) at.base + OV &&
                cta0 + W * per <= (int64_t) at.base + at.s.n + OV;
        at.st = in > OV ? in - OV : 0;
        if (in < OV) at.rem -= OV - in;     // no steps where the run has only units before a first step
    }
    Cursor<TS> ld = at;

    // ---- loads ----
    constexpr unsigned ALL = TS == 32 ? FULL : 0xFFFFu;
    const uint16_t * ld_kp = nullptr, * ld_vp = nullptr;     // the KV head's rows
    const uint32_t * ld_table = nullptr;                     // the sequence's table row; NULL: out of range
    unsigned ld_live = 0;                                    // live tokens of the step at ld
    int64_t ld_off[TM];                                      // WHOLE: element offsets of its 16-token groups
    int64_t ld_row = -1;                                     // of group (WHOLE) or token ld_win + lane; < 0: no page, or
    int ld_win = 0;                                          // not in the span
    uint32_t ld_next = SJKVARN_NO_BLOCK;                     // page of token ld_win + 32 + lane, asked for a window ahead:
    bool ld_has = false;                                     // read when needed, every step would wait for its pages
    auto group_of = [&](int tok) { return p.page_shift >= 0 ? (uint32_t) tok >> p.page_shift : (uint32_t) tok / (uint32_t) p.c.page_tokens; };
    auto row_of = [&](int tok, uint32_t g, uint32_t page) {
        if (page < p.c.n_pages)
            return (int64_t) page * p.c.page_stride + (int64_t) (((uint32_t) tok - g * (uint32_t) p.c.page_tokens) * (uint64_t) p.slot_stride);
        if (page != SJKVARN_NO_BLOCK) atomicOr(&g_kv16_status, (unsigned) SJK_DEVICE_PAGE);
        return (int64_t) -1;
    };
    auto enter = [&]() {                                     // the pair at ld
        const int64_t row = p.rows ? (int64_t) p.rows[ld.seq] : (int64_t) ld.seq;
        const bool on = row >= 0 && row < (int64_t) p.c.n_rows;
        if (!on) atomicOr(&g_kv16_status, (unsigned) SJK_DEVICE_PAGE);
        ld_table = on ? p.c.tables + row * p.c.table_stride : nullptr;
        const int64_t head = (int64_t) (ld.hp / p.tiles) * p.c.head_stride;
        ld_kp = static_cast<const uint16_t *>(p.c.k) + head;
        ld_vp = static_cast<const uint16_t *>(p.c.v) + head;
        ld_win = -64;
        ld_has = false;
    };
    auto look_up = [&]() {                                   // the step at ld
        const int step = ld.s.first + ld.st, tok0 = step * TS;
        const int a = ld.s.lo - tok0, b = ld.s.hi - tok0;    // its tokens [a, b) are in the span
        if constexpr (S::WHOLE) {
            const int g = step * TM;
            if (g - ld_win >= 32) {                          // the pages of the next 32 groups
                ld_win = g;
                const uint32_t tok = (uint32_t) (g + lane) * 16u;            // (past 2^31 - 1 behind the longest sequence)
                ld_row = -1;
                if (tok < (uint32_t) ld.s.hi && tok + 16u > (uint32_t) ld.s.lo && ld_table) {
                    const uint32_t q = group_of((int) tok);
                    ld_row = row_of((int) tok, q, ld_table[q]);
                }
            }
            ld_live = ALL;
            if (a > 0) ld_live &= FULL << a;
            if (b < TS) ld_live &= ~(FULL << b);
#pragma unroll
            for (int h = 0; h < TM; ++h) {
                ld_off[h] = __shfl_sync(FULL, ld_row, g + h - ld_win);
                if (ld_off[h] < 0) ld_live &= ~(0xFFFFu << (16 * h));
            }
        } else {
            if (tok0 - ld_win >= 32) {                       // the next 32 tokens
                ld_has = ld_has && tok0 == ld_win + 32;
                ld_win = tok0;
                const int left = ld.s.hi - tok0 - lane;      // tokens from this lane's on (positions reach 2^31 - 2)
                ld_row = -1;
                if (left > 0 && tok0 + lane >= ld.s.lo && ld_table) {
                    const uint32_t q = group_of(tok0 + lane);
                    ld_row = row_of(tok0 + lane, q, ld_has ? ld_next : ld_table[q]);
                }
                ld_has = true;
                if (left > 32 && ld_table) ld_next = ld_table[group_of(tok0 + lane + 32)];
            }
            ld_live = __ballot_sync(FULL, ld_row >= 0) >> (tok0 - ld_win) & ALL;
        }
    };
    auto copy = [&](uint32_t dst, const uint16_t * base) {
        constexpr int CH = D / 8;                            // 16-byte words of a row
        if constexpr (!S::WHOLE) {
            const int t0 = (ld.s.first + ld.st) * TS - ld_win;
#pragma unroll 4
            for (int i = 0; i < TS * CH / 32; ++i) {
                const int w = i * 32 + lane, r = w / CH, c = w - r * CH;
                const int64_t row = __shfl_sync(FULL, ld_row, t0 + r);
                const bool on = row >= 0;
                cp16_or_zero(dst + r * PITCH + c * 16, base + (on ? row : 0) + c * 8, on);
            }
        } else if (ld_live == ALL) {
#pragma unroll
            for (int h = 0; h < TM; ++h) {                   // 16 rows: 32 words at a time, D / 16 times
                const uint16_t * src = base + ld_off[h];
                if constexpr (32 % CH == 0) {
                    src += (uint64_t) (lane / CH) * p.slot_stride + (lane % CH) * 8;
                    const uint64_t step = (uint64_t) (32 / CH) * p.slot_stride;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i, src += step) cp16(dst + (16 * h + i * (32 / CH) + lane / CH) * PITCH + (lane % CH) * 16, src);
                } else {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const int w = i * 32 + lane, r = w / CH, c = w - r * CH;
                        cp16(dst + (16 * h + r) * PITCH + c * 16, src + (uint64_t) r * p.slot_stride + c * 8);
                    }
                }
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < TS * CH / 32; ++i) {
                const int w = i * 32 + lane, r = w / CH, c = w - r * CH;
                const int64_t row = (TM == 2 && r >= 16 ? ld_off[TM - 1] : ld_off[0]) + (int64_t) ((uint64_t) (r & 15) * p.slot_stride);
                const bool on = (ld_live >> r) & 1u;
                cp16_or_zero(dst + r * PITCH + c * 16, base + (on ? row : 0) + c * 8, on);
            }
        }
    };
    // tiles go out in the order K, V of the first step, K, V of the second, ...: K into the ring's first place, V behind it
    auto issue = [&](bool v) {
        if (ld.rem > 0) {
            const uint32_t dst = ring + (v ? S::ENTRY : 0);
            if (!v) {
                if (lane == 0) *s_mask = ld_live;
                copy(dst, ld_kp);
            } else {
                copy(dst, ld_vp);
                const bool crossed = ld.next(p);
                if (ld.rem > 0) {
                    if (crossed) enter();
                    look_up();
                }
            }
        }
        cp_commit();
    };

    // ---- products ----
    // Column lane / 4 of a tile, as B operand: head and term. This lane's columns 2 (lane & 3) + j, as results: heads
    // first + j, of which it has term `mine_t`; with several terms the lanes of a quad sum what they have of a head.
    const int qcol = lane >> 2, qhead = T == 1 ? qcol : T == 2 ? qcol & 3 : qcol & 1, qterm = T == 1 ? 0 : T == 2 ? qcol >> 2 : qcol >> 1;
    const int first = T == 1 ? (lane & 3) * 2 : T == 2 ? (lane & 1) * 2 : 0, mine_t = T == 1 ? 0 : T == 2 ? (lane & 3) >> 1 : lane & 3;
    auto terms = [](float x) {                               // the sum over a head's terms
        if (T == 2) x += __shfl_xor_sync(FULL, x, 2);
        if (T == 3) { x += __shfl_xor_sync(FULL, x, 1); x += __shfl_xor_sync(FULL, x, 2); }
        return x;
    };
    // A pair's results at its end: with several terms the lanes of a quad divide the sums over them among themselves. Each
    // has NJ heads (from own_j on) of its NT8 tiles, and NH of the two 8-channel halves (from own_h on) of every 16.
    constexpr int NJ = T == 3 ? 1 : 2, NH = T == 1 ? 2 : 1;
    constexpr int PT = T == 1 ? 2 : 1;      // words of a weight in this lane: both terms, or the one of the lane's column
    const int own_j = T == 3 ? lane & 1 : 0, own_h = T == 1 ? 0 : (lane >> 1) & 1;
    auto at_of = [&](int j, int h) { return T == 1 ? 2 * h + j : T == 2 ? j : 0; };      // where in o[n][k]
    uint32_t qf[KS][NT8][2];
    float o[NT8][KS][4], m[NT8][2], l[NT8][2], sc[NT8][2];
    bool fresh = true, begun = false, started = false;       // a pair comes next; its first step is in this run; loads are out
    // the first loads: behind those of the queries, which would wait for them
    auto start = [&]() {
        if (started) return;
        started = true;
        enter();
        look_up();
#pragma unroll 1
        for (int i = 0; i < 2; ++i) issue(i != 0);
    };
    while (at.rem > 0) {
        if (fresh) {                                         // a (sequence, KV head, row tile) begins
            fresh = false;
            begun = at.st == 0;
            const int kv = at.hp / p.tiles, r0 = (at.hp - kv * p.tiles) * R;
            int64_t src[NT8];
            bool on[NT8];
#pragma unroll
            for (int n = 0; n < NT8; ++n) {
                const int rel = r0 + HT * n + qhead;
                on[n] = rel < p.grp;
                src[n] = (int64_t) at.seq * p.q.row_stride + (int64_t) (kv * p.grp + rel) * p.q.head_stride + (lane & 3) * 2;
            }
            if constexpr (T == 1) {
#pragma unroll
                for (int n = 0; n < NT8; ++n) {
#pragma unroll
                    for (int k = 0; k < 2 * KS; ++k)
                        qf[k >> 1][n][k & 1] = on[n] ? *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(p.q.p) + src[n] + 8 * k) : 0u;
                    sc[n][0] = sc[n][1] = p.scale * 1.4426950408889634f;
                }
                start();
            } else {
                // The GT lanes with a head's terms split every GT-th pair of channels each and exchange the words.
                constexpr int GT = T == 3 ? 4 : 2, SH = T == 3 ? 8 : 16, NX = 2 * KS / GT;
                float2 x[NT8][NX];
#pragma unroll
                for (int n = 0; n < NT8; ++n) {
                    const int64_t from = src[n] + 8 * qterm;
                    if (p.q.type == SJK_F32) load_pairs<SJK_F32, GT>(x[n], p.q.p, from, on[n]);
                    else if (p.q.type == SJK_F16) load_pairs<SJK_F16, GT>(x[n], p.q.p, from, on[n]);
                    else load_pairs<SJK_BF16, GT>(x[n], p.q.p, from, on[n]);
                }
                start();
#pragma unroll
                for (int n = 0; n < NT8; ++n) {
                    float big = 0.0f;                        // the row's largest to [1, 2) by an exact power of two; f16
                                                             // terms, whose last bit is 2^-24, to [2^14, 2^15)
#pragma unroll
                    for (int k = 0; k < NX; ++k) big = fmaxf(big, fmaxf(fabsf(x[n][k].x), fabsf(x[n][k].y)));
                    big = fmaxf(big, __shfl_xor_sync(FULL, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(FULL, big, 2));
                    big = fmaxf(big, __shfl_xor_sync(FULL, big, SH));
                    if (T == 3) big = fmaxf(big, __shfl_xor_sync(FULL, big, 2 * SH));
                    const int e = big > 0.0f && big < INFINITY ? ilogbf(big) : 0;
                    constexpr int UP = S::TYPE == SJK_F16 ? 14 : 0;
                    const float mul = ldexpf(1.0f, UP - (e < UP - 127 ? UP - 127 : e > UP + 113 ? UP + 113 : e));
#pragma unroll
                    for (int j = 0; j < 2; ++j) sc[n][j] = p.scale * 1.4426950408889634f / __shfl_sync(FULL, mul, (first + j) * 4);
#pragma unroll
                    for (int k = 0; k < NX; ++k) {
                        float a = x[n][k].x * mul, b = x[n][k].y * mul;
                        uint32_t w[GT];                      // the terms: what is left after those before them
#pragma unroll
                        for (int t = 0; t < T; ++t) {
                            w[t] = pack2<S::TYPE>(a, b);
                            const float2 z = widen2<S::TYPE>(w[t]);
                            a -= z.x;
                            b -= z.y;
                        }
                        if constexpr (T == 3) w[3] = 0u;     // the column without a term
                        // word t to the lane with term t, which puts it at this lane's place
                        swap_by<GT>(w, qterm);
#pragma unroll
                        for (int d = 1; d < GT; ++d) w[d] = __shfl_xor_sync(FULL, w[d], d * SH);
                        swap_by<GT>(w, qterm);
#pragma unroll
                        for (int v = 0; v < GT; ++v) qf[(GT * k + v) >> 1][n][(GT * k + v) & 1] = w[v];
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT8; ++n) {
                m[n][0] = m[n][1] = -INFINITY;
                l[n][0] = l[n][1] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.0f;
            }
        }
        const uint32_t kb = ring, vb = ring + S::ENTRY;

        // S^T = K Q^T
        cp_wait<1>();
        __syncwarp();
        float s[TM][NT8][4];
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            constexpr int CH = T > 1 && (D < 256 || NT8 == 1) ? 4 : 2;       // several chains: products overlap, sums stay short
            float c[CH][NT8][4];
#pragma unroll
            for (int x = 0; x < CH; ++x)
#pragma unroll
                for (int n = 0; n < NT8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[x][n][e] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t a[4];
                ldsm4(a, kb + (tm * 16 + (lane & 15)) * PITCH + k * 32 + (lane >> 4) * 16);
#pragma unroll
                for (int n = 0; n < NT8; ++n) mma<S::TYPE>(c[k % CH][n], a, qf[k][n][0], qf[k][n][1]);
            }
#pragma unroll
            for (int n = 0; n < NT8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[tm][n][e] = terms(CH == 2 ? c[0][n][e] + c[1][n][e] : (c[0][n][e] + c[1][n][e]) + (c[CH - 2][n][e] + c[CH - 1][n][e]));
        }
        const unsigned live = *s_mask;
        __syncwarp();
        issue(false);

        // Softmax over the step's tokens: this lane has tokens lane / 4 (+ 8) of each 16 of its two heads. The maximum is
        // looked for only when some score is above the one so far: seldom after a sequence's first steps.
        uint32_t pb[PT][TM][NT8][2];
        bool above = false;
#pragma unroll
        for (int n = 0; n < NT8; ++n)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[tm][n][e] *= sc[n][e & 1];
        if (live != ALL) {
#pragma unroll
            for (int n = 0; n < NT8; ++n)
#pragma unroll
                for (int tm = 0; tm < TM; ++tm)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((live >> (tm * 16 + (lane >> 2) + (e >> 1) * 8)) & 1u)) s[tm][n][e] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < NT8; ++n)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm)
#pragma unroll
                for (int e = 0; e < 4; ++e) above |= s[tm][n][e] > m[n][e & 1];
        if (__any_sync(FULL, above)) {
#pragma unroll
            for (int n = 0; n < NT8; ++n) {
                float up[2] = {m[n][0], m[n][1]}, fix[2];
#pragma unroll
                for (int tm = 0; tm < TM; ++tm)
#pragma unroll
                    for (int e = 0; e < 4; ++e) up[e & 1] = fmaxf(up[e & 1], s[tm][n][e]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    up[j] = fmaxf(up[j], __shfl_xor_sync(FULL, up[j], 4));
                    up[j] = fmaxf(up[j], __shfl_xor_sync(FULL, up[j], 8));
                    up[j] = fmaxf(up[j], __shfl_xor_sync(FULL, up[j], 16));
                    fix[j] = up[j] == m[n][j] ? 1.0f : ex2(m[n][j] - up[j]);
                    l[n][j] *= fix[j];
                    m[n][j] = up[j];
                }
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][k][e] *= fix[e & 1];
            }
        }
#pragma unroll
        for (int n = 0; n < NT8; ++n) {
            const float use[2] = {m[n][0] == -INFINITY ? 0.0f : m[n][0], m[n][1] == -INFINITY ? 0.0f : m[n][1]};
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[tm][n][e] = ex2(s[tm][n][e] - use[e & 1]);
                    if constexpr (S::TYPE == SJK_F16) s[tm][n][e] *= F16_UP;
                    l[n][e & 1] += s[tm][n][e];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = s[tm][n][2 * h], y = s[tm][n][2 * h + 1];
                    uint32_t w = pack2<S::TYPE>(x, y);
                    if constexpr (T == 1) {
                        const float2 f = widen2<S::TYPE>(w);
                        pb[PT - 1][tm][n][h] = transpose8(pack2<S::TYPE>(x - f.x, y - f.y));
                    }
#pragma unroll
                    for (int t = 1; t < T; ++t) {
                        const float2 f = widen2<S::TYPE>(w);
                        x -= f.x;
                        y -= f.y;
                        const uint32_t v = pack2<S::TYPE>(x, y);
                        if (mine_t >= t) w = v;
                        else { x += f.x; y += f.y; }
                    }
                    if (T == 3 && mine_t == 3) w = 0u;
                    pb[0][tm][n][h] = transpose8(w);
                }
            }
        }

        // O^T += V^T P
        cp_wait<1>();
        __syncwarp();
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t a[4];
                ldsm4t(a, vb + (tm * 16 + (lane & 7) + (lane >> 4) * 8) * PITCH + k * 32 + ((lane >> 3) & 1) * 16);
#pragma unroll
                for (int n = 0; n < NT8; ++n) {
                    if constexpr (T == 1) {
                        mma<S::TYPE>(o[n][k], a, pb[1][tm][n][0], pb[1][tm][n][1]);
                        mma<S::TYPE>(o[n][k], a, pb[0][tm][n][0], pb[0][tm][n][1]);
                    } else {                                 // the step's sum apart, joined by a rounded addition
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma<S::TYPE>(c, a, pb[0][tm][n][0], pb[0][tm][n][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][k][e] += c[e];
                    }
                }
            }
        __syncwarp();
        issue(true);

        // the pair's last step of this run: its output, or its partial
        if (at.st + 1 == at.s.n || at.rem == 1) {
            const bool ended = at.st + 1 == at.s.n;
            fresh = true;
            if (begun && lane == 0) {
                const uint32_t end = at.base + (uint32_t) (at.s.n + OV - 1);
                const int last = ended ? worker : wph ? at.hp * wph + (int) (end / (uint32_t) per) : (int) (((int64_t) at.hp * list + end) / per);
                if (p.by_pair) p.split[at.seq * HP + at.hp] = make_int4(ended ? -1 : at.seq, at.hp, worker, last);
                else if (!ended) p.split[worker] = make_int4(at.seq, at.hp, worker, last);
            }
            const int kv = at.hp / p.tiles, r0 = (at.hp - kv * p.tiles) * R;
#pragma unroll
            for (int n = 0; n < NT8; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[n][j] += __shfl_xor_sync(FULL, l[n][j], 4);
                    l[n][j] += __shfl_xor_sync(FULL, l[n][j], 8);
                    l[n][j] += __shfl_xor_sync(FULL, l[n][j], 16);
                }
                if constexpr (T > 1) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float lo = o[n][k][j], hi = o[n][k][2 + j];
                            o[n][k][j] = (own_h ? hi : lo) + __shfl_xor_sync(FULL, own_h ? lo : hi, 2);
                        }
                        if constexpr (T == 3) {
                            const float x = o[n][k][0], y = o[n][k][1];
                            o[n][k][0] = (own_j ? y : x) + __shfl_xor_sync(FULL, own_j ? x : y, 1);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int r = HT * n + first + own_j + j;
                    if (r0 + r >= p.grp) continue;
                    if (joint) continue;                     // written below
                    const float mj = own_j ? m[n][1] : m[n][j], lj = own_j ? l[n][1] : l[n][j];
                    if (begun && ended) {
                        const float inv = lj == 0.0f ? 0.0f : 1.0f / lj;
                        const int64_t dst = (int64_t) at.seq * p.out.row_stride + (int64_t) (kv * p.grp + r0 + r) * p.out.head_stride + (lane >> 2) + 8 * own_h;
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            if (p.out.type == SJK_F32) store_channels<SJK_F32>(p.out.p, dst + 8 * h, o[n], at_of(j, h), inv);
                            else if (p.out.type == SJK_F16) store_channels<SJK_F16>(p.out.p, dst + 8 * h, o[n], at_of(j, h), inv);
                            else store_channels<SJK_BF16>(p.out.p, dst + 8 * h, o[n], at_of(j, h), inv);
                        }
                    } else {
                        const int64_t slot = ((int64_t) worker * 2 + (begun ? 1 : 0)) * R + r;
#pragma unroll
                        for (int h = 0; h < NH; ++h) store_channels<SJK_F32>(p.part, slot * D + (lane >> 2) + 8 * (own_h + h), o[n], at_of(j, h), 1.0f);
                        if (lane < 4 && own_h == 0) *reinterpret_cast<float2 *>(p.ml + slot * 2) = make_float2(mj, lj);
                    }
                }
            }
        }
        at.next(p);
    }
    cp_wait<0>();

    // The CTA's partials of one pair as the first warp's, in the warps' order; the others' slots are left without weight.
    if (!joint) return;                     // the same for all warps: each looks at the CTA's whole run
    __syncthreads();                        // nothing reads the rings any more
    float * s_o = reinterpret_cast<float *>(smem);          // [W][R][D]
    float2 * s_ml = reinterpret_cast<float2 *>(s_o + W * R * D);
    static_assert(W * R * (D + 2) * 4 <= S::CTA_BYTES, "partials in the rings' place");
    if (lane < 4 && mine_t == 0)
#pragma unroll
        for (int n = 0; n < NT8; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) s_ml[warp * R + HT * n + first + j] = make_float2(m[n][j], l[n][j]);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT8; ++n)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int r = HT * n + first + own_j + j;
            float top = -INFINITY;
            for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w * R + r].x);
            const float f = ex2((own_j ? m[n][1] : m[n][j]) - (top == -INFINITY ? 0.0f : top));
#pragma unroll
            for (int h = 0; h < NH; ++h) store_channels<SJK_F32>(s_o, (warp * R + r) * D + (lane >> 2) + 8 * (own_h + h), o[n], at_of(j, h), f);
        }
    __syncthreads();
    const bool first_begun = __syncthreads_or(warp == 0 && begun);
    const int64_t slot = ((int64_t) blockIdx.x * W * 2 + (first_begun ? 1 : 0)) * R;
    for (int i = threadIdx.x; i < R * D; i += 32 * W) {
        float x = 0.0f;
        for (int w = 0; w < W; ++w) x += s_o[w * R * D + i];
        p.part[slot * D + i] = x;
    }
    for (int i = threadIdx.x; i < W * R; i += 32 * W) {
        const int w = i / R, r = i - w * R;
        if (w) { *reinterpret_cast<float2 *>(p.ml + ((int64_t) (blockIdx.x * W + w) * 2 * R + r) * 2) = make_float2(-INFINITY, 0.0f); continue; }
        float top = -INFINITY, sum = 0.0f;
        for (int v = 0; v < W; ++v) top = fmaxf(top, s_ml[v * R + r].x);
        for (int v = 0; v < W; ++v) sum = fmaf(s_ml[v * R + r].y, ex2(s_ml[v * R + r].x - (top == -INFINITY ? 0.0f : top)), sum);
        *reinterpret_cast<float2 *>(p.ml + (slot + r) * 2) = make_float2(top, sum);
    }
}

// Joins the slots of a split pair, in list order, and writes the zeros of sequences without a live position. grid.x:
// entries of p.split, then a sequence per warp (before the wait: the lengths are older than the kernel waited for). G of
// the CTA's warps share a query head; grid.y CTAs and their other warps take the heads of an entry in turn.
template <int D>
__global__ void __launch_bounds__(512) kv16_merge_kernel(const __grid_constant__ Params p, int R, int G, int entries) {
    constexpr int NV = (D / 4 + 31) / 32;   // 16-byte words of a lane
    extern __shared__ __align__(16) float s_acc[];          // [warps][D + 4] where they share a head
    const int warps = blockDim.x >> 5;
    if (blockIdx.x >= entries) {
        const int seq = (blockIdx.x - entries) * warps + (threadIdx.x >> 5);
        if (blockIdx.y == 0 && seq < p.n_seq && p.len[seq] <= 0)
            for (int i = threadIdx.x & 31; i < p.out.n_head * D; i += 32)
                store1(p.out.p, (int64_t) seq * p.out.row_stride + (int64_t) (i / D) * p.out.head_stride + i % D, p.out.type, 0.0f);
        pdl_wait();
        pdl_release();
        return;
    }
    pdl_wait();
    pdl_release();
    // (in the order of pairs, the entry of a sequence without a live position was not written)
    if (p.by_pair && p.len[blockIdx.x / (p.c.n_head_kv * p.tiles)] <= 0) return;
    const int4 e = p.split[blockIdx.x];
    if (e.x < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % G;
    const int kv = e.y / p.tiles, r0 = (e.y - kv * p.tiles) * R, nr = p.grp - r0 < R ? p.grp - r0 : R;
    const int n = e.w - e.z + 1, lo = (int) ((int64_t) n * sub / G), hi = (int) ((int64_t) n * (sub + 1) / G);
    for (int r = blockIdx.y * (warps / G) + warp / G; r < nr; r += gridDim.y * (warps / G)) {
        float top = -INFINITY, sum = 0.0f;
        float4 o[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w0 = lo; w0 < hi; w0 += 32) {
            // slot 1 of the first worker, slot 0 of the others
            const int w = w0 + lane;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (w < hi) ml = *reinterpret_cast<const float2 *>(p.ml + (((int64_t) (e.z + w) * 2 + (w == 0 ? 1 : 0)) * R + r) * 2);
            float t = ml.x;
#pragma unroll
            for (int x = 16; x; x >>= 1) t = fmaxf(t, __shfl_xor_sync(FULL, t, x));
            t = fmaxf(t, top);
            const float use = t == -INFINITY ? 0.0f : t, fix = ex2(top - use), f = ex2(ml.x - use);
            top = t;
            sum = sum * fix + (w < hi ? ml.y * f : 0.0f);    // a lane's own share; joined below
#pragma unroll
            for (int v = 0; v < NV; ++v) { o[v].x *= fix; o[v].y *= fix; o[v].z *= fix; o[v].w *= fix; }
            for (unsigned some = __ballot_sync(FULL, f != 0.0f); some;) {   // four parts with a weight at a time
                float g[4];
                float4 x[4][NV];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = some ? __ffs(some) - 1 : 0;
                    g[i] = __shfl_sync(FULL, f, j);
                    if (!some) g[i] = 0.0f;
                    some &= some - 1u;
                    const float4 * src = reinterpret_cast<const float4 *>(p.part + (((int64_t) (e.z + w0 + j) * 2 + (w0 + j == 0 ? 1 : 0)) * R + r) * D);
#pragma unroll
                    for (int v = 0; v < NV; ++v) x[i][v] = g[i] != 0.0f && 32 * v + lane < D / 4 ? src[32 * v + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        o[v].x = fmaf(x[i][v].x, g[i], o[v].x); o[v].y = fmaf(x[i][v].y, g[i], o[v].y);
                        o[v].z = fmaf(x[i][v].z, g[i], o[v].z); o[v].w = fmaf(x[i][v].w, g[i], o[v].w);
                    }
            }
        }
#pragma unroll
        for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(FULL, sum, x);
        if (G > 1) {
            float * acc = s_acc + warp * (D + 4);
            if (lane == 0) { acc[0] = top; acc[1] = sum; }
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (32 * v + lane < D / 4) *reinterpret_cast<float4 *>(acc + 4 + 4 * (32 * v + lane)) = o[v];
            __syncthreads();
            if (sub == 0) {
                for (int g = 1; g < G; ++g) top = fmaxf(top, acc[g * (D + 4)]);
                const float use = top == -INFINITY ? 0.0f : top;
                sum = 0.0f;
#pragma unroll
                for (int v = 0; v < NV; ++v) o[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int g = 0; g < G; ++g) {
                    const float * y = acc + g * (D + 4);
                    const float f = ex2(y[0] - use);
                    sum = fmaf(y[1], f, sum);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (32 * v + lane < D / 4) {
                            const float4 x = *reinterpret_cast<const float4 *>(y + 4 + 4 * (32 * v + lane));
                            o[v].x = fmaf(x.x, f, o[v].x); o[v].y = fmaf(x.y, f, o[v].y);
                            o[v].z = fmaf(x.z, f, o[v].z); o[v].w = fmaf(x.w, f, o[v].w);
                        }
                }
            }
            __syncthreads();
        }
        if (sub == 0) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int64_t dst = (int64_t) e.x * p.out.row_stride + (int64_t) (kv * p.grp + r0 + r) * p.out.head_stride;
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (32 * v + lane < D / 4) {
                    const int d = 4 * (32 * v + lane);
                    store1(p.out.p, dst + d, p.out.type, o[v].x * inv);
                    store1(p.out.p, dst + d + 1, p.out.type, o[v].y * inv);
                    store1(p.out.p, dst + d + 2, p.out.type, o[v].z * inv);
                    store1(p.out.p, dst + d + 3, p.out.type, o[v].w * inv);
                }
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------

struct Plan { int work, R, nt8, tiles; size_t part, ml, bytes; };    // part, ml: floats

template <typename S>
int run(const Params & p0, const Plan & pl, sjk_stream st) {
    static_assert(S::CTA_BYTES <= 227 * 1024, "shared memory of a CTA");
    Params p = p0;
    int rc = smem_limit<kv16_attend_kernel<S>>(S::CTA_BYTES);
    if (rc) return rc;
    rc = launch(kv16_attend_kernel<S>, dim3(148), dim3(32 * S::W), S::CTA_BYTES, st, p);
    if (rc) return rc;
    // few pairs: many slots each, so a CTA per query head; many: two or three slots each, a warp per query head
    const int64_t pairs = (int64_t) p.n_seq * p.c.n_head_kv * p.tiles;
    const bool few = pairs * 8 <= p.n_work;
    const int rows = p.grp < pl.R ? p.grp : pl.R, entries = p.by_pair ? (int) pairs : p.n_work;
    // (16 warps for a head with hundreds of slots: 78.1 against 79.6 us at 100,000 tokens; 8 do for a few dozen)
    const double steps = fmin((double) p.c.table_stride * p.c.page_tokens, 2147483647.0) / S::TS;
    const int warps = few ? (fmin(steps / MIN_RUN, (double) p.n_work / pairs) > 64.0 ? 16 : 8) : rows < 8 ? rows : 8;
    return launch(kv16_merge_kernel<S::D>, dim3((unsigned) (entries + (p.n_seq + warps - 1) / warps), few ? (unsigned) rows : 1u), dim3(32 * warps),
                  few ? (size_t) warps * (S::D + 4) * sizeof(float) : 0, st, p, pl.R, few ? warps : 1, entries);
}

// f(Shape) for the call's types and sizes: nt8 1 or 2 tiles of columns in one pass over K and V
template <int TYPE, int D, bool WHOLE, typename F>
int with_terms(bool split, int nt8, F && f) {
    constexpr int T = TYPE == SJK_F16 ? 2 : 3;
    if (!split) return nt8 == 1 ? f(Shape<TYPE, D, 1, 1, WHOLE>()) : f(Shape<TYPE, D, 1, 2, WHOLE>());
    return nt8 == 1 ? f(Shape<TYPE, D, T, 1, WHOLE>()) : f(Shape<TYPE, D, T, 2, WHOLE>());
}
template <int TYPE, bool WHOLE, typename F>
int with_dim(int D, bool split, int nt8, F && f) {
    switch (D) {
        case 64: return with_terms<TYPE, 64, WHOLE>(split, nt8, f);
        case 96: return with_terms<TYPE, 96, WHOLE>(split, nt8, f);
        case 128: return with_terms<TYPE, 128, WHOLE>(split, nt8, f);
        case 256: return with_terms<TYPE, 256, WHOLE>(split, nt8, f);
        default: return SJK_ERR_UNSUPPORTED;
    }
}
template <typename F>
int with_shape(const sjk_kv16 * c, bool split, int nt8, F && f) {
    if (c->page_tokens % 16 == 0)
        return c->type == SJK_F16 ? with_dim<SJK_F16, true>(c->head_dim, split, nt8, f) : with_dim<SJK_BF16, true>(c->head_dim, split, nt8, f);
    return c->type == SJK_F16 ? with_dim<SJK_F16, false>(c->head_dim, split, nt8, f) : with_dim<SJK_BF16, false>(c->head_dim, split, nt8, f);
}

int plan_of(const sjk_kv16 * c, int n_head, bool split, Plan * pl) {
    const int grp = n_head / c->n_head_kv, ht = !split ? 8 : c->type == SJK_F16 ? 4 : 2;
    pl->nt8 = grp <= ht ? 1 : 2;
    const int rc = with_shape(c, split, pl->nt8, [&](auto s) { pl->work = 148 * decltype(s)::W; pl->R = decltype(s)::R; return 0; });
    if (rc) return rc;
    pl->tiles = (grp + pl->R - 1) / pl->R;
    pl->part = (size_t) pl->work * 2 * pl->R * c->head_dim;
    pl->ml = (size_t) pl->work * 2 * pl->R * 2;
    pl->bytes = (pl->part + pl->ml) * sizeof(float) + (size_t) pl->work * sizeof(int4);
    return 0;
}

}  // namespace

extern "C" size_t sjk_kv16_attend_scratch_bytes(const sjk_kv16 * c, int n_head) {
    if (!c || c->n_head_kv < 1 || n_head < 1 || n_head % c->n_head_kv) return 0;
    size_t most = 0;
    for (int split = 0; split < 2; ++split) {
        Plan pl;
        if (plan_of(c, n_head, split != 0, &pl)) return 0;
        if (pl.bytes > most) most = pl.bytes;
    }
    return most;
}

extern "C" int sjk_kv16_attend(const sjk_kv16 * c, const sjk_rows * q, const int32_t * len, const int32_t * rows, int n_seq,
                               float scale, int window, const sjk_rows * out, void * scratch, size_t scratch_bytes, sjk_stream st) {
    if (!c || !q || !out || !len || n_seq < 0 || window < 0 || !isfinite(scale)) return SJKVARN_ERR_ARG;
    if (sjk_kv16_check(c)) return SJKVARN_ERR_ARG;
    if (!q->p || !out->p || !type_ok(q->type) || !type_ok(out->type) || !rows_ok(*q) || !rows_ok(*out) || !list_ok(len) || !list_ok(rows) || q->n_head < 1 || q->n_head != out->n_head || q->n_head % c->n_head_kv)
        return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    const int64_t strides = c->page_stride | c->slot_stride | c->head_stride;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || (strides & 7)) return SJKVARN_ERR_ARG;
    // q of the cache's type is read two elements at a time
    const bool split = q->type != c->type || out->type == SJK_F32;
    if (!split && (!aligned(q->p, 4) || (q->row_stride & 1) || (q->head_stride & 1))) return SJKVARN_ERR_ARG;
    if (c->slot_stride > 0x7FFFFFFF) return SJK_ERR_UNSUPPORTED;
    Plan pl;
    const int rc = plan_of(c, q->n_head, split, &pl);
    if (rc) return rc;
    if (n_seq == 0) return 0;
    // a list counts its units in 32 bits, and a worker its run, whatever the lengths
    const double most = (fmin((double) c->table_stride * c->page_tokens, 2147483647.0) / 16 + OV + 1) * n_seq;
    const int HP = c->n_head_kv * pl.tiles;
    if (most > 2e9 || most * HP / pl.work > 2e9) return SJK_ERR_UNSUPPORTED;
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < pl.bytes) return SJKVARN_ERR_BUFFER;
    Params p = {};
    p.c = *c; p.q = *q; p.out = *out;
    p.len = len; p.rows = rows; p.n_seq = n_seq;
    p.grp = q->n_head / c->n_head_kv; p.tiles = pl.tiles;
    p.window = window; p.scale = scale;
    p.slot_stride = (uint32_t) c->slot_stride;
    p.page_shift = -1;
    for (int b = 0; b < 31; ++b)
        if (c->page_tokens == 1 << b) p.page_shift = b;
    p.n_work = pl.work;
    p.part = static_cast<float *>(scratch);
    p.ml = p.part + pl.part;
    p.split = reinterpret_cast<int4 *>(p.ml + pl.ml);
    p.by_pair = (int64_t) n_seq * HP <= p.n_work;
    // a list per head where that leaves under a sixteenth of the workers without one
    p.wph = HP * 16 <= p.n_work ? p.n_work / HP : 0;
    return with_shape(c, split, pl.nt8, [&](auto s) { return run<decltype(s)>(p, pl, st); });
}

int sjk_kv16_status_take(void) {
    unsigned v = 0;
    if (sjk_check(cudaMemcpyFromSymbol(&v, g_kv16_status, sizeof v))) return -1;
    if (v) {
        const unsigned z = 0;
        if (sjk_check(cudaMemcpyToSymbol(g_kv16_status, &z, sizeof z))) return -1;
    }
    return (int) v;
}
