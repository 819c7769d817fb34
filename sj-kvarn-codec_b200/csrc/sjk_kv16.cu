// sjk_kv16.cu - attention of one new token per sequence over a paged 16-bit cache, split over the cache's length and
// joined: out = sum_t softmax_t(scale q . k_t) v_t over the last min(len, window) positions of each sequence.
//
// Bound: HBM, every live K and V row once (4 D bytes per position and KV head for 4 D grp flops: at most 16 flops per
// byte for 16 query heads, far under the tensor cores' ridge). So the work is to keep loads in flight:
//  - A warp is a worker of its own. The (sequence, KV head, step of TS tokens) triples of a call form one list, cut
//    into equal runs, one per warp of a grid that fills the GPU; lengths are read from device memory, so every warp
//    finds its run with a scan over them. Ragged batches balance by construction and no CTA barrier exists.
//  - A warp streams its steps through a ring in shared memory with cp.async, NST steps ahead and across the ends of
//    sequences; positions that are not live are filled with zeros, not read.
//  - The grp query heads of a KV head are the N = 8 columns of mma.m16n8k16: S^T = K Q^T with 16 tokens as rows, and
//    O^T = V^T P with 16 channels as rows, so a group of up to 8 heads wastes no rows of the accumulators, P goes from
//    the first product's layout to the second's with one 8x8 transpose (movmatrix), and the rescaling of O needs
//    values of its own lane only. These instructions are bound to registers and issue per warp, which lets every warp
//    run on its own; the tensor pipe is far from its limit here (16 flops per byte at most).
//  - A worker that held all of a sequence and head writes the output; otherwise (m, l, o[D]) per query head goes to
//    the worker's slot in the scratch, and the merge kernel joins the slots in list order (the result does not depend
//    on which worker came first).
// Softmax statistics, sums and outputs are 32-bit. Queries of the cache's type enter as they are and P is rounded
// once to it (up to 2^-8 of each weight for bf16, the size of the output's own rounding). For 32-bit queries or outputs
// (or a type other than the cache's) q is the sum of two (f16) or three (bf16) 16-bit terms and P of two, which keeps
// the products' errors at 2^-16 and below.
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

#include <math.h>

namespace {

using namespace sjk16;

constexpr int W = 4;                        // warps of a CTA
constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int MIN_STEPS = 2;                // steps of a worker's run, at least
__device__ unsigned int g_kv16_status;

struct Params {
    sjk_kv16 c;
    sjk_rows q, out;
    const int32_t * len, * rows;
    int n_seq, grp, tiles;                  // tiles: row tiles of a KV head (8 NT8 query heads each)
    int window;
    float scale;
    int n_work;                             // workers
    float * part;                           // [n_work][2][8 NT8][D]
    float * ml;                             // [n_work][2][8 NT8][2]
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

SJK_DEV int64_t warp_sum(int64_t x) {
#pragma unroll
    for (int m = 16; m; m >>= 1) x += __shfl_xor_sync(FULL, x, m);
    return x;
}
// steps per (KV head, row tile) of all sequences before `seq` (all lanes get the sum)
template <int TS>
SJK_DEV int64_t steps_before(const Params & p, int seq, int lane) {
    int64_t n = 0;
    for (int s = lane; s < seq; s += 32) n += span_of<TS>(p, s).n;
    return warp_sum(n);
}
// steps of a worker's run: the list has `total` steps
SJK_DEV int64_t run_steps(int64_t total, int n_work) {
    const int64_t per = (total + n_work - 1) / n_work;
    return per < MIN_STEPS ? MIN_STEPS : per;
}

template <int TS>
struct Cursor {                             // a place in the list
    int seq, hp, st;                        // sequence, (KV head, row tile), step
    Span s;
    SJK_DEV void skip_empty(const Params & p) {
        while (seq < p.n_seq && (s = span_of<TS>(p, seq)).n == 0) ++seq;
    }
    SJK_DEV void next(const Params & p, int HP) {
        if (++st < s.n) return;
        st = 0;
        if (++hp < HP) return;
        hp = 0;
        ++seq;
        skip_empty(p);
    }
};

SJK_DEV uint32_t smem_addr(const void * p) { return (uint32_t) __cvta_generic_to_shared(p); }
SJK_DEV void cp16(uint32_t dst, const void * src, bool on) {
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

// Kernel shape: TYPE of the cache, head size, NQ 16-bit terms of q and NP of P, NT8 tiles of 8 query heads.
template <int TYPE_, int D_, int NQ_, int NP_, int NT8_>
struct Shape {
    static constexpr int TYPE = TYPE_, D = D_, NQ = NQ_, NP = NP_, NT8 = NT8_;
    static constexpr int TM = tok_tiles(D), TS = step_toks(D), KS = D / 16;
    static constexpr int PITCH = 2 * D + 16;                // an odd number of 16-byte words: ldmatrix without conflicts
    static constexpr int ENTRY = TS * PITCH;
    static constexpr bool Q_REG = KS * 2 * NT8 * NQ <= 64;  // q in registers, else in shared memory
    static constexpr int Q_BYTES = Q_REG ? 0 : NQ * NT8 * 8 * PITCH;
    static constexpr int NST = D >= 256 && NQ > 1 && NT8 > 1 ? 1 : D >= 256 && (NQ > 1 || NT8 > 1) ? 2 : 3;
    static constexpr int WARP_BYTES = 2 * NST * ENTRY + Q_BYTES + 16;
    static constexpr int CTA_BYTES = W * WARP_BYTES;
};

template <typename S>
__global__ void __launch_bounds__(32 * W) kv16_attend_kernel(const __grid_constant__ Params p) {
    constexpr int D = S::D, TS = S::TS, TM = S::TM, KS = S::KS, NT8 = S::NT8, NQ = S::NQ, NP = S::NP, NST = S::NST, PITCH = S::PITCH;
    constexpr int R = 8 * NT8;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t * mine = smem + (size_t) warp * S::WARP_BYTES;
    const uint32_t ring = smem_addr(mine);
    uint32_t * s_mask = reinterpret_cast<uint32_t *>(mine + 2 * NST * S::ENTRY + S::Q_BYTES);
    pdl_wait();
    pdl_release();

    // the worker's run [run0, run1) of the list
    const int worker = blockIdx.x * W + warp;
    const int HP = p.c.n_head_kv * p.tiles;
    const int64_t total = steps_before<TS>(p, p.n_seq, lane) * HP;
    const int64_t per = run_steps(total, p.n_work);
    const int64_t run0 = worker * per, run1 = run0 + per < total ? run0 + per : total;
    if (run0 >= run1) return;
    Cursor<TS> at;                          // where the products are; `ld` below: where the loads are
    {
        int64_t before = 0;
        int s0 = 0;
        for (;; s0 += 32) {                 // the sequence that holds step run0: 32 sequences at a time
            const int64_t n = s0 + lane < p.n_seq ? (int64_t) span_of<TS>(p, s0 + lane).n * HP : 0;
            int64_t incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t y = __shfl_up_sync(FULL, incl, o);
                if (lane >= o) incl += y;
            }
            const unsigned past = __ballot_sync(FULL, before + incl > run0);
            if (past) {
                const int f = __ffs(past) - 1;
                const int64_t start = before + __shfl_sync(FULL, incl - n, f);
                at.seq = s0 + f;
                at.s = span_of<TS>(p, at.seq);
                at.hp = (int) ((run0 - start) / at.s.n);
                at.st = (int) ((run0 - start) - (int64_t) at.hp * at.s.n);
                break;
            }
            before += __shfl_sync(FULL, incl, 31);
        }
    }
    Cursor<TS> ld = at;
    const int64_t steps = run1 - run0;

    // ---- loads: the row of token `lane` of the step at ld, as an element offset; < 0 where it is not live ----
    int64_t ld_row = -1;
    const uint16_t * ld_k = nullptr, * ld_v = nullptr;      // the KV head's rows
    int64_t issued = 0;                                      // steps whose K and V went out
    auto look_up = [&]() {
        ld_row = -1;
        const int tok = (ld.s.first + ld.st) * TS + (lane & (TS - 1));
        if (tok >= ld.s.lo && tok < ld.s.hi) {
            const uint32_t g = (uint32_t) tok / (uint32_t) p.c.page_tokens;
            const int64_t row = p.rows ? (int64_t) p.rows[ld.seq] : (int64_t) ld.seq;
            const uint32_t page = row >= 0 && row < (int64_t) p.c.n_rows ? p.c.tables[row * p.c.table_stride + g] : SJKVARN_NO_BLOCK - 1u;
            if (page < p.c.n_pages)
                ld_row = (int64_t) page * p.c.page_stride + (int64_t) ((uint32_t) tok - g * (uint32_t) p.c.page_tokens) * p.c.slot_stride;
            else if (page != SJKVARN_NO_BLOCK)
                atomicOr(&g_kv16_status, (unsigned) SJK_DEVICE_PAGE);
        }
        const int64_t head = (int64_t) (ld.hp / p.tiles) * p.c.head_stride;
        ld_k = static_cast<const uint16_t *>(p.c.k) + head;
        ld_v = static_cast<const uint16_t *>(p.c.v) + head;
    };
    auto copy = [&](uint32_t dst, const uint16_t * base) {
        constexpr int CH = D / 8;                            // 16-byte words of a row
#pragma unroll
        for (int i = 0; i < (TS * CH + 31) / 32; ++i) {
            const int w = i * 32 + lane, r = w / CH, c = w - r * CH;
            const int64_t row = __shfl_sync(FULL, ld_row, r & (TS - 1));
            if (TS * CH % 32 == 0 || w < TS * CH) cp16(dst + r * PITCH + c * 16, base + (row < 0 ? 0 : row) + c * 8, row >= 0);
        }
    };
    auto issue_k = [&]() {
        if (issued < steps) {
            const unsigned live = __ballot_sync(FULL, ld_row >= 0);
            const int slot = (int) (issued % NST);
            if (lane == 0) s_mask[slot] = TS == 32 ? live : live & 0xFFFFu;
            copy(ring + slot * 2 * S::ENTRY, ld_k);
        }
        cp_commit();
    };
    auto issue_v = [&]() {
        if (issued < steps) {
            copy(ring + (int) (issued % NST) * 2 * S::ENTRY + S::ENTRY, ld_v);
            if (++issued < steps) { ld.next(p, HP); look_up(); }
        }
        cp_commit();
    };
    look_up();
#pragma unroll
    for (int i = 0; i < NST; ++i) { issue_k(); issue_v(); }

    // ---- products ----
    const int col = (lane & 3) * 2;                          // this lane's query heads of a tile of 8: col, col + 1
    uint32_t qf[S::Q_REG ? KS * NQ * NT8 * 2 : 1];
    float o[NT8][KS][4], m[NT8][2], l[NT8][2], sc[NT8][2];
    for (int64_t i = 0; i < steps; ++i) {
        if (i == 0 || at.st == 0) {                          // a (sequence, KV head, row tile) begins
            const int kv = at.hp / p.tiles, h0 = kv * p.grp + (at.hp - kv * p.tiles) * R;
            const int64_t qrow = (int64_t) at.seq * p.q.row_stride;
#pragma unroll
            for (int n = 0; n < NT8; ++n) {
                const int rel = h0 - kv * p.grp + 8 * n + (lane >> 2);
                const bool on = rel < p.grp;
                const int64_t src = qrow + (int64_t) (h0 + 8 * n + (lane >> 2)) * p.q.head_stride + (lane & 3) * 2;
                float mul = 1.0f;
                if constexpr (NQ > 1) {                      // the row to [1, 2) by an exact power of two
                    float big = 0.0f;
                    for (int k = 0; k < 2 * KS; ++k)
                        if (on) big = fmaxf(big, fmaxf(fabsf(load1(p.q.p, src + 8 * k, p.q.type)), fabsf(load1(p.q.p, src + 8 * k + 1, p.q.type))));
                    big = fmaxf(big, __shfl_xor_sync(FULL, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(FULL, big, 2));
                    const int e = big > 0.0f && big < INFINITY ? ilogbf(big) : 0;
                    mul = ldexpf(1.0f, e < -120 ? 120 : e > 120 ? -120 : -e);
                    const float c0 = __shfl_sync(FULL, mul, (col) * 4), c1 = __shfl_sync(FULL, mul, (col + 1) * 4);
                    sc[n][0] = p.scale * 1.4426950408889634f / c0;
                    sc[n][1] = p.scale * 1.4426950408889634f / c1;
                } else {
                    sc[n][0] = sc[n][1] = p.scale * 1.4426950408889634f;
                }
#pragma unroll
                for (int k = 0; k < 2 * KS; ++k) {
                    float2 x = make_float2(0.0f, 0.0f);
                    uint32_t w[NQ];
                    if constexpr (NQ == 1) {
                        w[0] = on ? *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(p.q.p) + src + 8 * k) : 0u;
                    } else {
                        if (on) x = make_float2(load1(p.q.p, src + 8 * k, p.q.type) * mul, load1(p.q.p, src + 8 * k + 1, p.q.type) * mul);
#pragma unroll
                        for (int t = 0; t < NQ; ++t) {
                            w[t] = pack2<S::TYPE>(x.x, x.y);
                            const float2 y = widen2<S::TYPE>(w[t]);
                            x.x -= y.x;
                            x.y -= y.y;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NQ; ++t) {
                        if constexpr (S::Q_REG) qf[((k >> 1) * NQ + t) * NT8 * 2 + n * 2 + (k & 1)] = w[t];
                        else
                            *reinterpret_cast<uint32_t *>(mine + 2 * NST * S::ENTRY + (t * NT8 * 8 + n * 8 + (lane >> 2)) * PITCH + k * 16 + (lane & 3) * 4) = w[t];
                    }
                }
                m[n][0] = m[n][1] = -INFINITY;
                l[n][0] = l[n][1] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.0f;
            }
            if constexpr (!S::Q_REG) __syncwarp();
        }
        const int slot = (int) (i % NST);
        const uint32_t kb = ring + slot * 2 * S::ENTRY, vb = kb + S::ENTRY;

        // S^T = K Q^T
        cp_wait<2 * NST - 1>();
        __syncwarp();
        float s[TM][NT8][4];
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            float s2[NT8][4];                                // two chains, so that products overlap
#pragma unroll
            for (int n = 0; n < NT8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[tm][n][e] = s2[n][e] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t a[4];
                ldsm4(a, kb + (tm * 16 + (lane & 15)) * PITCH + k * 32 + (lane >> 4) * 16);
#pragma unroll
                for (int t = 0; t < NQ; ++t) {
#pragma unroll
                    for (int n = 0; n < NT8; ++n) {
                        uint32_t b0, b1;
                        if constexpr (S::Q_REG) {
                            b0 = qf[(k * NQ + t) * NT8 * 2 + n * 2];
                            b1 = qf[(k * NQ + t) * NT8 * 2 + n * 2 + 1];
                        } else {
                            const uint8_t * qs = mine + 2 * NST * S::ENTRY + (t * NT8 * 8 + n * 8 + (lane >> 2)) * PITCH + k * 32 + (lane & 3) * 4;
                            b0 = *reinterpret_cast<const uint32_t *>(qs);
                            b1 = *reinterpret_cast<const uint32_t *>(qs + 16);
                        }
                        if ((k + t) & 1) mma<S::TYPE>(s2[n], a, b0, b1);
                        else mma<S::TYPE>(s[tm][n], a, b0, b1);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[tm][n][e] += s2[n][e];
        }
        const unsigned live = s_mask[slot];
        __syncwarp();
        issue_k();

        // softmax over the step's tokens: this lane has tokens lane / 4 (+ 8) of each 16, heads col and col + 1
        uint32_t pb[TM][NP][NT8][2];
#pragma unroll
        for (int n = 0; n < NT8; ++n) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int tm = 0; tm < TM; ++tm)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int tok = tm * 16 + (lane >> 2) + (e >> 1) * 8;
                    float x = s[tm][n][e] * sc[n][e & 1];
                    if (!((live >> tok) & 1u)) x = -INFINITY;
                    s[tm][n][e] = x;
                    top[e & 1] = fmaxf(top[e & 1], x);
                }
            float use[2], fix[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                top[j] = fmaxf(top[j], __shfl_xor_sync(FULL, top[j], 4));
                top[j] = fmaxf(top[j], __shfl_xor_sync(FULL, top[j], 8));
                top[j] = fmaxf(top[j], __shfl_xor_sync(FULL, top[j], 16));
                top[j] = fmaxf(top[j], m[n][j]);
                use[j] = top[j] == -INFINITY ? 0.0f : top[j];
                fix[j] = ex2(m[n][j] - use[j]);
            }
            if (__any_sync(FULL, top[0] != m[n][0] || top[1] != m[n][1])) {
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][k][e] *= fix[e & 1];
#pragma unroll
                for (int j = 0; j < 2; ++j) { l[n][j] *= fix[j]; m[n][j] = top[j]; }
            }
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[tm][n][e] = ex2(s[tm][n][e] - use[e & 1]);
                    l[n][e & 1] += s[tm][n][e];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = s[tm][n][2 * h], y = s[tm][n][2 * h + 1];
#pragma unroll
                    for (int t = 0; t < NP; ++t) {
                        const uint32_t w = pack2<S::TYPE>(x, y);
                        pb[tm][t][n][h] = transpose8(w);
                        if (t + 1 < NP) { const float2 f = widen2<S::TYPE>(w); x -= f.x; y -= f.y; }
                    }
                }
            }
        }

        // O^T += V^T P
        cp_wait<2 * NST - 1>();
        __syncwarp();
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t a[4];
                ldsm4t(a, vb + (tm * 16 + (lane & 7) + (lane >> 4) * 8) * PITCH + k * 32 + ((lane >> 3) & 1) * 16);
#pragma unroll
                for (int t = 0; t < NP; ++t)
#pragma unroll
                    for (int n = 0; n < NT8; ++n) mma<S::TYPE>(o[n][k], a, pb[tm][t][n][0], pb[tm][t][n][1]);
            }
        __syncwarp();
        issue_v();

        // the pair's last step of this run: its output, or its partial
        if (at.st + 1 == at.s.n || i + 1 == steps) {
            const bool begun = i >= at.st, ended = at.st + 1 == at.s.n;     // begun: its first step is in this run
            const int kv = at.hp / p.tiles, r0 = (at.hp - kv * p.tiles) * R;
#pragma unroll
            for (int n = 0; n < NT8; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[n][j] += __shfl_xor_sync(FULL, l[n][j], 4);
                    l[n][j] += __shfl_xor_sync(FULL, l[n][j], 8);
                    l[n][j] += __shfl_xor_sync(FULL, l[n][j], 16);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = 8 * n + col + j;
                    if (r0 + r >= p.grp) continue;
                    if (begun && ended) {
                        const float inv = l[n][j] == 0.0f ? 0.0f : 1.0f / l[n][j];
                        const int64_t dst = (int64_t) at.seq * p.out.row_stride + (int64_t) (kv * p.grp + r0 + r) * p.out.head_stride + (lane >> 2);
#pragma unroll
                        for (int k = 0; k < KS; ++k) {
                            store1(p.out.p, dst + 16 * k, p.out.type, o[n][k][j] * inv);
                            store1(p.out.p, dst + 16 * k + 8, p.out.type, o[n][k][2 + j] * inv);
                        }
                    } else {
                        const int64_t slot_row = ((int64_t) worker * 2 + (begun ? 1 : 0)) * R + r;
                        float * dst = p.part + slot_row * D + (lane >> 2);
#pragma unroll
                        for (int k = 0; k < KS; ++k) { dst[16 * k] = o[n][k][j]; dst[16 * k + 8] = o[n][k][2 + j]; }
                        if (lane < 4) { p.ml[slot_row * 2] = m[n][j]; p.ml[slot_row * 2 + 1] = l[n][j]; }
                    }
                }
            }
        }
        at.next(p, HP);
    }
    cp_wait<0>();
}

// Joins the slots of every (sequence, query head) that was split, in list order; G warps share one.
template <int TS>
__global__ void __launch_bounds__(256) kv16_merge_kernel(const __grid_constant__ Params p, int D, int R, int G) {
    extern __shared__ float s_acc[];        // [8 / G][G][D + 2]
    pdl_wait();
    pdl_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % G;
    const int n_head = p.q.n_head;
    const int64_t item = (int64_t) blockIdx.x * (8 / G) + warp / G;
    const bool on = item < (int64_t) p.n_seq * n_head;
    const int seq = on ? (int) (item / n_head) : 0, h = on ? (int) (item - (int64_t) seq * n_head) : 0;
    const int HP = p.c.n_head_kv * p.tiles;
    const int64_t total = steps_before<TS>(p, p.n_seq, lane) * HP, per = run_steps(total, p.n_work);
    const Span s = span_of<TS>(p, seq);
    const int kv = h / p.grp, rel = h - kv * p.grp, tile = rel / R, r = rel - tile * R;
    const int64_t a = steps_before<TS>(p, seq, lane) * HP + (int64_t) (kv * p.tiles + tile) * s.n;
    const int64_t first = s.n ? a / per : 0, last = s.n ? (a + s.n - 1) / per : 0;
    const bool join = on && s.n && first != last, zero = on && !s.n;
    const int64_t dst = (int64_t) seq * p.out.row_stride + (int64_t) h * p.out.head_stride;
    if (zero && sub == 0)
        for (int d = lane; d < D; d += 32) store1(p.out.p, dst + d, p.out.type, 0.0f);
    float top = -INFINITY, sum = 0.0f, o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.0f;
    if (join) {
        const int64_t n = last - first + 1, lo = first + n * sub / G, hi = first + n * (sub + 1) / G;
        for (int64_t w = lo + lane; w < hi; w += 32) top = fmaxf(top, p.ml[((w * 2 + (w == first ? 1 : 0)) * R + r) * 2]);
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, x));
        const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
        for (int64_t w = lo; w < hi; ++w) {
            const int64_t slot = (w * 2 + (w == first ? 1 : 0)) * R + r;
            const float2 ml = *reinterpret_cast<const float2 *>(p.ml + slot * 2);
            const float f = ex2(ml.x - use);
            sum = fmaf(ml.y, f, sum);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (32 * k + lane < D) o[k] = fmaf(p.part[slot * D + 32 * k + lane], f, o[k]);
        }
    }
    if (G > 1) {
        float * acc = s_acc + (size_t) warp * (D + 2);
        if (lane == 0) { acc[0] = top; acc[1] = sum; }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (32 * k + lane < D) acc[2 + 32 * k + lane] = o[k];
        __syncthreads();
        if (sub == 0 && join) {
            const float * all = s_acc + (size_t) warp * (D + 2);
            for (int g = 1; g < G; ++g) top = fmaxf(top, all[(size_t) g * (D + 2)]);
            const float use = top == -INFINITY ? 0.0f : top;
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = 0.0f;
            for (int g = 0; g < G; ++g) {
                const float * x = all + (size_t) g * (D + 2);
                const float f = ex2(x[0] - use);
                sum = fmaf(x[1], f, sum);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (32 * k + lane < D) o[k] = fmaf(x[2 + 32 * k + lane], f, o[k]);
            }
        }
    }
    if (join && sub == 0) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (32 * k + lane < D) store1(p.out.p, dst + 32 * k + lane, p.out.type, o[k] * inv);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------

struct Plan { int ctas, R, tiles; size_t part, ml; };       // part, ml: floats

template <typename S>
int ctas_per_sm() { return S::CTA_BYTES <= 75 * 1024 ? 3 : S::CTA_BYTES <= 113 * 1024 ? 2 : 1; }

template <typename S>
int run(const Params & p0, const Plan & pl, sjk_stream st) {
    static_assert(S::CTA_BYTES <= 227 * 1024, "shared memory of a CTA");
    Params p = p0;
    if (sjk_check(cudaFuncSetAttribute(kv16_attend_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::CTA_BYTES))) return SJK_ERR_DEVICE;
    const int rc = launch(kv16_attend_kernel<S>, dim3((unsigned) pl.ctas), dim3(32 * W), S::CTA_BYTES, st, p);
    if (rc) return rc;
    const int64_t items = (int64_t) p.n_seq * p.q.n_head;
    const int G = items <= 148 * 8 ? 8 : 1;                 // few outputs: a CTA each
    const int64_t ctas = (items + 8 / G - 1) / (8 / G);
    return launch(kv16_merge_kernel<S::TS>, dim3((unsigned) ctas), dim3(256), G > 1 ? (size_t) 8 * (S::D + 2) * sizeof(float) : 0, st, p, S::D, pl.R, G);
}

template <typename S>
int ctas_of() { return 148 * ctas_per_sm<S>(); }

// f(Shape) for the call's types and sizes
template <int TYPE, int D, typename F>
int with_terms(bool split, int nt8, F && f) {
    constexpr int NQ = TYPE == SJK_F16 ? 2 : 3;
    if (!split) return nt8 == 1 ? f(Shape<TYPE, D, 1, 1, 1>()) : f(Shape<TYPE, D, 1, 1, 2>());
    return nt8 == 1 ? f(Shape<TYPE, D, NQ, 2, 1>()) : f(Shape<TYPE, D, NQ, 2, 2>());
}
template <int TYPE, typename F>
int with_dim(int D, bool split, int nt8, F && f) {
    switch (D) {
        case 64: return with_terms<TYPE, 64>(split, nt8, f);
        case 96: return with_terms<TYPE, 96>(split, nt8, f);
        case 128: return with_terms<TYPE, 128>(split, nt8, f);
        case 256: return with_terms<TYPE, 256>(split, nt8, f);
        default: return SJK_ERR_UNSUPPORTED;
    }
}
template <typename F>
int with_shape(int type, int D, bool split, int nt8, F && f) {
    return type == SJK_F16 ? with_dim<SJK_F16>(D, split, nt8, f) : with_dim<SJK_BF16>(D, split, nt8, f);
}

int plan_of(const sjk_kv16 * c, int n_head, bool split, Plan * pl) {
    const int grp = n_head / c->n_head_kv, nt8 = grp <= 8 ? 1 : 2;
    pl->R = 8 * nt8;
    pl->tiles = (grp + pl->R - 1) / pl->R;
    const int rc = with_shape(c->type, c->head_dim, split, nt8, [&](auto s) { pl->ctas = ctas_of<decltype(s)>(); return 0; });
    if (rc) return rc;
    pl->part = (size_t) pl->ctas * W * 2 * pl->R * c->head_dim;
    pl->ml = (size_t) pl->ctas * W * 2 * pl->R * 2;
    return 0;
}

}  // namespace

extern "C" size_t sjk_kv16_attend_scratch_bytes(const sjk_kv16 * c, int n_head) {
    if (!c || c->n_head_kv < 1 || n_head < 1 || n_head % c->n_head_kv) return 0;
    size_t most = 0;
    for (int split = 0; split < 2; ++split) {
        Plan pl;
        if (plan_of(c, n_head, split != 0, &pl)) return 0;
        const size_t n = (pl.part + pl.ml) * sizeof(float);
        if (n > most) most = n;
    }
    return most;
}

extern "C" int sjk_kv16_attend(const sjk_kv16 * c, const sjk_rows * q, const int32_t * len, const int32_t * rows, int n_seq,
                               float scale, int window, const sjk_rows * out, void * scratch, size_t scratch_bytes, sjk_stream st) {
    if (!c || !q || !out || !len || n_seq < 0 || window < 0 || !isfinite(scale)) return SJKVARN_ERR_ARG;
    if (sjk_kv16_check(c)) return SJKVARN_ERR_ARG;
    if (!q->p || !out->p || !type_ok(q->type) || !type_ok(out->type) || q->n_head < 1 || q->n_head != out->n_head || q->n_head % c->n_head_kv)
        return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    const int64_t strides = c->page_stride | c->slot_stride | c->head_stride;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || (strides & 7)) return SJKVARN_ERR_ARG;
    // q of the cache's type is read two elements at a time
    const bool split = q->type != c->type || out->type == SJK_F32;
    if (!split && (!aligned(q->p, 4) || (q->row_stride & 1) || (q->head_stride & 1))) return SJKVARN_ERR_ARG;
    Plan pl;
    const int rc = plan_of(c, q->n_head, split, &pl);
    if (rc) return rc;
    if (n_seq == 0) return 0;
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < (pl.part + pl.ml) * sizeof(float)) return SJKVARN_ERR_BUFFER;
    Params p = {};
    p.c = *c; p.q = *q; p.out = *out;
    p.len = len; p.rows = rows; p.n_seq = n_seq;
    p.grp = q->n_head / c->n_head_kv; p.tiles = pl.tiles;
    p.window = window; p.scale = scale;
    p.n_work = pl.ctas * W;
    p.part = static_cast<float *>(scratch);
    p.ml = p.part + pl.part;
    return with_shape(c->type, c->head_dim, split, pl.R / 8, [&](auto s) { return run<decltype(s)>(p, pl, st); });
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
