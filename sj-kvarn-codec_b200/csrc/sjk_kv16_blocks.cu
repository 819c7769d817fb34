// sjk_kv16_blocks.cu - attention to a part of a long context: bounds of the keys of every page (sjk_kv16_bounds), the
// pages that these bounds choose for a query (sjk_kv16_select), and the lists that the attention over them reads
// (sjk_kv16_attend_blocks, whose kernel is that of sjk_kv16_attend).
//
// For a query head q and a page whose keys lie in [lo, hi] channel by channel, q . k <= sum_d max(q_d lo_d, q_d hi_d). The
// heads of a KV head's group share their pages, and the sum of their bounds is one product of the page's 2 D bounds:
//   u = sum_d up_d hi_d + down_d lo_d,   up_d = sum_g max(q_gd, 0),  down_d = sum_g min(q_gd, 0),
// so the score costs the same for any group. A choice hangs on the order of these numbers, so they are held in 64 bits:
// the products of 16-bit bounds are exact there, and a sum of 512 is off by 2^-44 of its terms, where 32-bit sums (2^-15)
// would swap neighbours of the border at some hundreds of pages.
//
// Bound: the bytes of the bounds (4 D a page and KV head) and of the keys (2 D a position and KV head); for few sequences the five
// launches of a choice with its attention, each a chain of dependent loads. Measured (us on the GPU by CUDA graphs): bounds of a
// decode step of 64 sequences in 4 layers 4.7, of a prompt of 32,700 tokens in 2 layers 29 (138 MB: 4.8 TB/s; 31 with a CTA per page
// and its warps joined in shared memory); the choice among 6,250 pages for each of 8 heads 19, among up to 512 for 128 lists 24, the
// attention over the chosen 2,048 positions 13 and 59 (268 MB of rows: 4.6 TB/s). Long lists: 22 among 8,192 pages (in registers), 24
// among 8,200 (read anew in every round), 148 among 62,500 (a million tokens: 256 MB of bounds, 39 us at a copy's rate).
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

#include <math.h>

namespace {

using namespace sjk16;

constexpr unsigned FULL = 0xFFFFFFFFu;
constexpr int NT = 256;
__device__ unsigned int g_blocks_status;

SJK_DEV void flag() { atomicOr(&g_blocks_status, (unsigned) SJK_DEVICE_PAGE); }

// a sequence's table row (NULL: none) and the positions that fit in it
SJK_DEV const uint32_t * table_of(const sjk_kv16 & c, const int32_t * rows, int i) {
    const int64_t row = rows ? (int64_t) rows[i] : (int64_t) i;
    if (row < 0 || row >= (int64_t) c.n_rows) { flag(); return nullptr; }
    return c.tables + row * c.table_stride;
}
SJK_DEV int fit(const sjk_kv16 & c, int32_t len) {
    const int64_t most = (int64_t) c.table_stride * c.page_tokens;
    if (len > most) { flag(); return (int) most; }
    return len < 0 ? 0 : len;
}

// ---- bounds ---------------------------------------------------------------------------------------------------
struct BoundParams {
    sjk_kv16 c;
    int64_t layer_stride, b_layer_stride;
    uint16_t * bounds;                      // [n_pages][2][H][D] of a layer
    const int32_t * first, * end, * rows;
};

// smaller (larger) of two pairs; a NaN stays one, so that its page is chosen and read, as all pages would be
template <int TYPE, bool MAX>
SJK_DEV uint32_t pick2(uint32_t a, uint32_t b) {
    if constexpr (TYPE == SJK_F16) {
        const __half2 x = *reinterpret_cast<const __half2 *>(&a), y = *reinterpret_cast<const __half2 *>(&b);
        const __half2 z = MAX ? __hmax2_nan(x, y) : __hmin2_nan(x, y);
        return *reinterpret_cast<const uint32_t *>(&z);
    } else {
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162 *>(&a), y = *reinterpret_cast<const __nv_bfloat162 *>(&b);
        const __nv_bfloat162 z = MAX ? __hmax2_nan(x, y) : __hmin2_nan(x, y);
        return *reinterpret_cast<const uint32_t *>(&z);
    }
}
template <int TYPE, bool MAX>
SJK_DEV uint4 pick8(const uint4 & a, const uint4 & b) {
    return make_uint4(pick2<TYPE, MAX>(a.x, b.x), pick2<TYPE, MAX>(a.y, b.y), pick2<TYPE, MAX>(a.z, b.z), pick2<TYPE, MAX>(a.w, b.w));
}

// A warp takes 32 neighbouring 16-byte words of a page's key rows (all heads side by side; fewer words: several tokens at a
// time), BATCH rows in flight. grid: sequences, CTAs whose warps take a sequence's (page, words) in turn, layers.
template <int TYPE>
__global__ void __launch_bounds__(NT) bounds_kernel(const __grid_constant__ BoundParams p) {
    constexpr int BATCH = 8;
    pdl_wait();
    pdl_release();
    const int i = blockIdx.x, lane = threadIdx.x & 31, P = p.c.page_tokens, per = p.c.head_dim / 8, words = p.c.n_head_kv * per;
    const uint32_t * table = table_of(p.c, p.rows, i);
    const int first = max(p.first[i], 0), end = fit(p.c, p.end[i]);
    if (!table || first >= end) return;
    const uint16_t * keys = static_cast<const uint16_t *>(p.c.k) + (int64_t) blockIdx.z * p.layer_stride;
    uint4 * out = reinterpret_cast<uint4 *>(p.bounds + (int64_t) blockIdx.z * p.b_layer_stride);
    const int span = words < 32 ? words : 32, rows = 32 / span, at = lane / span, groups = (words + 31) / 32;
    const int g0 = first / P;
    const int64_t units = (int64_t) ((end - 1) / P - g0 + 1) * groups;
    for (int64_t u = (int64_t) blockIdx.y * (NT / 32) + (threadIdx.x >> 5); u < units; u += (int64_t) gridDim.y * (NT / 32)) {
        const int g = g0 + (int) (u / groups), w = (int) (u % groups) * 32 + lane - at * span, h = w / per;
        const uint32_t page = table[g];
        if (page >= p.c.n_pages) {
            if (page != SJKVARN_NO_BLOCK) flag();
            continue;
        }
        const int64_t left = (int64_t) end - (int64_t) g * P;
        const int live = (int) (left < P ? left : P);
        const bool on = at < rows && w < words;
        const uint16_t * src = keys + (int64_t) page * p.c.page_stride + (int64_t) h * p.c.head_stride + (w - h * per) * 8;
        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
        if (on) {
            // (a lane without a token of its own takes the first one)
            lo = hi = *reinterpret_cast<const uint4 *>(src + (int64_t) (at < live ? at : 0) * p.c.slot_stride);
            for (int t0 = at + rows; t0 < live; t0 += BATCH * rows) {
                uint4 x[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    const int t = t0 + b * rows;
                    x[b] = *reinterpret_cast<const uint4 *>(src + (int64_t) (t < live ? t : t0) * p.c.slot_stride);
                }
#pragma unroll
                for (int b = 0; b < BATCH; ++b) { lo = pick8<TYPE, false>(lo, x[b]); hi = pick8<TYPE, true>(hi, x[b]); }
            }
        }
        __syncwarp();
        for (int r = 1; r < rows; ++r) {
            const int from = (lane + r * span) & 31;        // (what lanes behind the first row's get is not used)
            uint4 a, b;
            a.x = __shfl_sync(FULL, lo.x, from); a.y = __shfl_sync(FULL, lo.y, from); a.z = __shfl_sync(FULL, lo.z, from); a.w = __shfl_sync(FULL, lo.w, from);
            b.x = __shfl_sync(FULL, hi.x, from); b.y = __shfl_sync(FULL, hi.y, from); b.z = __shfl_sync(FULL, hi.z, from); b.w = __shfl_sync(FULL, hi.w, from);
            if (at == 0) { lo = pick8<TYPE, false>(lo, a); hi = pick8<TYPE, true>(hi, b); }
        }
        if (on && at == 0) {
            uint4 * dst = out + (int64_t) page * 2 * words + w;
            dst[0] = lo;
            dst[words] = hi;
        }
    }
}

// ---- select: scores --------------------------------------------------------------------------------------------
struct SelectParams {
    sjk_kv16 c;
    const uint16_t * bounds;
    sjk_rows q;
    const int32_t * len, * rows;
    int n_seq, grp, budget, sink, recent;
    uint64_t * keys;                        // [n_seq][H][table_stride]
    int32_t * blocks, * count;
};

// A 16-bit number's sign, exponent and fraction moved to their places in a 64-bit one: the value times 2^-896 (bf16) or
// 2^-1008 (f16), subnormals included, in two operations; infinities and NaNs by way of 32 bits. The weights are held
// larger by that less 2^192, which leaves room for every product of 32-bit floats: scores are 2^-192 of their size.
template <int TYPE>
constexpr double moved_by() { return TYPE == SJK_F16 ? 0x1p-1008 : 0x1p-896; }
template <int TYPE>
constexpr double weight_by() { return TYPE == SJK_F16 ? 0x1p816 : 0x1p704; }
template <int TYPE>
SJK_DEV double moved(uint32_t top) {                        // the number in the upper half of a word
    constexpr int SH = TYPE == SJK_F16 ? 6 : 3;
    constexpr uint32_t KEEP = TYPE == SJK_F16 ? 0x81FFFC00u : 0x8FFFE000u;
    return __hiloint2double((int) ((uint32_t) ((int32_t) top >> SH) & KEEP), 0);
}
template <int TYPE>
SJK_DEV bool odd2(uint32_t w) {                             // an infinity or NaN in a word
    constexpr uint32_t E = TYPE == SJK_F16 ? 0x7C00u : 0x7F80u;
    return (w & E) == E || (w & (E << 16)) == (E << 16);
}
// order of 64-bit floats as unsigned integers; NaN above all numbers
SJK_DEV uint64_t order_of(double x) {
    if (x != x) x = __longlong_as_double(0x7FF0000000000000ll);
    const uint64_t b = (uint64_t) __double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
constexpr uint64_t NEVER = 0ull, ALWAYS = ~0ull;            // no page; first and newest ones

// A warp scores PG pages of a (sequence, KV head) at a time: a lane has 8 channels of one side (16 where D is 256), and a
// partial sum of every page, which an exchange by halves leaves in the lane of each page. The CTA makes the weights, which
// all its warps share. grid: sequences, heads, groups of pages. Smaller groups of pages make more warps, whose loads are out
// at the same time (the whole pass with groups of 32, 16 and 8: 63, 43 and 38 us for one sequence, 134, 99 and 89 for 32, the
// quicker choice included). Asking for the first pages' bounds before the weights are made was slower (registers: 42 and 92).
constexpr int NQ = 128, PG = 8;             // threads; pages of a warp at a time
template <int TYPE, int D>
__global__ void __launch_bounds__(NQ) score_kernel(const __grid_constant__ SelectParams p) {
    constexpr int WORDS = D / 8, NW = D == 256 ? 2 : 1;     // words of a side; words of a lane
    constexpr int HALF = D == 64 ? 2 : 1;                   // pages of one load
    constexpr int NA = PG / HALF;                           // loads
    __shared__ double s_w[2][D];                            // sums over the group's heads of the queries below and above zero
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, i = blockIdx.x, h = blockIdx.y, P = p.c.page_tokens;
    const int len = fit(p.c, p.len[i]), nb = (int) (((int64_t) len + P - 1) / P);
    const uint32_t * table = table_of(p.c, p.rows, i);
    uint64_t * keys = p.keys + ((int64_t) i * p.c.n_head_kv + h) * p.c.table_stride;
    constexpr int CTA = NQ / 32 * PG;                       // pages of a CTA at a time
    if ((int64_t) blockIdx.z * CTA >= nb) return;
    if (!table || nb <= p.budget) {                         // all pages
        for (int64_t b = (int64_t) blockIdx.z * NQ + threadIdx.x; b < nb; b += (int64_t) gridDim.z * NQ) {
            const uint32_t page = table ? table[b] : SJKVARN_NO_BLOCK;
            if (page >= p.c.n_pages && page != SJKVARN_NO_BLOCK) flag();
            keys[b] = page < p.c.n_pages ? ALWAYS : NEVER;
        }
        return;
    }
    for (int d = threadIdx.x; d < D; d += NQ) {
        const int64_t q0 = (int64_t) i * p.q.row_stride + (int64_t) h * p.grp * p.q.head_stride + d;
        double down = 0.0, up = 0.0;
        for (int g = 0; g < p.grp; ++g) {
            const double x = (double) load1(p.q.p, q0 + (int64_t) g * p.q.head_stride, p.q.type);
            down += x > 0.0 ? 0.0 : x;                      // (a NaN goes to one of them, and from there to every score)
            up += x > 0.0 ? x : 0.0;
        }
        s_w[0][d] = down * weight_by<TYPE>();
        s_w[1][d] = up * weight_by<TYPE>();
    }
    __syncthreads();
    const int sub = HALF == 2 ? lane & 15 : lane;
    const int side = NW == 2 ? 0 : sub / WORDS, c0 = NW == 2 ? lane : sub - side * WORDS;    // (D = 256: a word of both sides)
    const bool on = NW == 2 || sub < 2 * WORDS;
    double wt[NW][8];
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) wt[n][e] = on ? s_w[NW == 2 ? n : side][c0 * 8 + e] : 0.0;
    const int64_t row_words = (int64_t) p.c.n_head_kv * WORDS;
    const uint4 * base = reinterpret_cast<const uint4 *>(p.bounds) + (int64_t) h * WORDS + side * row_words + c0;
    for (int64_t b0 = (int64_t) blockIdx.z * CTA + (threadIdx.x >> 5) * PG; b0 < nb; b0 += (int64_t) gridDim.z * CTA) {
        const int64_t b = b0 + (lane & (PG - 1));
        uint32_t page = SJKVARN_NO_BLOCK;
        if (b < nb) page = table[b];
        const bool have = page < p.c.n_pages;
        if (!have && page != SJKVARN_NO_BLOCK) flag();
        const uint32_t read = have ? page : 0u;
        double acc[NA];
        uint4 x[NA][NW];
#pragma unroll
        for (int u = 0; u < NA; ++u) {
            // (D = 64: the lower lanes have page u, the upper ones the one NA after it)
            const uint32_t at = __shfl_sync(FULL, read, HALF == 2 ? u + (lane >> 4) * NA : u);
            const uint4 * src = base + (int64_t) at * 2 * row_words;
#pragma unroll
            for (int n = 0; n < NW; ++n) x[u][n] = on ? src[n * row_words] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < NA; ++u) {
            double s = 0.0;
#pragma unroll
            for (int n = 0; n < NW; ++n) {
                const uint32_t w[4] = {x[u][n].x, x[u][n].y, x[u][n].z, x[u][n].w};
                if (odd2<TYPE>(w[0]) || odd2<TYPE>(w[1]) || odd2<TYPE>(w[2]) || odd2<TYPE>(w[3])) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = widen2<TYPE>(w[e]);
                        // (an infinity on the side that no head looks at does not count)
                        if (f.x != f.x || wt[n][2 * e] != 0.0) s = fma((double) f.x * moved_by<TYPE>(), wt[n][2 * e], s);
                        if (f.y != f.y || wt[n][2 * e + 1] != 0.0) s = fma((double) f.y * moved_by<TYPE>(), wt[n][2 * e + 1], s);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s = fma(moved<TYPE>(w[e] << 16), wt[n][2 * e], s);
                        s = fma(moved<TYPE>(w[e]), wt[n][2 * e + 1], s);
                    }
                }
            }
            acc[u] = s;
        }
        // lane l gets the sum of page l % NA (of its half's)
#pragma unroll
        for (int o = NA / 2; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < o; ++u) {
                const bool up = lane & o;
                const double send = up ? acc[u] : acc[u + o], keep = up ? acc[u + o] : acc[u];
                acc[u] = keep + __shfl_xor_sync(FULL, send, o);
            }
#pragma unroll
        for (int o = NA; o < 32 / HALF; o <<= 1) acc[0] += __shfl_xor_sync(FULL, acc[0], o);
        // (D = 64: pages 4 to 7 are in the upper half)
        const double mine = HALF == 2 ? __shfl_sync(FULL, acc[0], (lane & (NA - 1)) + ((lane & (PG - 1)) / NA) * 16) : acc[0];
        if (lane < PG && b < nb) keys[b] = !have ? NEVER : b < p.sink || b >= nb - p.recent ? ALWAYS : order_of(mine);
    }
}

// ---- select: the largest `budget` keys of a list ------------------------------------------------------------------
constexpr int KR = 8;                       // keys that a thread holds in registers
// Exclusive sum over the CTA's NS threads, and the whole. s: NS / 32 words, free again behind the caller's next barrier.
template <int NS>
SJK_DEV uint32_t cta_before(uint32_t x, uint32_t * s, uint32_t * all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(FULL, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s[warp] = incl;
    __syncthreads();
    const uint32_t w = lane < NS / 32 ? s[lane] : 0u;
    *all = __reduce_add_sync(FULL, w);
    return __reduce_add_sync(FULL, lane < warp ? w : 0u) + incl - x;
}

// A CTA per (sequence, head): the threshold by counting the keys in BINS equal parts of their range, then those of the part in
// which it lies in BINS parts of that, until exactly as many are left as are wanted (twice, for keys apart from one
// another); then the keys above it and the first of those equal to it, in ascending order of their pages. A thread has a run
// of KR pages in registers; lists of more than NS KR pages are read anew in every round. Counts alone are atomic: the same
// lists every time. NS threads: 256 for lists of up to 2,048 pages, whose barriers cost less (128 lists of up to 512: the
// choice with its scores 24.7 us against 26.4 with 1,024).
template <int NS, bool NEAR>
__global__ void __launch_bounds__(NS) choose_kernel(const __grid_constant__ SelectParams p) {
    constexpr int BINS = 2 * NS, LOG = NS == 1024 ? 11 : 9;
    static_assert(BINS == 1 << LOG, "two bins a thread");
    __shared__ uint32_t s_bin[BINS], s_sum[4][NS / 32];
    __shared__ uint64_t s_min[NS / 32], s_max[NS / 32], s_from;
    __shared__ uint32_t s_above, s_in;
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = blockIdx.x, h = blockIdx.y, P = p.c.page_tokens;
    const int64_t list = (int64_t) i * p.c.n_head_kv + h;
    const int len = fit(p.c, p.len[i]), nb = (int) (((int64_t) len + P - 1) / P);
    const uint64_t * keys = p.keys + list * p.c.table_stride;
    int32_t * out = p.blocks + list * p.budget;
    const int run = NEAR ? KR : (nb + NS - 1) / NS;
    const int64_t b0 = (int64_t) tid * run;
    uint64_t mine[KR];
    if (NEAR)
#pragma unroll
        for (int j = 0; j < KR; ++j) mine[j] = b0 + j < nb ? keys[b0 + j] : NEVER;
    // f(key, page) of the thread's run
    auto each = [&](auto && f) {
        if (NEAR) {
#pragma unroll
            for (int j = 0; j < KR; ++j) f(mine[j], (int) b0 + j);
        } else
            for (int64_t b = b0; b < b0 + run && b < nb; ++b) f(keys[b], (int) b);
    };
    // the range of the keys that are neither chosen in any case nor never
    uint64_t lo = ALWAYS, hi = NEVER;
    uint32_t some = 0, always = 0;
    each([&](uint64_t k, int) {
        some += k != NEVER ? 1u : 0u;
        always += k == ALWAYS ? 1u : 0u;
        if (k == NEVER || k == ALWAYS) return;
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(FULL, lo, o), b = __shfl_xor_sync(FULL, hi, o);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    if (lane == 0) { s_min[warp] = lo; s_max[warp] = hi; }
    some = __reduce_add_sync(FULL, some);
    always = __reduce_add_sync(FULL, always);
    if (lane == 0) { s_sum[0][warp] = some; s_sum[1][warp] = always; }
    __syncthreads();
    const bool on = lane < NS / 32;
    some = __reduce_add_sync(FULL, on ? s_sum[0][lane] : 0u);
    always = __reduce_add_sync(FULL, on ? s_sum[1][lane] : 0u);
    const uint32_t want = min((uint32_t) p.budget, some);
    lo = on ? s_min[lane] : ALWAYS;
    hi = on ? s_max[lane] : NEVER;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(FULL, lo, o), b = __shfl_xor_sync(FULL, hi, o);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    // the largest t with at least `want` keys >= t. Keys of [from, from + 2^bits) are in question, `over` ones lie above.
    uint64_t t = always >= want ? ALWAYS : lo;
    if (always < want && some > want) {
        uint64_t from = lo;
        uint32_t over = always;
        int bits = 64 - __clzll((long long) (hi - lo | 1ull));              // hi - lo < 2^bits
        for (;;) {
            const int shift = bits > LOG ? bits - LOG : 0;
            const uint64_t parts = 1ull << (bits - shift);                  // BINS, or fewer in a last round: keys behind them are in `over`
            s_bin[tid] = s_bin[tid + NS] = 0u;
            __syncthreads();
            each([&](uint64_t k, int) {
                if (k == NEVER || k == ALWAYS || k < from) return;
                const uint64_t d = (k - from) >> shift;
                if (d < parts) atomicAdd(&s_bin[d], 1u);
            });
            __syncthreads();
            // from the highest part down: the first with `want` keys at or above it
            const uint32_t hi_n = s_bin[BINS - 1 - 2 * tid], lo_n = s_bin[BINS - 2 - 2 * tid];
            uint32_t all;
            const uint32_t before = over + cta_before<NS>(hi_n + lo_n, s_sum[2], &all);
            if (before < want && before + hi_n + lo_n >= want) {
                const bool first = before + hi_n >= want;
                s_from = from + ((uint64_t) (first ? BINS - 1 - 2 * tid : BINS - 2 - 2 * tid) << shift);
                s_above = first ? before : before + hi_n;
                s_in = first ? hi_n : lo_n;
            }
            __syncthreads();
            from = s_from;
            over = s_above;
            bits = shift;
            if (shift == 0 || over + s_in == want) break;
        }
        t = from;                           // keys >= from: `want`, or more that are all equal
    }
    // keys above t, and the first `ties` of those equal to it
    uint32_t above = 0, equal = 0;
    each([&](uint64_t k, int) {
        above += k > t ? 1u : 0u;
        equal += k == t && k != NEVER ? 1u : 0u;
    });
    __syncthreads();
    uint32_t above_all, equal_all;
    const uint32_t xa = cta_before<NS>(above, s_sum[0], &above_all);
    uint32_t xe = cta_before<NS>(equal, s_sum[1], &equal_all);
    const uint32_t ties = want - above_all;
    uint32_t at = xa + (xe < ties ? xe : ties);
    each([&](uint64_t k, int b) {
        bool take = k > t;
        if (k == t && k != NEVER) take = xe++ < ties;
        if (take) out[at++] = b;
    });
    for (uint32_t e = want + tid; e < (uint32_t) p.budget; e += NS) out[e] = -1;
    if (tid == 0 && p.count) p.count[list] = (int32_t) want;
}

// ---- lists of pages for the attention -----------------------------------------------------------------------------
struct ListParams {
    sjk_kv16 c;
    const int32_t * len, * rows, * blocks;
    int n_seq, budget;
    uint32_t * tables;                      // [n_seq][H][budget]: pages
    int32_t * lens;                         // [n_seq][H]: positions on them
};

// A warp per (sequence, head): pages of the listed blocks up to the first entry that is none (-1), does not ascend or
// lies behind the sequence; only the sequence's newest block, which is then the last, holds fewer than a page's tokens.
__global__ void __launch_bounds__(NT) lists_kernel(const __grid_constant__ ListParams p) {
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, P = p.c.page_tokens;
    const int64_t list = (int64_t) blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
    if (list >= (int64_t) p.n_seq * p.c.n_head_kv) return;
    const int i = (int) (list / p.c.n_head_kv);
    const int len = fit(p.c, p.len[i]), nb = (int) (((int64_t) len + P - 1) / P);
    const uint32_t * table = table_of(p.c, p.rows, i);
    const int32_t * blocks = p.blocks + list * p.budget;
    uint32_t * pages = p.tables + list * p.budget;
    int count = 0, last = -1;
    for (int e0 = 0; table && e0 < p.budget; e0 += 32) {
        const int e = e0 + lane;
        const int b = e < p.budget ? blocks[e] : -1;
        int before = __shfl_up_sync(FULL, b, 1);
        if (lane == 0) before = last;
        const bool ok = b >= 0 && b < nb && b > before;
        const unsigned good = __ballot_sync(FULL, ok);
        const int n = good == FULL ? 32 : __ffs(~good) - 1;      // up to the first that is none
        if (lane == n && e < p.budget && b != -1) flag();        // (what lies behind it is not looked at)
        if (lane < n) pages[e] = table[b];
        count += n;
        if (n) last = __shfl_sync(FULL, b, n - 1);
        if (n < 32) break;
    }
    if (lane == 0) p.lens[list] = count == 0 ? 0 : (int32_t) ((int64_t) (count - 1) * P + (last == nb - 1 ? len - (int64_t) last * P : P));
}

template <int TYPE>
int score_launch(const SelectParams & p, dim3 grid, sjk_stream st) {
    switch (p.c.head_dim) {
        case 64: return launch(score_kernel<TYPE, 64>, grid, dim3(NQ), 0, st, p);
        case 96: return launch(score_kernel<TYPE, 96>, grid, dim3(NQ), 0, st, p);
        case 128: return launch(score_kernel<TYPE, 128>, grid, dim3(NQ), 0, st, p);
        default: return launch(score_kernel<TYPE, 256>, grid, dim3(NQ), 0, st, p);
    }
}

int check_of(const sjk_kv16 * c) {
    if (!c || sjk_kv16_check(c)) return SJKVARN_ERR_ARG;
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256) return SJK_ERR_UNSUPPORTED;
    return 0;
}

}  // namespace

extern "C" int sjk_kv16_bounds(const sjk_kv16 * c, int n_layers, int64_t layer_stride, void * bounds, int64_t bounds_stride,
                               const int32_t * first, const int32_t * end, const int32_t * rows, int n_seq, sjk_stream st) {
    const int rc = check_of(c);
    if (rc) return rc;
    if (n_layers < 1 || n_layers > 65535 || layer_stride < 0 || bounds_stride < 0 || !bounds || n_seq < 0 || (n_seq && (!first || !end))) return SJKVARN_ERR_ARG;
    const int64_t strides = c->page_stride | c->slot_stride | c->head_stride | (n_layers > 1 ? layer_stride | bounds_stride : 0);
    if (!aligned(c->k, 16) || !aligned(bounds, 16) || (strides & 7) || !list_ok(first) || !list_ok(end) || !list_ok(rows)) return SJKVARN_ERR_ARG;
    if (n_layers > 1 && bounds_stride < (int64_t) c->n_pages * 2 * c->n_head_kv * c->head_dim) return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    if (n_seq == 0) return 0;
    const BoundParams p = {*c, layer_stride, bounds_stride, static_cast<uint16_t *>(bounds), first, end, rows};
    int64_t y = 148 * 8 / ((int64_t) n_seq * n_layers) + 1;                 // a wave over all sequences
    if (y > (int64_t) c->table_stride) y = c->table_stride;
    const dim3 grid((unsigned) n_seq, (unsigned) y, (unsigned) n_layers);
    return c->type == SJK_F16 ? launch(bounds_kernel<SJK_F16>, grid, dim3(NT), 0, st, p) : launch(bounds_kernel<SJK_BF16>, grid, dim3(NT), 0, st, p);
}

extern "C" size_t sjk_kv16_select_scratch_bytes(const sjk_kv16 * c, int n_seq) {
    if (check_of(c) || n_seq < 0) return 0;
    return ((size_t) n_seq * c->n_head_kv * c->table_stride + 2) * sizeof(uint64_t);
}

extern "C" int sjk_kv16_select(const sjk_kv16 * c, const void * bounds, const sjk_rows * q, const int32_t * len, const int32_t * rows, int n_seq,
                               int budget, int sink, int recent, int32_t * blocks, int32_t * count, void * scratch, size_t scratch_bytes,
                               sjk_stream st) {
    const int rc = check_of(c);
    if (rc) return rc;
    if (!bounds || !aligned(bounds, 16) || !q || n_seq < 0 || budget < 1 || sink < 0 || recent < 0 || sink > budget || recent > budget - sink) return SJKVARN_ERR_ARG;
    if (!list_ok(len) || !list_ok(rows) || !list_ok(blocks) || !list_ok(count) || !type_ok(q->type) || !rows_ok(*q) || q->n_head < 1 || q->n_head % c->n_head_kv)
        return SJKVARN_ERR_ARG;
    if (n_seq && (!len || !blocks || !q->p)) return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    if (c->n_head_kv > 65535) return SJK_ERR_UNSUPPORTED;
    if (n_seq == 0) return 0;
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < sjk_kv16_select_scratch_bytes(c, n_seq)) return SJKVARN_ERR_BUFFER;
    // the lists of a sequence's other heads are still chosen by its length when one head's are written
    const size_t lens = (size_t) n_seq * sizeof(int32_t), all = lens * c->n_head_kv;
    if (!apart(len, lens, blocks, all * budget) || !apart(len, lens, count, all)) return SJKVARN_ERR_ARG;
    const SelectParams p = {*c, static_cast<const uint16_t *>(bounds), *q, len, rows, n_seq, q->n_head / c->n_head_kv, budget, sink, recent,
                            static_cast<uint64_t *>(scratch), blocks, count};
    const int64_t lists = (int64_t) n_seq * c->n_head_kv, groups = ((int64_t) c->table_stride + NQ / 32 * PG - 1) / (NQ / 32 * PG);
    int64_t z = 148 * 16 / lists + 1;                       // two waves over all lists
    if (z > groups) z = groups;
    const dim3 grid((unsigned) n_seq, (unsigned) c->n_head_kv, (unsigned) z), one((unsigned) n_seq, (unsigned) c->n_head_kv);
    const int rs = c->type == SJK_F16 ? score_launch<SJK_F16>(p, grid, st) : score_launch<SJK_BF16>(p, grid, st);
    if (rs) return rs;
    if (c->table_stride <= 256u * KR) return launch(choose_kernel<256, true>, one, dim3(256), 0, st, p);
    if (c->table_stride <= 1024u * KR) return launch(choose_kernel<1024, true>, one, dim3(1024), 0, st, p);
    return launch(choose_kernel<1024, false>, one, dim3(1024), 0, st, p);
}

// The attention's part of the scratch behind the lists.
static size_t lists_bytes(const sjk_kv16 * c, int n_seq, int budget) {
    return (((size_t) n_seq * c->n_head_kv * ((size_t) budget + 1)) * sizeof(uint32_t) + 15) & ~(size_t) 15;
}

extern "C" size_t sjk_kv16_attend_blocks_scratch_bytes(const sjk_kv16 * c, int n_head, int n_seq, int budget) {
    if (check_of(c) || n_seq < 0 || budget < 1 || c->n_head_kv < 1 || n_head < 1 || n_head % c->n_head_kv) return 0;
    sjk_kv16 one = *c;
    one.n_head_kv = 1;
    const size_t rest = sjk_kv16_attend_scratch_bytes(&one, n_head / c->n_head_kv);
    return rest ? rest + lists_bytes(c, n_seq, budget) : 0;
}

extern "C" int sjk_kv16_attend_blocks(const sjk_kv16 * c, const sjk_rows * q, const int32_t * len, const int32_t * rows, const int32_t * blocks,
                                      int n_seq, int budget, float scale, const sjk_rows * out, void * scratch, size_t scratch_bytes, sjk_stream st) {
    const int rc = check_of(c);
    if (rc) return rc;
    if (!q || !out || n_seq < 0 || budget < 1 || !list_ok(blocks) || !list_ok(len) || !list_ok(rows) || (n_seq && (!len || !blocks))) return SJKVARN_ERR_ARG;
    if (q->n_head < 1 || q->n_head != out->n_head || q->n_head % c->n_head_kv) return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    const int64_t lists = (int64_t) n_seq * c->n_head_kv;
    if (lists > 0x7FFFFFFF / 2) return SJK_ERR_UNSUPPORTED;
    const size_t front = lists_bytes(c, n_seq, budget);
    if (n_seq == 0) return sjk_kv16_attend(c, q, reinterpret_cast<const int32_t *>(c->tables), nullptr, 0, scale, 0, out, nullptr, 0, st);
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < sjk_kv16_attend_blocks_scratch_bytes(c, q->n_head, n_seq, budget)) return SJKVARN_ERR_BUFFER;
    // the lists as sequences of one head each
    sjk_kv16 one = *c;
    one.tables = static_cast<uint32_t *>(scratch);
    one.n_rows = (uint32_t) lists;
    one.table_stride = (uint32_t) budget;
    one.n_head_kv = 1;
    int32_t * lens = reinterpret_cast<int32_t *>(one.tables + lists * budget);
    const int bad = sjk_kv16_attend_folded(&one, c->n_head_kv, q, lens, (int) lists, scale, out, static_cast<uint8_t *>(scratch) + front,
                                           scratch_bytes - front, st, true);
    if (bad) return bad;
    const ListParams p = {*c, len, rows, blocks, n_seq, budget, one.tables, lens};
    const int rl = launch(lists_kernel, dim3((unsigned) ((lists + NT / 32 - 1) / (NT / 32))), dim3(NT), 0, st, p);
    if (rl) return rl;
    return sjk_kv16_attend_folded(&one, c->n_head_kv, q, lens, (int) lists, scale, out, static_cast<uint8_t *>(scratch) + front,
                                  scratch_bytes - front, st, false);
}

int sjk_blocks_status_take(void) {
    unsigned v = 0;
    if (sjk_check(cudaMemcpyFromSymbol(&v, g_blocks_status, sizeof v))) return -1;
    if (v) {
        const unsigned z = 0;
        if (sjk_check(cudaMemcpyToSymbol(g_blocks_status, &z, sizeof z))) return -1;
    }
    return (int) v;
}
