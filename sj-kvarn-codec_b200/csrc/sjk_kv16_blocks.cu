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
// Bound: the bytes of the bounds (4 D a page and KV head) and of the keys (2 D a position and KV head).
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

// grid: sequences, CTAs that take a sequence's pages in turn, layers. A thread has a 16-byte word of a token's key row
// (all heads side by side) and every TG-th token of the page; groups of threads join in shared memory.
template <int TYPE>
__global__ void __launch_bounds__(NT) bounds_kernel(const __grid_constant__ BoundParams p) {
    constexpr int BATCH = 8;
    __shared__ uint4 s_lo[NT], s_hi[NT];
    pdl_wait();
    pdl_release();
    const int i = blockIdx.x, P = p.c.page_tokens, per = p.c.head_dim / 8, words = p.c.n_head_kv * per;
    const uint32_t * table = table_of(p.c, p.rows, i);
    const int first = max(p.first[i], 0), end = fit(p.c, p.end[i]);
    if (!table || first >= end) return;
    const uint16_t * keys = static_cast<const uint16_t *>(p.c.k) + (int64_t) blockIdx.z * p.layer_stride;
    uint4 * out = reinterpret_cast<uint4 *>(p.bounds + (int64_t) blockIdx.z * p.b_layer_stride);
    const int span = words < NT ? words : NT, TG = NT / span, tg = threadIdx.x / span, w0 = threadIdx.x - tg * span;
    const int last = (end - 1) / P;
    for (int g = first / P + (int) blockIdx.y; g <= last; g += (int) gridDim.y) {
        const uint32_t page = table[g];
        if (page >= p.c.n_pages) {
            if (page != SJKVARN_NO_BLOCK) flag();
            continue;
        }
        const int64_t left = (int64_t) end - (int64_t) g * P;
        const int live = (int) (left < P ? left : P);
        for (int wb = 0; wb < words; wb += span) {
            const int w = wb + w0, h = w / per;
            const bool on = tg < TG && w < words;
            const uint16_t * src = keys + (int64_t) page * p.c.page_stride + (int64_t) h * p.c.head_stride + (w - h * per) * 8;
            uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
            if (on) {
                // a thread without a token of its own takes the first one
                lo = hi = *reinterpret_cast<const uint4 *>(src + (int64_t) (tg < live ? tg : 0) * p.c.slot_stride);
                for (int t0 = tg + TG; t0 < live; t0 += BATCH * TG) {
                    uint4 x[BATCH];
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) {
                        const int t = t0 + b * TG;
                        x[b] = *reinterpret_cast<const uint4 *>(src + (int64_t) (t < live ? t : t0) * p.c.slot_stride);
                    }
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) { lo = pick8<TYPE, false>(lo, x[b]); hi = pick8<TYPE, true>(hi, x[b]); }
                }
            }
            if (TG > 1) {
                s_lo[threadIdx.x] = lo;
                s_hi[threadIdx.x] = hi;
                __syncthreads();
                if (tg == 0 && on)
                    for (int q = 1; q < TG; ++q) {
                        lo = pick8<TYPE, false>(lo, s_lo[q * span + w0]);
                        hi = pick8<TYPE, true>(hi, s_hi[q * span + w0]);
                    }
                __syncthreads();
            }
            if (tg == 0 && on) {
                uint4 * dst = out + (int64_t) page * 2 * words + w;
                dst[0] = lo;
                dst[words] = hi;
            }
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

// A warp scores 32 pages of a (sequence, KV head) at a time: a lane has 8 channels of one side (16 where D is 256), and
// 32 partial sums, which an exchange by halves leaves in the lane of each page. grid: sequences, heads, groups of pages.
template <int TYPE, int D>
__global__ void __launch_bounds__(NT) score_kernel(const __grid_constant__ SelectParams p) {
    constexpr int WORDS = D / 8, NW = D == 256 ? 2 : 1;     // words of a side; words of a lane
    constexpr int HALF = D == 64 ? 2 : 1;                   // pages of one load
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, i = blockIdx.x, h = blockIdx.y, P = p.c.page_tokens;
    const int len = fit(p.c, p.len[i]), nb = (int) (((int64_t) len + P - 1) / P);
    const uint32_t * table = table_of(p.c, p.rows, i);
    uint64_t * keys = p.keys + ((int64_t) i * p.c.n_head_kv + h) * p.c.table_stride;
    const int step = (int) gridDim.z * (NT / 32) * 32, b00 = ((int) blockIdx.z * (NT / 32) + (int) (threadIdx.x >> 5)) * 32;
    if (b00 >= nb) return;
    if (!table || nb <= p.budget) {                         // all pages
        for (int b0 = b00; b0 < nb; b0 += step)
            if (b0 + lane < nb) {
                const uint32_t page = table ? table[b0 + lane] : SJKVARN_NO_BLOCK;
                if (page >= p.c.n_pages && page != SJKVARN_NO_BLOCK) flag();
                keys[b0 + lane] = page < p.c.n_pages ? ALWAYS : NEVER;
            }
        return;
    }
    // weights of the lane's channels
    const int sub = HALF == 2 ? lane & 15 : lane;
    const int side = NW == 2 ? 0 : sub / WORDS, c0 = NW == 2 ? lane : sub - side * WORDS;    // (D = 256: a word of both sides)
    const bool on = NW == 2 || sub < 2 * WORDS;
    double wt[NW][8];
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) wt[n][e] = 0.0;
    if (on) {
        const int64_t q0 = (int64_t) i * p.q.row_stride + (int64_t) h * p.grp * p.q.head_stride + c0 * 8;
        for (int g = 0; g < p.grp; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double x = (double) load1(p.q.p, q0 + (int64_t) g * p.q.head_stride + e, p.q.type);
                if (NW == 2) { wt[0][e] += x < 0.0 ? x : 0.0; wt[NW - 1][e] += x > 0.0 ? x : 0.0; }
                else wt[0][e] += side ? (x > 0.0 ? x : 0.0) : (x < 0.0 ? x : 0.0);
                if (x != x) wt[0][e] = x;
            }
#pragma unroll
        for (int n = 0; n < NW; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) wt[n][e] *= weight_by<TYPE>();
    }
    const int64_t row_words = (int64_t) p.c.n_head_kv * WORDS;
    const uint4 * base = reinterpret_cast<const uint4 *>(p.bounds) + (int64_t) h * WORDS + side * row_words + c0;
    for (int b0 = b00; b0 < nb; b0 += step) {
        const int b = b0 + lane;
        uint32_t page = SJKVARN_NO_BLOCK;
        if (b < nb) page = table[b];
        const bool have = page < p.c.n_pages;
        if (!have && page != SJKVARN_NO_BLOCK) flag();
        const uint32_t read = have ? page : 0u;
        double acc[32 / HALF];
#pragma unroll
        for (int u0 = 0; u0 < 32 / HALF; u0 += 8) {
            uint4 x[8][NW];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                // (D = 64: the lower lanes have page u0 + u, the upper ones the one 16 after it)
                const uint32_t at = __shfl_sync(FULL, read, HALF == 2 ? u0 + u + (lane & 16) : u0 + u);
                const uint4 * src = base + (int64_t) at * 2 * row_words;
#pragma unroll
                for (int n = 0; n < NW; ++n) x[u][n] = on ? src[n * row_words] : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                double s = 0.0;
#pragma unroll
                for (int n = 0; n < NW; ++n) {
                    const uint32_t w[4] = {x[u][n].x, x[u][n].y, x[u][n].z, x[u][n].w};
                    if (odd2<TYPE>(w[0]) || odd2<TYPE>(w[1]) || odd2<TYPE>(w[2]) || odd2<TYPE>(w[3])) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 f = widen2<TYPE>(w[e]);
                            s = fma((double) f.x * moved_by<TYPE>(), wt[n][2 * e], s);
                            s = fma((double) f.y * moved_by<TYPE>(), wt[n][2 * e + 1], s);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s = fma(moved<TYPE>(w[e] << 16), wt[n][2 * e], s);
                            s = fma(moved<TYPE>(w[e]), wt[n][2 * e + 1], s);
                        }
                    }
                }
                acc[u0 + u] = s;
            }
        }
        // lane l gets the sum of page l (of its half)
#pragma unroll
        for (int o = 16 / HALF; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < o; ++u) {
                const bool up = lane & o;
                const double send = up ? acc[u] : acc[u + o], keep = up ? acc[u + o] : acc[u];
                acc[u] = keep + __shfl_xor_sync(FULL, send, o);
            }
        if (b < nb) keys[b] = !have ? NEVER : b < p.sink || b >= nb - p.recent ? ALWAYS : order_of(acc[0]);
    }
}

// ---- select: the largest `budget` keys of a list ------------------------------------------------------------------
constexpr int NS = 512;
// Sum over the CTA; every thread gets it. One barrier: successive calls take the places by turns.
SJK_DEV uint32_t cta_sum(uint32_t x, uint32_t (*s)[NS / 32], int turn) {
    x = __reduce_add_sync(FULL, x);
    if ((threadIdx.x & 31) == 0) s[turn & 1][threadIdx.x >> 5] = x;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < NS / 32; ++w) all += s[turn & 1][w];
    return all;
}

// A CTA per (sequence, head): the threshold by bisection over the keys' bits from the first one in which they differ (a
// count of the keys above a middle each time, until exactly `budget` are left), then the keys above it and the first of
// those equal to it, in ascending order of their pages. No atomics: the same lists every time.
__global__ void __launch_bounds__(NS) choose_kernel(const __grid_constant__ SelectParams p, int room) {
    extern __shared__ uint64_t s_keys[];
    __shared__ uint32_t s_sum[2][NS / 32];
    __shared__ uint64_t s_min[NS / 32], s_max[NS / 32];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, i = blockIdx.x, h = blockIdx.y, P = p.c.page_tokens;
    const int64_t list = (int64_t) i * p.c.n_head_kv + h;
    const int len = fit(p.c, p.len[i]), nb = (int) (((int64_t) len + P - 1) / P);
    const uint64_t * far = p.keys + list * p.c.table_stride;
    int32_t * out = p.blocks + list * p.budget;
    const bool near = nb <= room;
    if (near)
        for (int b = tid; b < nb; b += NS) s_keys[b] = far[b];
    __syncthreads();
    const uint64_t * keys = near ? s_keys : far;
    // the keys' range, without the pages that are never chosen
    uint64_t lo = ALWAYS, hi = NEVER;
    uint32_t some = 0;
    for (int b = tid; b < nb; b += NS) {
        const uint64_t k = keys[b];
        if (k == NEVER) continue;
        ++some;
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(FULL, lo, o), b = __shfl_xor_sync(FULL, hi, o);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    if (lane == 0) { s_min[warp] = lo; s_max[warp] = hi; }
    int turn = 0;
    const uint32_t all = cta_sum(some, s_sum, turn++), want = min((uint32_t) p.budget, all);
    for (int w = 0; w < NS / 32; ++w) {
        lo = s_min[w] < lo ? s_min[w] : lo;
        hi = s_max[w] > hi ? s_max[w] : hi;
    }
    // the largest t with at least `want` keys >= t: lo is one such, hi + 1 is none (unless all keys are ALWAYS)
    uint64_t t = lo;
    uint32_t at_t = all;                    // keys >= t
    if (want && all > want) {
        uint64_t top = hi;                  // t <= top
        while (t < top && at_t != want) {
            const uint64_t d = top - t, mid = t + (d >> 1) + (d & 1ull);
            uint32_t n = 0;
            for (int b = tid; b < nb; b += NS) n += keys[b] >= mid ? 1u : 0u;
            n = cta_sum(n, s_sum, turn++);
            if (n >= want) { t = mid; at_t = n; }
            else top = mid - 1ull;
        }
    }
    // keys above t, and the first `ties` of those equal to it: a thread has a run of pages
    const int run = (nb + NS - 1) / NS, b0 = min(tid * run, nb), b1 = min(b0 + run, nb);
    uint32_t above = 0, equal = 0;
    if (want)
        for (int b = b0; b < b1; ++b) {
            const uint64_t k = keys[b];
            above += k > t ? 1u : 0u;
            equal += k == t ? 1u : 0u;
        }
    const uint32_t above_all = cta_sum(above, s_sum, turn++), ties = want - above_all;
    // exclusive sums over the threads, both in one word each
    uint32_t xa = above, xe = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t ya = __shfl_up_sync(FULL, xa, o), ye = __shfl_up_sync(FULL, xe, o);
        if (lane >= o) { xa += ya; xe += ye; }
    }
    __syncthreads();                        // the range's places are free
    if (lane == 31) { s_min[warp] = xa; s_max[warp] = xe; }
    __syncthreads();
    xa -= above;
    xe -= equal;
    for (int w = 0; w < warp; ++w) { xa += (uint32_t) s_min[w]; xe += (uint32_t) s_max[w]; }
    uint32_t at = xa + (xe < ties ? xe : ties);
    if (want)
        for (int b = b0; b < b1; ++b) {
            const uint64_t k = keys[b];
            bool take = k > t;
            if (k == t) take = xe++ < ties;
            if (take) out[at++] = b;
        }
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
        if (!ok && e < p.budget && b != -1) flag();
        const unsigned good = __ballot_sync(FULL, ok);
        const int n = good == FULL ? 32 : __ffs(~good) - 1;      // up to the first that is none
        if (lane < n) pages[e] = table[b];
        count += n;
        if (n) last = __shfl_sync(FULL, b, n - 1);
        if (n < 32) break;
    }
    if (lane == 0) p.lens[list] = count == 0 ? 0 : (int32_t) ((int64_t) (count - 1) * P + (last == nb - 1 ? len - (int64_t) last * P : P));
}

// keys that lie in shared memory, for tables of up to so many pages
int room_of(uint32_t stride) { return (int) (stride < 24576u ? stride : 24576u); }

template <int TYPE>
int score_launch(const SelectParams & p, dim3 grid, sjk_stream st) {
    switch (p.c.head_dim) {
        case 64: return launch(score_kernel<TYPE, 64>, grid, dim3(NT), 0, st, p);
        case 96: return launch(score_kernel<TYPE, 96>, grid, dim3(NT), 0, st, p);
        case 128: return launch(score_kernel<TYPE, 128>, grid, dim3(NT), 0, st, p);
        default: return launch(score_kernel<TYPE, 256>, grid, dim3(NT), 0, st, p);
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
    const SelectParams p = {*c, static_cast<const uint16_t *>(bounds), *q, len, rows, n_seq, q->n_head / c->n_head_kv, budget, sink, recent,
                            static_cast<uint64_t *>(scratch), blocks, count};
    const int64_t lists = (int64_t) n_seq * c->n_head_kv, groups = ((int64_t) c->table_stride + NT - 1) / NT;
    int64_t z = 148 * 8 / lists + 1;
    if (z > groups) z = groups;
    const dim3 grid((unsigned) n_seq, (unsigned) c->n_head_kv, (unsigned) z);
    const int rs = c->type == SJK_F16 ? score_launch<SJK_F16>(p, grid, st) : score_launch<SJK_BF16>(p, grid, st);
    if (rs) return rs;
    const int room = room_of(c->table_stride);
    const size_t smem = (size_t) room * sizeof(uint64_t);
    if (smem > 40 * 1024 && smem_limit<choose_kernel>(24576 * sizeof(uint64_t))) return SJK_ERR_DEVICE;
    return launch(choose_kernel, dim3((unsigned) n_seq, (unsigned) c->n_head_kv), dim3(NS), smem, st, p, room);
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
