// sjk_qkv.cu - from a projection's output to cache rows in one pass: RMS norm of every query and key head, rotary
// positions, and the write of K and V into the pages of a 16-bit cache (or into rows).
//
//   y = x / sqrt(mean x^2 + eps) * (w + norm_bias)
//   (a, b) -> amp (a cos t - b sin t, a sin t + b cos t),  t = pos * f_i
//
// The angle is an integer: pos * step_i modulo 2^64, in units of 2^-64 turns, of which the top 32 bits, read as a
// signed fraction of a turn, go to sincospif as a float: off by 2^-26 of a turn at most (24 bits of half a turn; 1e-7 rad,
// the size of a cosine's own rounding), at every position alike, for one wide multiply.
//
// Bound: HBM, every element once in and once out; a launch's latency for a decode step's few tokens. The vector kernels
// give a lane 16 channels of a head, as 16-byte words that lie side by side over the head's lanes; in the half layout
// its last 8 channels are the partners of its first 8, in the pair layout pairs stay together, so the rotation needs no
// exchange between lanes. The norm's sum is a butterfly over the head's D / 16 lanes (a fixed order). Products of channel
// pairs are packed (f32x2). The cosines and sines of a token are computed once into shared memory for all its heads
// (n_rot / 2 of each per token instead of per head).
//  - Many tokens: a few waves of CTAs, each with a run of tokens that it takes in tiles of up to MAX_T.
//  - Few tokens: a token per CTA and the heads over grid.y (one token of 48 heads of 128 channels: 3.2 us a launch).
// Where n_rot is no multiple of 16 partners are in other lanes: lanes take words of the whole head, and the rotating
// channels go once through shared memory (8,046 tokens of 12 heads of 256 bf16 channels, 20 of them rotating: 26 us; the
// scalar kernel took 93, at five tokens 4.5 against 3.4). Shapes without whole words (head_dim not a multiple of 16,
// rows off 16 bytes) take the scalar kernel, one warp per (token, head) through shared memory.
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

#include <math.h>
#include <type_traits>

namespace {

using namespace sjk16;

constexpr int NT = 256;
constexpr int MAX_T = 16;                   // tokens of a tile, at most
// CTAs of the many-token kernel per SM: 64 registers do for the 16-bit types (prefill of 32,768 tokens 145 us with four,
// 162 with three), floats need 80 (8,320 rows 67 us with three, 76 with four)
constexpr int ctas_of(int type) { return type == SJK_F32 ? 3 : 4; }
// Runs per CTA slot: a run costs about 2.5 us to begin, and SMs are not equally fast. Where a slot moves WAVE_BYTES or more,
// several; below that one. The border is a compromise: head counts and types pull it either way by a few percent (us with
// one / four; MB that a slot moves):
//   floats, 12 heads of 256: 0.5 MB 41.1 / 42.1, 0.6 MB 49.3 / 49.3, 0.75 MB 63.9 / 58.9, 0.9 MB 72.6 / 70.1, 1.6 MB 121.4 / 117.9
//   floats,  6 heads of 256: 0.5 MB 45.0 / 48.2, 0.75 MB 64.6 / 67.2, 0.9 MB 76.8 / 78.7, 1.6 MB 131.4 / 133.3
//   bf16,   12 heads of 256: 0.5 MB 62.9 / 65.8, 0.75 MB 91.9 / 91.7, 1.0 MB 122.3 / 122.9, 1.6 MB 192.5 / 190.4
//   bf16,   24 heads of 256: 0.5 MB 58.0 / 62.6, 0.75 MB 83.7 / 86.1, 1.0 MB 110.1 / 112.1, 1.6 MB 173.3 / 174.0
constexpr int WAVES = 4;
constexpr int64_t WAVE_BYTES = 768 * 1024;
__device__ unsigned int g_qkv_status;

struct Params {
    int n_tok, D, T;
    int n_q, n_k, n_v, n_all;               // heads; n_all their sum
    sjk_rows in[3], out[3];
    const void * w[2];
    int w_type;
    float w_bias, eps, inv_d;
    int n_rot, layout;
    float amp;
    const uint64_t * step;
    const int32_t * pos, * rows;
    sjk_kv16 c;
};

// Element offset of the token's slot in the cache's K and V, or -1 where it has none.
SJK_DEV int64_t cache_slot(const Params & p, int tok, int32_t pos) {
    const int64_t row = p.rows ? (int64_t) p.rows[tok] : (int64_t) tok;
    const uint32_t g = (uint32_t) pos / (uint32_t) p.c.page_tokens;
    if (row >= 0 && row < (int64_t) p.c.n_rows && g < p.c.table_stride) {
        const uint32_t page = p.c.tables[row * p.c.table_stride + g];
        if (page < p.c.n_pages)
            return (int64_t) page * p.c.page_stride + (int64_t) ((uint32_t) pos - g * (uint32_t) p.c.page_tokens) * p.c.slot_stride;
    }
    atomicOr(&g_qkv_status, (unsigned) SJK_DEVICE_PAGE);
    return -1;
}

SJK_DEV float2 angle(uint64_t step, int32_t pos, float amp) {
    const int32_t turn = (int32_t) (uint32_t) (((uint64_t) (uint32_t) pos * step) >> 32);   // in 2^-32 turns
    float s, c;
    sincospif((float) turn * 0x1p-31f, &s, &c);
    return make_float2(c * amp, s * amp);
}

// Which of q, k, v head h (over all heads) belongs to, and its index there.
SJK_DEV int part_of(const Params & p, int h, int * hh) {
    if (h < p.n_q) { *hh = h; return 0; }
    if (h < p.n_q + p.n_k) { *hh = h - p.n_q; return 1; }
    *hh = h - p.n_q - p.n_k;
    return 2;
}

// two floats in one 64-bit register, and their packed products
SJK_DEV uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
SJK_DEV float2 both(uint64_t x) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(x));
    return f;
}
SJK_DEV uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
SJK_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
SJK_DEV uint64_t neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }

// A lane's 16 channels: 16-byte words that lie side by side over the head's lanes, so that every load and store is of
// whole sectors. Region: the rotating channels, or those behind them; the lane's words are a half (16-bit types: two
// words) or a quarter (floats: four) of the region apart. In the half layout the last 8 are the partners of the first 8.
template <int TYPE>
struct Lane {
    static constexpr int N = TYPE == SJK_F32 ? 4 : 2, WORD = 16 / N;    // words, and channels of one
    int first, apart;                       // first channel of word 0, and from word to word
    bool rot, on;                           // rotates; has channels at all
    SJK_DEV Lane(const Params & p, int n_rot, int c) {
        const int nr = n_rot / 16, all = p.D / 16;
        rot = c < nr;
        on = c < all;
        first = rot ? WORD * c : on ? n_rot + WORD * (c - nr) : 0;
        apart = rot ? n_rot / N : on ? (p.D - n_rot) / N : 0;
    }
};

template <int TYPE>
struct Raw { uint4 w[TYPE == SJK_F32 ? 4 : 2]; };

template <int TYPE>
SJK_DEV Raw<TYPE> load16(const void * base, int64_t off, const Lane<TYPE> & l) {
    using E = typename std::conditional<TYPE == SJK_F32, float, uint16_t>::type;
    Raw<TYPE> r;
#pragma unroll
    for (int i = 0; i < Lane<TYPE>::N; ++i) r.w[i] = *reinterpret_cast<const uint4 *>(static_cast<const E *>(base) + off + l.first + i * l.apart);
    return r;
}
template <int TYPE>
SJK_DEV void widen16(const Raw<TYPE> & r, uint64_t (&x)[8]) {
#pragma unroll
    for (int i = 0; i < Lane<TYPE>::N; ++i) {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
        if constexpr (TYPE == SJK_F32) {
            x[2 * i] = two(__uint_as_float(w[0]), __uint_as_float(w[1]));
            x[2 * i + 1] = two(__uint_as_float(w[2]), __uint_as_float(w[3]));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) { const float2 f = widen2<TYPE>(w[k]); x[4 * i + k] = two(f.x, f.y); }
        }
    }
}
// the lane's channels to a row of any type (TYPE is the input's, which chose the channels)
template <int TYPE>
SJK_DEV void store16(void * base, int64_t off, const Lane<TYPE> & l, int type, const uint64_t (&x)[8]) {
    constexpr int N = Lane<TYPE>::N, P = 8 / N;             // words, and channel pairs of one
    off += l.first;
    if (type == SJK_F32) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            ulonglong2 * d = reinterpret_cast<ulonglong2 *>(static_cast<float *>(base) + off + i * l.apart);
#pragma unroll
            for (int k = 0; k < P / 2; ++k) d[k] = make_ulonglong2(x[P * i + 2 * k], x[P * i + 2 * k + 1]);
        }
        return;
    }
    uint32_t w[8];
    if (type == SJK_F16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { const float2 f = both(x[i]); w[i] = pack2<SJK_F16>(f.x, f.y); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) { const float2 f = both(x[i]); w[i] = pack2<SJK_BF16>(f.x, f.y); }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint16_t * d = static_cast<uint16_t *>(base) + off + i * l.apart;
        if constexpr (P == 4) *reinterpret_cast<uint4 *>(d) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        else *reinterpret_cast<uint2 *>(d) = make_uint2(w[2 * i], w[2 * i + 1]);
    }
}

// What the tokens of a tile share: positions, cache slots, and the cosines and sines of every lane's 8 angles, as
// tab[t][4][n_rot / 16]: cosines 0-3, 4-7, sines 0-3, 4-7. ODD (n_rot no multiple of 16): (cosine, sine) by angle.
SJK_DEV int table_words(const Params & p) { return (p.n_rot + 3) / 4; }         // of a token, in 16 bytes
template <int TYPE, bool ODD>
SJK_DEV void tile_table(const Params & p, int t0, int nt, float4 * tab, int32_t * s_pos, int64_t * s_slot) {
    const int tid = threadIdx.x, half = p.n_rot / 2, nr = p.n_rot / 16;
    if (tid < nt) {
        const int32_t pos = p.pos ? p.pos[t0 + tid] : 0;
        s_pos[tid] = pos;
        s_slot[tid] = p.c.k && pos >= 0 ? cache_slot(p, t0 + tid, pos) : -1;
    }
    if (half == 0) return;
    // angles of a word (side by side in the head), as a power of two: a channel each, or in pairs
    const int lw = (TYPE == SJK_F32 ? 2 : 3) - (p.layout == SJK_ROPE_PAIR ? 1 : 0);
    const int dt = NT / half, dj = NT - dt * half;
    for (int t = tid / half, j = tid - t * half; t < nt;) {
        const float2 cs = angle(p.step[j], p.pos[t0 + t], p.amp);
        if constexpr (ODD) {
            reinterpret_cast<float2 *>(tab + (size_t) t * table_words(p))[j] = cs;
        } else {
            int q = 0, k = j;               // word, and angle within the words q of all lanes
            while (k >= nr << lw) { k -= nr << lw; ++q; }
            const int c = k >> lw, e = (q << lw) + (k & ((1 << lw) - 1));
            float * d = reinterpret_cast<float *>(tab + (size_t) t * 4 * nr) + (e >> 2) * nr * 4 + c * 4 + (e & 3);
            d[0] = cs.x;
            d[2 * nr * 4] = cs.y;
        }
        t += dt;
        j += dj;
        if (j >= half) { j -= half; ++t; }
    }
}
SJK_DEV void norm_weights(const Params & p, float * s_w) {
    for (int i = threadIdx.x; i < 2 * p.D; i += NT) {
        const void * w = i < p.D ? p.w[0] : p.w[1];
        if (w) s_w[i] = load1(w, i < p.D ? i : i - p.D, p.w_type) + p.w_bias;
    }
}

// Groups of G neighbouring heads of q, of k and of v, one head per L lanes of a warp: what a warp takes at a time.
template <int L>
struct Groups {
    static constexpr int G = 32 / L;
    int q, k, all;                          // groups of q; of q and k; of all three
    SJK_DEV explicit Groups(const Params & p) {
        q = (p.n_q + G - 1) / G;
        k = q + (p.n_k + G - 1) / G;
        all = k + (p.n_v + G - 1) / G;
    }
};
// A lane's head of group g, and its channels' row for token `tok`.
template <int TYPE, int L>
struct Place {
    int part, hh;
    bool on;
    Raw<TYPE> raw;
    SJK_DEV void load(const Params & p, const Groups<L> & gr, const Lane<TYPE> & l, int g, int tok, bool live) {
        part = g < gr.q ? 0 : g < gr.k ? 1 : 2;
        hh = (g - (part == 0 ? 0 : part == 1 ? gr.q : gr.k)) * Groups<L>::G + (threadIdx.x & 31) / L;
        const sjk_rows & in = part == 0 ? p.in[0] : part == 1 ? p.in[1] : p.in[2];
        on = live && l.on && hh < (part == 0 ? p.n_q : part == 1 ? p.n_k : p.n_v);
        raw = Raw<TYPE>();
        if (on) raw = load16<TYPE>(in.p, (int64_t) tok * in.row_stride + (int64_t) hh * in.head_stride, l);
    }
};

// Norm (NORM) and rotation (ROT) of the lanes' heads for token t of a tile (token `tok` of the call), and their stores.
// ODD: partners are in other lanes, so the rotating channels go through the head's row s_x, where the lanes take a pair
// each. A lane writes and reads its own words there, and others' only between the two barriers.
template <int TYPE, int L, bool NORM, bool ROT, bool ODD>
SJK_DEV void head_row(const Params & p, const Lane<TYPE> & l, int part, int hh, bool on, const Raw<TYPE> & raw, int t, int tok, const float4 * tab0,
                      const float * s_w, float * s_x, const int32_t * s_pos, const int64_t * s_slot) {
    constexpr int N = Lane<TYPE>::N, WORD = Lane<TYPE>::WORD;
    uint64_t a[8];
    widen16<TYPE>(raw, a);
    if constexpr (NORM) {
        uint64_t s0 = mul2(a[0], a[0]), s1 = mul2(a[1], a[1]);          // idle lanes hold zeros
#pragma unroll
        for (int i = 2; i < 8; i += 2) { s0 = fma2(a[i], a[i], s0); s1 = fma2(a[i + 1], a[i + 1], s1); }
        const float2 f0 = both(s0), f1 = both(s1);
        float ss = (f0.x + f0.y) + (f1.x + f1.y);
#pragma unroll
        for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
        const float r = rsqrtf(ss * p.inv_d + p.eps);
        const uint64_t r2 = two(r, r);
        const float * w = s_w + (part ? p.D : 0) + l.first;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < WORD / 4; ++j) {
                const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(w + i * l.apart + 4 * j);
                uint64_t & u = a[i * WORD / 2 + 2 * j], & v = a[i * WORD / 2 + 2 * j + 1];
                u = mul2(u, mul2(r2, y.x));
                v = mul2(v, mul2(r2, y.y));
            }
    }
    if constexpr (ROT && ODD) {
        const int half = p.n_rot / 2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = l.first + i * l.apart;
            if (!l.on || at >= p.n_rot) continue;
#pragma unroll
            for (int j = 0; j < WORD / 4; ++j)
                *reinterpret_cast<ulonglong2 *>(s_x + at + 4 * j) = make_ulonglong2(a[i * WORD / 2 + 2 * j], a[i * WORD / 2 + 2 * j + 1]);
        }
        __syncwarp();
        const float2 * tab = reinterpret_cast<const float2 *>(tab0 + (size_t) t * table_words(p));
        const bool pair = p.layout == SJK_ROPE_PAIR;
        for (int j = threadIdx.x & (L - 1); j < half; j += L) {
            const float2 cs = tab[j];
            const int iu = pair ? 2 * j : j, iv = pair ? 2 * j + 1 : j + half;
            const float u = s_x[iu], v = s_x[iv];
            s_x[iu] = fmaf(u, cs.x, -v * cs.y);
            s_x[iv] = fmaf(v, cs.x, u * cs.y);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = l.first + i * l.apart;
            if (!l.on || at >= p.n_rot) continue;
#pragma unroll
            for (int j = 0; j < WORD / 4; ++j) {
                const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(s_x + at + 4 * j);
                a[i * WORD / 2 + 2 * j] = y.x;
                a[i * WORD / 2 + 2 * j + 1] = y.y;
            }
        }
    } else if (ROT && l.rot) {
        const int nr = p.n_rot / 16;
        const float4 * tab = tab0 + (size_t) t * 4 * nr + (threadIdx.x & (L - 1));
        if (p.layout == SJK_ROPE_HALF) {
            const ulonglong2 c0 = *reinterpret_cast<const ulonglong2 *>(tab), c1 = *reinterpret_cast<const ulonglong2 *>(tab + nr);
            const ulonglong2 s0 = *reinterpret_cast<const ulonglong2 *>(tab + 2 * nr), s1 = *reinterpret_cast<const ulonglong2 *>(tab + 3 * nr);
            const uint64_t cs[4] = {c0.x, c0.y, c1.x, c1.y}, sn[4] = {s0.x, s0.y, s1.x, s1.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t u = a[i], v = a[4 + i];
                a[i] = fma2(u, cs[i], mul2(neg2(v), sn[i]));
                a[4 + i] = fma2(v, cs[i], mul2(u, sn[i]));
            }
        } else {
            const float4 c0 = tab[0], c1 = tab[nr], s0 = tab[2 * nr], s1 = tab[3 * nr];
            const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
            const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 u = both(a[i]);
                a[i] = two(fmaf(u.x, cs[i], -u.y * sn[i]), fmaf(u.y, cs[i], u.x * sn[i]));
            }
        }
    }
    if (!on || s_pos[t] < 0) return;
    const sjk_rows & out = part == 0 ? p.out[0] : part == 1 ? p.out[1] : p.out[2];
    if (out.p) store16<TYPE>(out.p, (int64_t) tok * out.row_stride + (int64_t) hh * out.head_stride, l, out.type, a);
    if (part && s_slot[t] >= 0) store16<TYPE>(part == 1 ? p.c.k : p.c.v, s_slot[t] + (int64_t) hh * p.c.head_stride, l, p.c.type, a);
}
template <int TYPE, int L, bool ODD>
SJK_DEV void head_group(const Params & p, const Lane<TYPE> & l, const Place<TYPE, L> & x, int t, int tok, const float4 * tab, const float * s_w,
                        float * s_x, const int32_t * s_pos, const int64_t * s_slot) {
    if (x.part == 2) head_row<TYPE, L, false, false, ODD>(p, l, 2, x.hh, x.on, x.raw, t, tok, tab, s_w, s_x, s_pos, s_slot);
    else if (x.part == 0 ? p.w[0] : p.w[1]) head_row<TYPE, L, true, true, ODD>(p, l, x.part, x.hh, x.on, x.raw, t, tok, tab, s_w, s_x, s_pos, s_slot);
    else head_row<TYPE, L, false, true, ODD>(p, l, x.part, x.hh, x.on, x.raw, t, tok, tab, s_w, s_x, s_pos, s_slot);
}
// ODD: floats of a head's row, and the row of the lane's head behind the norm weights
SJK_DEV float * head_buffer(const Params & p, float * s_w, int L) {
    return s_w + 2 * p.D + (threadIdx.x / L) * ((p.n_rot + 15) & ~15);
}

// Few tokens. grid.x: tokens; grid.y CTAs share the groups of heads, a warp each. L: lanes of a head, the power of two
// from D / 16 on.
template <int TYPE, int L, bool ODD>
__global__ void __launch_bounds__(NT) qkv_token_kernel(const __grid_constant__ Params p) {
    extern __shared__ float4 s_tab[];       // the table, the norm weights of q and k, and (ODD) a row per head of the warps
    __shared__ int32_t s_pos[1];
    __shared__ int64_t s_slot[1];
    pdl_wait();
    pdl_release();
    float * s_w = reinterpret_cast<float *>(s_tab + table_words(p));
    const int tok = blockIdx.x, g = blockIdx.y * (NT / 32) + threadIdx.x / 32;
    const Groups<L> gr(p);
    const Lane<TYPE> l(p, ODD ? 0 : p.n_rot, threadIdx.x & (L - 1));
    Place<TYPE, L> x;
    x.load(p, gr, l, g, tok, g < gr.all);
    tile_table<TYPE, ODD>(p, tok, 1, s_tab, s_pos, s_slot);
    if (p.w[0] || p.w[1]) norm_weights(p, s_w);
    __syncthreads();
    if (g < gr.all) head_group<TYPE, L, ODD>(p, l, x, 0, tok, s_tab, s_w, head_buffer(p, s_w, L), s_pos, s_slot);
}

// Many tokens. A CTA has the tokens [n i / ctas, n (i + 1) / ctas), in tiles of T; the table of the next tile is made
// while one is worked on. Its warps take the groups of a token's heads in turn, so that the CTA goes through its rows in
// the order of memory, with the next item's loads out while one is worked on (32,768 tokens of 24 heads of 256 bf16
// channels: 145 us = 5.5 TB/s of rows read and written, 85 % of a plain copy's rate, bound by instruction issue; 8,320
// rows of floats 67 us = 6.1 TB/s, 93 %). Staying with a head over the tile's tokens took 160 us, several tokens per item
// 217 and more: both need registers that four CTAs an SM do not have.
template <int TYPE, int L, bool ODD>
__global__ void __launch_bounds__(NT, ctas_of(TYPE)) qkv_tile_kernel(const __grid_constant__ Params p) {
    extern __shared__ float4 s_tab[];       // two tables, the norm weights of q and k, and (ODD) a row per head of the warps
    __shared__ int32_t s_pos[2][MAX_T];
    __shared__ int64_t s_slot[2][MAX_T];
    pdl_wait();
    pdl_release();
    constexpr int WARPS = NT / 32;
    const int one = p.T * table_words(p);
    float * s_w = reinterpret_cast<float *>(s_tab + 2 * one);
    const Groups<L> gr(p);
    const Lane<TYPE> l(p, ODD ? 0 : p.n_rot, threadIdx.x & (L - 1));
    if (p.w[0] || p.w[1]) norm_weights(p, s_w);
    const int last = (int) ((int64_t) p.n_tok * (blockIdx.x + 1) / gridDim.x), warp = threadIdx.x / 32;
    int t0 = (int) ((int64_t) p.n_tok * blockIdx.x / gridDim.x);
    if (t0 < last) tile_table<TYPE, ODD>(p, t0, min(p.T, last - t0), s_tab, s_pos[0], s_slot[0]);
    // the warp's next item: token (of the CTA's) and group, and its rows
    int tok = t0, g = warp;
    while (g >= gr.all) { g -= gr.all; ++tok; }
    Place<TYPE, L> x;
    x.load(p, gr, l, g, tok, tok < last);
    for (int s = 0; t0 < last; t0 += p.T, s ^= 1) {
        const int end = min(t0 + p.T, last), next = t0 + p.T;
        __syncthreads();                    // this tile's table is complete, the other one is free
        if (next < last) tile_table<TYPE, ODD>(p, next, min(p.T, last - next), s_tab + (s ? 0 : one), s_pos[s ^ 1], s_slot[s ^ 1]);
        while (tok < end) {
            const Place<TYPE, L> y = x;
            const int now = tok;
            g += WARPS;
            while (g >= gr.all) { g -= gr.all; ++tok; }
            x.load(p, gr, l, g, tok, tok < last);
            head_group<TYPE, L, ODD>(p, l, y, now - t0, now, s_tab + (s ? one : 0), s_w, head_buffer(p, s_w, L), s_pos[s], s_slot[s]);
        }
    }
}

// Any shape and alignment: a warp per (token, head), the row in shared memory between the norm and the rotation.
__global__ void __launch_bounds__(NT) qkv_scalar_kernel(const __grid_constant__ Params p) {
    extern __shared__ float s_rows[];       // [NT / 32][D]
    pdl_wait();
    pdl_release();
    const int lane = threadIdx.x & 31, D = p.D;
    float * x = s_rows + (threadIdx.x >> 5) * D;
    const int64_t n = (int64_t) p.n_tok * p.n_all;
    for (int64_t i = (int64_t) blockIdx.x * (NT / 32) + (threadIdx.x >> 5); i < n; i += (int64_t) gridDim.x * (NT / 32)) {
        const int tok = (int) (i / p.n_all);
        int hh;
        const int part = part_of(p, (int) (i - (int64_t) tok * p.n_all), &hh);
        const int32_t pos = p.pos ? p.pos[tok] : 0;
        if (pos < 0) continue;
        const sjk_rows & in = p.in[part];
        const sjk_rows & out = p.out[part];
        const int64_t src = (int64_t) tok * in.row_stride + (int64_t) hh * in.head_stride;
        const void * w = part < 2 ? p.w[part] : nullptr;
        float ss = 0.0f;
        for (int d = lane; d < D; d += 32) {
            const float v = load1(in.p, src + d, in.type);
            x[d] = v;
            ss = fmaf(v, v, ss);
        }
        if (w) {
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
            const float r = rsqrtf(ss * p.inv_d + p.eps);
            for (int d = lane; d < D; d += 32) x[d] *= r * (load1(w, d, p.w_type) + p.w_bias);
        }
        __syncwarp();
        if (part < 2) {
            const int half = p.n_rot / 2;
            for (int j = lane; j < half; j += 32) {
                const float2 cs = angle(p.step[j], pos, p.amp);
                const int ia = p.layout == SJK_ROPE_HALF ? j : 2 * j, ib = p.layout == SJK_ROPE_HALF ? j + half : 2 * j + 1;
                const float a = x[ia], b = x[ib];
                x[ia] = a * cs.x - b * cs.y;
                x[ib] = a * cs.y + b * cs.x;
            }
            __syncwarp();
        }
        if (out.p) {
            const int64_t dst = (int64_t) tok * out.row_stride + (int64_t) hh * out.head_stride;
            for (int d = lane; d < D; d += 32) store1(out.p, dst + d, out.type, x[d]);
        }
        if (part && p.c.k) {
            const int64_t slot = cache_slot(p, tok, pos);
            if (slot >= 0) {
                void * base = part == 1 ? p.c.k : p.c.v;
                for (int d = lane; d < D; d += 32) store1(base, slot + (int64_t) hh * p.c.head_stride + d, p.c.type, x[d]);
            }
        }
        __syncwarp();
    }
}

template <int TYPE, int L, bool ODD>
int launch_vec(sjk_stream st, Params & p) {
    const size_t table = (size_t) ((p.n_rot + 3) / 4) * 16;             // of a token
    const size_t rest = 2 * (size_t) p.D * sizeof(float) + (ODD ? (size_t) (NT / L) * ((p.n_rot + 15) & ~15) * sizeof(float) : 0);
    constexpr int slots = 148 * ctas_of(TYPE);
    if (p.n_tok >= slots) {
        // rows read and written: their types are near enough the input's
        const int64_t bytes = (int64_t) p.n_tok * p.n_all * p.D * (2 * (int) type_bytes(TYPE));
        const int waves = bytes / slots < WAVE_BYTES || p.n_tok < 4 * WAVES * slots ? 1 : WAVES;    // (four tokens of a run, at least)
        const int ctas = slots * waves, run = (p.n_tok + ctas - 1) / ctas, tiles = (run + MAX_T - 1) / MAX_T;
        p.T = (run + tiles - 1) / tiles;
        const size_t smem = 2 * (size_t) p.T * table + rest;
        // (the rows of a CTA's heads hold at most the 16 channels of every thread)
        if (smem > 47 * 1024 && smem_limit<qkv_tile_kernel<TYPE, L, ODD>>(2 * (size_t) MAX_T * 512 * sizeof(float) + 4096 + (ODD ? NT * 64 : 0)))
            return SJK_ERR_DEVICE;
        return launch(qkv_tile_kernel<TYPE, L, ODD>, dim3((unsigned) ctas), dim3(NT), smem, st, p);
    }
    p.T = 1;
    constexpr int G = 32 / L;
    const int groups = (p.n_q + G - 1) / G + (p.n_k + G - 1) / G + (p.n_v + G - 1) / G;
    const dim3 grid((unsigned) p.n_tok, (unsigned) ((groups + NT / 32 - 1) / (NT / 32)));
    return launch(qkv_token_kernel<TYPE, L, ODD>, grid, dim3(NT), table + rest, st, p);
}
template <int TYPE, bool ODD>
int launch_lanes(sjk_stream st, Params & p) {
    return p.D <= 16 ? launch_vec<TYPE, 1, ODD>(st, p) : p.D <= 32 ? launch_vec<TYPE, 2, ODD>(st, p) :
           p.D <= 64 ? launch_vec<TYPE, 4, ODD>(st, p) : p.D <= 128 ? launch_vec<TYPE, 8, ODD>(st, p) :
           p.D <= 256 ? launch_vec<TYPE, 16, ODD>(st, p) : launch_vec<TYPE, 32, ODD>(st, p);
}
template <int TYPE>
int launch_type(sjk_stream st, Params & p) {
    return p.n_rot % 16 ? launch_lanes<TYPE, true>(st, p) : launch_lanes<TYPE, false>(st, p);
}

bool rows_vec(const sjk_rows & r) {
    if (!r.p) return true;
    const int64_t q = (int64_t) (16 / type_bytes(r.type)) - 1;      // strides in whole 16-byte words
    return aligned(r.p, 16) && (r.row_stride & q) == 0 && (r.head_stride & q) == 0;
}

// The fractions of a turn per position, in 64-bit mantissas (long double).
int rope_check(const sjk_rope_config * c) {
    if (!c || c->n_rot < 2 || c->n_rot > 512 || (c->n_rot & 1)) return SJKVARN_ERR_ARG;
    if (c->layout != SJK_ROPE_HALF && c->layout != SJK_ROPE_PAIR) return SJKVARN_ERR_ARG;
    if (c->scaling < SJK_ROPE_NONE || c->scaling > SJK_ROPE_BANDS) return SJKVARN_ERR_ARG;
    if (!(c->base > 1.0) || !isfinite(c->base) || !(c->amp >= 0.0) || !isfinite(c->amp)) return SJKVARN_ERR_ARG;
    if (c->scaling != SJK_ROPE_NONE && (!(c->factor > 0.0) || !isfinite(c->factor))) return SJKVARN_ERR_ARG;
    if (c->scaling == SJK_ROPE_YARN && (!(c->n_ctx > 0.0) || !isfinite(c->n_ctx) || !(c->beta_slow > 0.0) || !(c->beta_fast >= c->beta_slow) || !isfinite(c->beta_fast)))
        return SJKVARN_ERR_ARG;
    if (c->scaling == SJK_ROPE_BANDS && (!(c->n_ctx > 0.0) || !isfinite(c->n_ctx) || !(c->low > 0.0) || !(c->high > c->low) || !isfinite(c->high)))
        return SJKVARN_ERR_ARG;
    return 0;
}

}  // namespace

extern "C" int sjk_rope_steps(const sjk_rope_config * c, uint64_t * step, float * amp) {
    const int rc = rope_check(c);
    if (rc || !step || !amp) return SJKVARN_ERR_ARG;
    const long double two_pi = 6.283185307179586476925286766559005768L;
    const int n = c->n_rot;
    long double base = c->base;
    const long double f = c->scaling == SJK_ROPE_NONE ? 1.0L : (long double) c->factor;
    if (c->scaling == SJK_ROPE_NTK && n > 2) base *= powl(f, (long double) n / (n - 2));
    long double lo = 0.0L, hi = 0.0L;
    if (c->scaling == SJK_ROPE_YARN) {
        lo = floorl(n * logl(c->n_ctx / (c->beta_fast * two_pi)) / (2.0L * logl(base)));
        hi = ceill(n * logl(c->n_ctx / (c->beta_slow * two_pi)) / (2.0L * logl(base)));
        if (lo < 0.0L) lo = 0.0L;
        if (hi > n - 1) hi = n - 1;
    }
    for (int i = 0; i < n / 2; ++i) {
        long double w = powl(base, -2.0L * i / n);
        if (c->scaling == SJK_ROPE_LINEAR) w /= f;
        if (c->scaling == SJK_ROPE_YARN) {
            const long double span = hi - lo > 0.001L ? hi - lo : 0.001L;
            long double r = (i - lo) / span;
            r = r < 0.0L ? 0.0L : r > 1.0L ? 1.0L : r;
            w = w / f * r + w * (1.0L - r);
        }
        if (c->scaling == SJK_ROPE_BANDS) {
            long double s = (c->n_ctx * w / two_pi - c->low) / ((long double) c->high - c->low);
            s = s < 0.0L ? 0.0L : s > 1.0L ? 1.0L : s;
            w = w / f * (1.0L - s) + w * s;
        }
        const long double turn = fmodl(w / two_pi, 1.0L);
        const long double u = roundl(turn * 18446744073709551616.0L);
        step[i] = u >= 18446744073709551616.0L ? 0u : (uint64_t) u;
    }
    *amp = c->amp != 0.0 ? (float) c->amp : c->scaling == SJK_ROPE_YARN && c->factor > 1.0 ? (float) (0.1 * log(c->factor) + 1.0) : 1.0f;
    return 0;
}

extern "C" int sjk_rope_init(sjk_rope * r, const sjk_rope_config * c) {
    if (!r) return SJKVARN_ERR_ARG;
    uint64_t step[256];
    float amp;
    r->n_rot = 0; r->layout = 0; r->amp = 0.0f; r->step = nullptr;
    const int rc = sjk_rope_steps(c, step, &amp);
    if (rc) return rc;
    const size_t bytes = (size_t) (c->n_rot / 2) * sizeof(uint64_t);
    void * d = nullptr;
    if (cudaMalloc(&d, bytes) != cudaSuccess) { cudaGetLastError(); return SJKVARN_ERR_NOMEM; }
    if (sjk_check(cudaMemcpy(d, step, bytes, cudaMemcpyHostToDevice))) { cudaFree(d); return SJK_ERR_DEVICE; }
    r->n_rot = c->n_rot;
    r->layout = c->layout;
    r->amp = amp;
    r->step = static_cast<uint64_t *>(d);
    return 0;
}

extern "C" void sjk_rope_free(sjk_rope * r) {
    if (!r) return;
    if (r->step) cudaFree(r->step);
    r->step = nullptr;
    r->n_rot = 0;
}

int sjk_kv16_check(const sjk_kv16 * c) {
    if (!c->k || !c->v || !c->tables || !aligned(c->k, 2) || !aligned(c->v, 2) || !aligned(c->tables, 4) || c->page_tokens < 1 || c->n_head_kv < 1 || c->head_dim < 1 || c->n_pages < 1 ||
        c->n_pages >= SJKVARN_NO_BLOCK || c->n_rows < 1 || c->table_stride < 1 || (c->type != SJK_F16 && c->type != SJK_BF16) ||
        c->page_stride < 0 || c->slot_stride < 0 || c->head_stride < 0)
        return SJKVARN_ERR_ARG;
    return 0;
}

extern "C" int sjk_qkv(const sjk_qkv_args * a, sjk_stream st) {
    if (!a || a->n_tok < 0) return SJKVARN_ERR_ARG;
    if (a->head_dim < 2 || a->head_dim > 512 || (a->head_dim & 1)) return SJKVARN_ERR_HEAD_DIM;
    Params p = {};
    const sjk_rows in[3] = {a->q, a->k, a->v}, out[3] = {a->q_out, a->k_out, a->v_out};
    const bool cached = a->cache.k || a->cache.v;
    if (cached) {
        if (sjk_kv16_check(&a->cache)) return SJKVARN_ERR_ARG;
        if (a->cache.head_dim != a->head_dim || !a->k.p || !a->v.p || a->k.n_head != a->cache.n_head_kv || a->v.n_head != a->cache.n_head_kv)
            return SJKVARN_ERR_ARG;
        if (!a->rows && (int64_t) a->n_tok > (int64_t) a->cache.n_rows) return SJKVARN_ERR_ARG;
    }
    int type = -1, n[3];
    for (int i = 0; i < 3; ++i) {
        n[i] = 0;
        if (!in[i].p) {
            if (out[i].p) return SJKVARN_ERR_ARG;
            continue;
        }
        if (in[i].n_head < 1 || in[i].n_head > 65535 || !type_ok(in[i].type) || !rows_ok(in[i]) || (type >= 0 && in[i].type != type)) return SJKVARN_ERR_ARG;
        type = in[i].type;
        if (out[i].p && (out[i].n_head != in[i].n_head || !type_ok(out[i].type) || !rows_ok(out[i]))) return SJKVARN_ERR_ARG;
        // rows in place: an element has to stay where it was read
        if (out[i].p == in[i].p && (out[i].type != type || out[i].row_stride != in[i].row_stride || out[i].head_stride != in[i].head_stride))
            return SJKVARN_ERR_ARG;
        if (out[i].p || (cached && i > 0)) n[i] = in[i].n_head;       // heads that nobody wants are not read
        p.in[i] = in[i];
        p.out[i] = out[i];
    }
    if (type < 0) return SJKVARN_ERR_ARG;
    if ((a->q_norm || a->k_norm) && (!type_ok(a->norm_type) || !(a->eps >= 0.0f) || !isfinite(a->eps))) return SJKVARN_ERR_ARG;
    for (const void * w : {a->q_norm, a->k_norm})
        if (w && !aligned(w, type_bytes(a->norm_type))) return SJKVARN_ERR_ARG;
    const bool rope = a->rope.n_rot != 0;
    if (rope && (a->rope.n_rot < 2 || (a->rope.n_rot & 1) || a->rope.n_rot > a->head_dim || !a->rope.step || !aligned(a->rope.step, 8) ||
                 (a->rope.layout != SJK_ROPE_HALF && a->rope.layout != SJK_ROPE_PAIR)))
        return SJKVARN_ERR_ROTATION;
    if (((rope || cached) && !a->pos) || !list_ok(a->pos) || !list_ok(a->rows)) return SJKVARN_ERR_ARG;
    if (a->n_tok == 0) return 0;
    p.n_tok = a->n_tok; p.D = a->head_dim;
    p.n_q = n[0]; p.n_k = n[1]; p.n_v = n[2];
    p.n_all = n[0] + n[1] + n[2];
    if (p.n_all == 0) return 0;
    p.w[0] = a->q_norm; p.w[1] = a->k_norm;
    p.w_type = a->norm_type; p.w_bias = a->norm_bias; p.eps = a->eps; p.inv_d = 1.0f / (float) a->head_dim;
    p.n_rot = a->rope.n_rot; p.layout = a->rope.layout; p.amp = a->rope.amp; p.step = a->rope.step;
    p.pos = a->pos; p.rows = a->rows;
    if (cached) p.c = a->cache;
    bool vec = p.D % 16 == 0;
    for (int i = 0; i < 3; ++i) vec = vec && rows_vec(p.in[i]) && rows_vec(p.out[i]);
    if (cached) {
        const int64_t s = p.c.page_stride | p.c.slot_stride | p.c.head_stride;
        vec = vec && aligned(p.c.k, 16) && aligned(p.c.v, 16) && (s & 7) == 0;
    }
    if (!vec) {
        const int64_t warps = (int64_t) p.n_tok * p.n_all, ctas = (warps + NT / 32 - 1) / (NT / 32);
        return launch(qkv_scalar_kernel, dim3((unsigned) (ctas < 148 * 8 ? ctas : 148 * 8)), dim3(NT), (size_t) (NT / 32) * p.D * sizeof(float), st, p);
    }
    switch (type) {
        case SJK_F32: return launch_type<SJK_F32>(st, p);
        case SJK_F16: return launch_type<SJK_F16>(st, p);
        default: return launch_type<SJK_BF16>(st, p);
    }
}

int sjk_qkv_status_take(void) {
    unsigned v = 0;
    if (sjk_check(cudaMemcpyFromSymbol(&v, g_qkv_status, sizeof v))) return -1;
    if (v) {
        const unsigned z = 0;
        if (sjk_check(cudaMemcpyToSymbol(g_qkv_status, &z, sizeof z))) return -1;
    }
    return (int) v;
}
