// sjk_qkv.cu - from a projection's output to cache rows in one pass: RMS norm of every query and key head, rotary
// positions, and the write of K and V into the pages of a 16-bit cache (or into rows).
//
//   y = x / sqrt(mean x^2 + eps) * (w + norm_bias)
//   (a, b) -> amp (a cos t - b sin t, a sin t + b cos t),  t = pos * f_i
//
// The angle is an integer: pos * step_i modulo 2^64, in units of 2^-64 turns, of which the top 32 bits, read as a
// signed fraction of a turn, go to sincospif. That keeps 2^-32 of a turn at every position, for one wide multiply.
//
// Bound: HBM, every element once in and once out. The vector kernel gives a lane 16 channels of a head: for the half
// layout the two 8-channel chunks that rotate into one another, so the rotation needs no exchange between lanes, and
// the norm's sum is a butterfly over the head's D / 16 lanes (a fixed order). A CTA works on T tokens: their cosines
// and sines are computed once into shared memory for all heads (n_rot / 2 sincos per token instead of per head), and
// every lane keeps its channels and its head over the tokens, so that norm weights are loaded once per head.
// Shapes whose chunks would straddle (n_rot or head_dim not a multiple of 16, rows off 16 bytes) take the scalar
// kernel, one warp per (token, head) through shared memory.
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

#include <math.h>

namespace {

using namespace sjk16;

constexpr int NT = 256;
constexpr int MAX_T = 32;                   // tokens of a CTA, at most
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

template <int TYPE>
struct Raw { uint4 a, b; };                 // 8 channels: 16 bytes, or 32 for floats

template <int TYPE>
SJK_DEV Raw<TYPE> load8(const void * base, int64_t off) {
    Raw<TYPE> r;
    if constexpr (TYPE == SJK_F32) {
        const uint4 * s = reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + off);
        r.a = s[0]; r.b = s[1];
    } else {
        r.a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + off);
    }
    return r;
}
template <int TYPE>
SJK_DEV void widen8(const Raw<TYPE> & r, float (&x)[8]) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    if constexpr (TYPE == SJK_F32) {
        const uint32_t u[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = __uint_as_float(w[i]); x[4 + i] = __uint_as_float(u[i]); }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = widen2<TYPE>(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
}
template <int TYPE>
SJK_DEV uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack2<TYPE>(x[0], x[1]), pack2<TYPE>(x[2], x[3]), pack2<TYPE>(x[4], x[5]), pack2<TYPE>(x[6], x[7]));
}
SJK_DEV void store16(void * base, int64_t off, int d0, int d1, int type, const float (&a)[8], const float (&b)[8]) {
    if (type == SJK_F32) {
        float * x = static_cast<float *>(base) + off;
        float4 * u = reinterpret_cast<float4 *>(x + d0), * v = reinterpret_cast<float4 *>(x + d1);
        u[0] = make_float4(a[0], a[1], a[2], a[3]);
        u[1] = make_float4(a[4], a[5], a[6], a[7]);
        v[0] = make_float4(b[0], b[1], b[2], b[3]);
        v[1] = make_float4(b[4], b[5], b[6], b[7]);
    } else {
        uint16_t * x = static_cast<uint16_t *>(base) + off;
        uint4 u, v;
        if (type == SJK_F16) { u = pack8<SJK_F16>(a); v = pack8<SJK_F16>(b); }
        else { u = pack8<SJK_BF16>(a); v = pack8<SJK_BF16>(b); }
        *reinterpret_cast<uint4 *>(x + d0) = u;
        *reinterpret_cast<uint4 *>(x + d1) = v;
    }
}

// Lane c of a head: its two chunks' first channels, and whether they rotate.
SJK_DEV bool lane_chunks(const Params & p, int c, int * d0, int * d1) {
    const int nr = p.n_rot / 16;
    const bool rot = c < nr;
    if (p.layout == SJK_ROPE_HALF && rot) { *d0 = 8 * c; *d1 = p.n_rot / 2 + 8 * c; }
    else { *d0 = 16 * c; *d1 = 16 * c + 8; }
    return rot;
}

// The tokens of blocks [ka, kb) of a tile in one head of q, k or v: norm (NORM) and rotation (ROT). A block is a token
// for each of the warp's groups of L lanes; the loads of the next block are out while one is worked on.
template <int TYPE, int L, bool NORM, bool ROT>
SJK_DEV void head_tokens(const Params & p, int part, int hh, int t0, int nt, int ka, int kb, const float4 * s_tab, const float * s_w,
                         const int32_t * s_pos, const int64_t * s_slot) {
    const sjk_rows & in = part == 0 ? p.in[0] : part == 1 ? p.in[1] : p.in[2];
    const sjk_rows & out = part == 0 ? p.out[0] : part == 1 ? p.out[1] : p.out[2];
    void * cache = part == 0 ? nullptr : part == 1 ? p.c.k : p.c.v;
    const int c = threadIdx.x & (L - 1), nr = p.n_rot / 16;
    int d0, d1;
    const bool rot = lane_chunks(p, c, &d0, &d1) && ROT;
    const bool on = 16 * L == p.D || 16 * c < p.D;
    constexpr int G = 32 / L;
    int t = ka * G + (threadIdx.x & 31) / L;
    const int end = min(nt, kb * G);
    int64_t src = (int64_t) (t0 + t) * in.row_stride + (int64_t) hh * in.head_stride;
    int64_t dst = (int64_t) (t0 + t) * out.row_stride + (int64_t) hh * out.head_stride;
    const int64_t head = (int64_t) hh * p.c.head_stride;
    float w0[8], w1[8];
    if constexpr (NORM) {
        const float4 * w = reinterpret_cast<const float4 *>(s_w + (part ? p.D : 0));
        const float4 x[4] = {w[d0 / 4 * on], w[(d0 / 4 + 1) * on], w[d1 / 4 * on], w[(d1 / 4 + 1) * on]};
        w0[0] = x[0].x; w0[1] = x[0].y; w0[2] = x[0].z; w0[3] = x[0].w; w0[4] = x[1].x; w0[5] = x[1].y; w0[6] = x[1].z; w0[7] = x[1].w;
        w1[0] = x[2].x; w1[1] = x[2].y; w1[2] = x[2].z; w1[3] = x[2].w; w1[4] = x[3].x; w1[5] = x[3].y; w1[6] = x[3].z; w1[7] = x[3].w;
    }
    Raw<TYPE> ra = {}, rb = {};
    if (on && t < end) { ra = load8<TYPE>(in.p, src + d0); rb = load8<TYPE>(in.p, src + d1); }
    for (int k = ka; k < kb; ++k, t += G) {
        float a[8], b[8];
        widen8<TYPE>(ra, a);
        widen8<TYPE>(rb, b);
        src += G * in.row_stride;
        if (on && t + G < end) { ra = load8<TYPE>(in.p, src + d0); rb = load8<TYPE>(in.p, src + d1); }
        if constexpr (NORM) {
            float s0 = 0.0f, s1 = 0.0f;     // idle lanes hold zeros
#pragma unroll
            for (int i = 0; i < 8; ++i) { s0 = fmaf(a[i], a[i], s0); s1 = fmaf(b[i], b[i], s1); }
            float ss = s0 + s1;
#pragma unroll
            for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
            const float r = rsqrtf(ss * p.inv_d + p.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) { a[i] *= r * w0[i]; b[i] *= r * w1[i]; }
        }
        if (t >= end) break;                // (its groups' last tokens; the sums above needed all lanes)
        if (rot) {
            const float4 * tab = s_tab + (size_t) t * 4 * nr + c;
            const float4 c0 = tab[0], c1 = tab[nr], s0 = tab[2 * nr], s1 = tab[3 * nr];
            const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
            const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
            if (p.layout == SJK_ROPE_HALF) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = a[i], y = b[i];
                    a[i] = x * cs[i] - y * sn[i];
                    b[i] = x * sn[i] + y * cs[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = a[2 * i], y = a[2 * i + 1];
                    a[2 * i] = x * cs[i] - y * sn[i];
                    a[2 * i + 1] = x * sn[i] + y * cs[i];
                    x = b[2 * i]; y = b[2 * i + 1];
                    b[2 * i] = x * cs[4 + i] - y * sn[4 + i];
                    b[2 * i + 1] = x * sn[4 + i] + y * cs[4 + i];
                }
            }
        }
        const bool live = on && s_pos[t] >= 0;
        if (live && out.p) store16(out.p, dst, d0, d1, out.type, a, b);
        if (live && cache && s_slot[t] >= 0) store16(cache, s_slot[t] + head, d0, d1, p.c.type, a, b);
        dst += G * out.row_stride;
    }
}

// grid.x: tiles of T tokens; grid.y CTAs share a tile's heads. L: lanes of a head, the power of two from D / 16 on.
// The (head, block of tokens) items of a tile, in the order of heads, are cut into equal runs, one per warp: its groups of L
// lanes work on as many tokens of the same head.
template <int TYPE, int L>
__global__ void __launch_bounds__(NT, 3) qkv_vec_kernel(const __grid_constant__ Params p) {
    extern __shared__ float4 s_tab[];       // [T][4][n_rot / 16]: cosines 0-3, 4-7, sines 0-3, 4-7 of a lane's 8 angles,
    __shared__ int32_t s_pos[MAX_T];        // then the norm weights of q and k
    __shared__ int64_t s_slot[MAX_T];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, t0 = blockIdx.x * p.T, nt = min(p.T, p.n_tok - t0);
    const int half = p.n_rot / 2, nr = p.n_rot / 16;
    float * s_w = reinterpret_cast<float *>(s_tab + p.T * 4 * nr);
    if (tid < nt) {
        const int32_t pos = p.pos ? p.pos[t0 + tid] : 0;
        s_pos[tid] = pos;
        s_slot[tid] = p.c.k && pos >= 0 ? cache_slot(p, t0 + tid, pos) : -1;
    }
    for (int i = tid; i < 2 * p.D; i += NT) {
        const void * w = i < p.D ? p.w[0] : p.w[1];
        if (w) s_w[i] = load1(w, i < p.D ? i : i - p.D, p.w_type) + p.w_bias;
    }
    for (int i = tid; i < nt * half; i += NT) {
        const int t = i / half, j = i - t * half, c = j >> 3, e = j & 7;
        const float2 cs = angle(p.step[j], p.pos[t0 + t], p.amp);
        float * d = reinterpret_cast<float *>(s_tab + (size_t) t * 4 * nr);
        d[((e >> 2) * nr + c) * 4 + (e & 3)] = cs.x;
        d[((2 + (e >> 2)) * nr + c) * 4 + (e & 3)] = cs.y;
    }
    __syncthreads();
    constexpr int G = 32 / L, WARPS = NT / 32;
    const int blocks = (nt + G - 1) / G, items = blocks * p.n_all;
    const int each = (items + WARPS * (int) gridDim.y - 1) / (WARPS * (int) gridDim.y);
    int item = ((int) blockIdx.y * WARPS + tid / 32) * each;
    const int end = min(item + each, items);
    while (item < end) {
        const int h = item / blocks, ka = item - h * blocks, kb = min(blocks, ka + end - item);
        int hh;
        const int part = part_of(p, h, &hh);
        if (part == 2) head_tokens<TYPE, L, false, false>(p, part, hh, t0, nt, ka, kb, s_tab, s_w, s_pos, s_slot);
        else if (part == 0 ? p.w[0] : p.w[1]) head_tokens<TYPE, L, true, true>(p, part, hh, t0, nt, ka, kb, s_tab, s_w, s_pos, s_slot);
        else head_tokens<TYPE, L, false, true>(p, part, hh, t0, nt, ka, kb, s_tab, s_w, s_pos, s_slot);
        item += kb - ka;
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

template <int TYPE>
int launch_vec(int L, dim3 grid, size_t smem, sjk_stream st, const Params & p) {
    switch (L) {
        case 1: return launch(qkv_vec_kernel<TYPE, 1>, grid, dim3(NT), smem, st, p);
        case 2: return launch(qkv_vec_kernel<TYPE, 2>, grid, dim3(NT), smem, st, p);
        case 4: return launch(qkv_vec_kernel<TYPE, 4>, grid, dim3(NT), smem, st, p);
        case 8: return launch(qkv_vec_kernel<TYPE, 8>, grid, dim3(NT), smem, st, p);
        case 16: return launch(qkv_vec_kernel<TYPE, 16>, grid, dim3(NT), smem, st, p);
        default: return launch(qkv_vec_kernel<TYPE, 32>, grid, dim3(NT), smem, st, p);
    }
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
    *amp = c->amp != 0.0 ? (float) c->amp : c->scaling == SJK_ROPE_YARN ? (float) (0.1 * log(c->factor) + 1.0) : 1.0f;
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
    if (!c->k || !c->v || !c->tables || c->page_tokens < 1 || c->n_head_kv < 1 || c->head_dim < 1 || c->n_pages < 1 ||
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
        if (in[i].n_head < 1 || in[i].n_head > 65535 || !type_ok(in[i].type) || (type >= 0 && in[i].type != type)) return SJKVARN_ERR_ARG;
        type = in[i].type;
        if (out[i].p && (out[i].n_head != in[i].n_head || !type_ok(out[i].type))) return SJKVARN_ERR_ARG;
        // rows in place: an element has to stay where it was read
        if (out[i].p == in[i].p && (out[i].type != type || out[i].row_stride != in[i].row_stride || out[i].head_stride != in[i].head_stride))
            return SJKVARN_ERR_ARG;
        if (out[i].p || (cached && i > 0)) n[i] = in[i].n_head;       // heads that nobody wants are not read
        p.in[i] = in[i];
        p.out[i] = out[i];
    }
    if (type < 0) return SJKVARN_ERR_ARG;
    if ((a->q_norm || a->k_norm) && (!type_ok(a->norm_type) || !(a->eps >= 0.0f) || !isfinite(a->eps))) return SJKVARN_ERR_ARG;
    const bool rope = a->rope.n_rot != 0;
    if (rope && (a->rope.n_rot < 2 || (a->rope.n_rot & 1) || a->rope.n_rot > a->head_dim || !a->rope.step ||
                 (a->rope.layout != SJK_ROPE_HALF && a->rope.layout != SJK_ROPE_PAIR)))
        return SJKVARN_ERR_ROTATION;
    if ((rope || cached) && !a->pos) return SJKVARN_ERR_ARG;
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
    bool vec = p.D % 16 == 0 && p.n_rot % 16 == 0;
    for (int i = 0; i < 3; ++i) vec = vec && rows_vec(p.in[i]) && rows_vec(p.out[i]);
    if (cached) {
        const int64_t s = p.c.page_stride | p.c.slot_stride | p.c.head_stride;
        vec = vec && aligned(p.c.k, 16) && aligned(p.c.v, 16) && (s & 7) == 0;
    }
    if (!vec) {
        const int64_t warps = (int64_t) p.n_tok * p.n_all, ctas = (warps + NT / 32 - 1) / (NT / 32);
        return launch(qkv_scalar_kernel, dim3((unsigned) (ctas < 148 * 8 ? ctas : 148 * 8)), dim3(NT), (size_t) (NT / 32) * p.D * sizeof(float), st, p);
    }
    int L = 1;
    while (16 * L < p.D) L <<= 1;
    // Few tokens: one token per CTA and the heads over grid.y. Many: all heads in one CTA and several tokens (a block
    // of 32 / L at least), so that the table and the norm weights serve several rows.
    int T = 1, ny = (p.n_all + NT / 32 - 1) / (NT / 32);
    if (p.n_tok >= 148 * 8) {
        ny = 1;
        T = 32 / L > 8 ? 32 / L : 8;
        while (T > 32 / L && p.n_tok / T < 148 * 4) T /= 2;
    }
    p.T = T;
    const dim3 grid((unsigned) ((p.n_tok + T - 1) / T), (unsigned) ny);
    const size_t smem = ((size_t) T * p.n_rot + 2 * (size_t) p.D) * sizeof(float);
    switch (type) {
        case SJK_F32: return launch_vec<SJK_F32>(L, grid, smem, st, p);
        case SJK_F16: return launch_vec<SJK_F16>(L, grid, smem, st, p);
        default: return launch_vec<SJK_BF16>(L, grid, smem, st, p);
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
