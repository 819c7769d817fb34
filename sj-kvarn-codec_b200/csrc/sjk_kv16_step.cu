// sjk_kv16_step.cu - what a step that brings several tokens of every sequence needs beside its attention: the maps from
// the sequences' lengths to tokens (sjk_kv16_maps), and the move of accepted drafts to their places (sjk_kv16_keep).
//
// Bound: a launch's latency, and for large calls the bytes: 20 written per token, a row once in and once out. Measured (us a
// pass from Python, on the GPU by CUDA graphs): maps of one chat's 8 drafts 5.4 and 2.3, of 512 requests with 15,500 tokens 5.0 and
// 3.1; paths of up to 5 tokens in 16 layers 6.8 and 2.9; 64 paths of up to 9 in 32 layers of 4 x 256 f16 channels 16.1 and 16.1
// (75 MB: 4.7 TB/s; 20 with 256 threads a CTA, of which half had no word).
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

namespace {

using namespace sjk16;

constexpr int NT = 256;                     // maps
// keep: a thread a 16-byte word of a row, and more of wider rows in turn. 1,024 channels are 128 words (20 us with 256 threads, 16.1 with 128);
// of narrower rows' CTAs some threads have none, which such calls, of a few us, do not show
constexpr int NK = 128;
__device__ unsigned int g_step_status;

SJK_DEV void flag() { atomicOr(&g_step_status, (unsigned) SJK_DEVICE_PAGE); }

// page of a table entry, or NO_BLOCK; ids that are no page are reported
SJK_DEV uint32_t page_of(const sjk_kv16 & c, int64_t row, uint32_t g) {
    if (row < 0 || row >= (int64_t) c.n_rows || g >= c.table_stride) { flag(); return SJKVARN_NO_BLOCK; }
    const uint32_t page = c.tables[row * c.table_stride + g];
    if (page < c.n_pages) return page;
    if (page != SJKVARN_NO_BLOCK) flag();
    return SJKVARN_NO_BLOCK;
}

// ---- maps -----------------------------------------------------------------------------------------------------
struct MapParams {
    sjk_kv16 c;
    const int32_t * len, * add, * rows;
    const uint64_t * masks;
    int n_seq, n_tok;
    sjk_kv16_step out;
};

// Every CTA sums all sequences' counts (a few KB that lie in L2 after the first one), then takes its tokens: a look-up in
// the sums, a table entry, five stores.
__global__ void __launch_bounds__(NT) maps_kernel(const __grid_constant__ MapParams p) {
    extern __shared__ int32_t s_first[];    // [n_seq + 1]
    __shared__ int64_t s_warp[NT / 32];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t base = 0;
    for (int i0 = 0; i0 < p.n_seq; i0 += NT) {
        const int i = i0 + tid;
        int64_t x = 0;
        if (i < p.n_seq) {
            const int32_t a = p.add[i];
            if (a < 0) { if (blockIdx.x == 0) flag(); }
            else x = a;
        }
        const int64_t own = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_warp[warp] = x;
        __syncthreads();
        int64_t before = base, all = 0;
        for (int w = 0; w < NT / 32; ++w) {
            if (w < warp) before += s_warp[w];
            all += s_warp[w];
        }
        const int64_t at = before + x - own;
        if (i < p.n_seq) s_first[i] = (int32_t) (at < p.n_tok ? at : p.n_tok);
        base += all;
        __syncthreads();
    }
    if (tid == 0) {
        s_first[p.n_seq] = (int32_t) (base < p.n_tok ? base : p.n_tok);
        if (base > p.n_tok && blockIdx.x == 0) flag();
    }
    __syncthreads();
    if (blockIdx.x == 0 && p.out.first)
        for (int i = tid; i <= p.n_seq; i += NT) p.out.first[i] = s_first[i];
    const int total = s_first[p.n_seq];
    for (int64_t t = (int64_t) blockIdx.x * NT + tid; t < p.n_tok; t += (int64_t) gridDim.x * NT) {
        int32_t row = 0, pos = -1, at = -1;
        int64_t slot = -1;
        if (t < total) {
            int lo = 0, hi = p.n_seq - 1;                   // the last sequence that begins at or before the token
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_first[mid] <= (int32_t) t) lo = mid; else hi = mid - 1;
            }
            const int j = (int) t - s_first[lo], count = s_first[lo + 1] - s_first[lo];
            const int32_t len = p.len[lo];
            row = p.rows ? p.rows[lo] : lo;
            const int64_t place = (int64_t) len + j;
            if (len < 0 || place > 0x7FFFFFFE) flag();
            else {
                at = pos = (int32_t) place;
                if (p.masks) {
                    uint64_t m = p.masks[t];
                    if (count < 64) m &= (1ull << count) - 1ull;
                    if (j < 64) m &= ~(1ull << j);
                    const int64_t deep = (int64_t) len + __popcll(m);
                    pos = (int32_t) (deep < 0x7FFFFFFF ? deep : 0x7FFFFFFE);
                }
                const uint32_t g = (uint32_t) at / (uint32_t) p.c.page_tokens, page = page_of(p.c, row, g);
                if (page != SJKVARN_NO_BLOCK) slot = (int64_t) page * p.c.page_tokens + ((uint32_t) at - g * (uint32_t) p.c.page_tokens);
            }
        }
        if (p.out.row) p.out.row[t] = row;
        if (p.out.pos) p.out.pos[t] = pos;
        if (p.out.at) p.out.at[t] = at;
        if (p.out.slot) p.out.slot[t] = slot;
    }
}

// ---- keep -----------------------------------------------------------------------------------------------------
struct KeepParams {
    sjk_kv16 c;
    int64_t layer_stride;
    const int32_t * len, * path, * count, * rows;
    int n_seq, width;
    int32_t * new_len;
};

// grid: sequences, layers, K and V. The path ascends, so that row j comes from a place behind all rows written before it:
// a thread has the same channels of every row and goes through them in order, BATCH reads ahead of the writes (a read of
// rows j .. j + BATCH - 1 is of places j and on, which only writes of the same batch and later ones touch). E: a 16-byte word
// or an element. The path's checks and page look-ups are one per thread, before the rows move.
template <typename E>
__global__ void __launch_bounds__(NK) keep_kernel(const __grid_constant__ KeepParams p) {
    constexpr int BATCH = 8;
    __shared__ int64_t s_from[SJK_KEEP_MAX], s_to[SJK_KEEP_MAX];
    pdl_wait();
    pdl_release();
    const int i = blockIdx.x, tid = threadIdx.x, P = p.c.page_tokens;
    const int32_t len = p.len[i], count = p.count[i];
    const int64_t row = p.rows ? (int64_t) p.rows[i] : (int64_t) i;
    int bad = len < 0 || count < 0 || count > p.width || row < 0 || row >= (int64_t) p.c.n_rows ? 1 : 0;
    if (p.rows)
        for (int j = tid; j < i && !bad; j += NK) bad = p.rows[j] == (int32_t) row;        // an earlier entry has the row
    for (int j = tid; j < count && !bad; j += NK) {
        const int32_t * path = p.path + (int64_t) i * p.width;
        const int32_t from = path[j];
        const int64_t a = (int64_t) len + from, b = (int64_t) len + j;
        bad = from < j || (j > 0 && path[j - 1] >= from) || a >= (int64_t) p.c.table_stride * P || a > 0x7FFFFFFE;   // (lengths are 32 bits)
        if (bad) break;
        const uint32_t ga = (uint32_t) (a / P), gb = (uint32_t) (b / P), pa = page_of(p.c, row, ga), pb = page_of(p.c, row, gb);
        bad = pa == SJKVARN_NO_BLOCK || pb == SJKVARN_NO_BLOCK;
        s_from[j] = (int64_t) pa * p.c.page_stride + (a - (int64_t) ga * P) * p.c.slot_stride;
        s_to[j] = (int64_t) pb * p.c.page_stride + (b - (int64_t) gb * P) * p.c.slot_stride;
    }
    bad = __syncthreads_or(bad);
    const bool first = blockIdx.y == 0 && blockIdx.z == 0 && tid == 0;
    if (bad) {                              // nothing of the sequence moves
        if (first) {
            flag();
            if (p.new_len) p.new_len[i] = len;
        }
        return;
    }
    if (first && p.new_len) p.new_len[i] = len + count;
    constexpr int EL = sizeof(E) / 2;
    uint16_t * base = static_cast<uint16_t *>(blockIdx.z ? p.c.v : p.c.k) + (int64_t) blockIdx.y * p.layer_stride;
    const int per = p.c.head_dim / EL, words = p.c.n_head_kv * per;
    int skip = 0;                           // rows that are in their places
    while (skip < count && s_from[skip] == s_to[skip]) ++skip;
    for (int w = tid; w < words; w += NK) {
        const int h = w / per;
        uint16_t * mine = base + (int64_t) h * p.c.head_stride + (w - h * per) * EL;
        for (int j0 = skip; j0 < count; j0 += BATCH) {
            E x[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (j0 + j < count) x[j] = *reinterpret_cast<const E *>(mine + s_from[j0 + j]);
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
                if (j0 + j < count) *reinterpret_cast<E *>(mine + s_to[j0 + j]) = x[j];
        }
    }
}

}  // namespace

extern "C" int sjk_kv16_maps(const sjk_kv16 * c, const int32_t * len, const int32_t * add, const int32_t * rows, const uint64_t * masks,
                             int n_seq, int n_tok, const sjk_kv16_step * out, sjk_stream st) {
    if (!c || !out || sjk_kv16_check(c) || n_seq < 0 || n_seq > SJK_MAPS_MAX || n_tok < 0) return SJKVARN_ERR_ARG;
    if ((n_seq && (!len || !add)) || !list_ok(len) || !list_ok(add) || !list_ok(rows) || !aligned(masks, 8) || !list_ok(out->first) ||
        !list_ok(out->row) || !list_ok(out->pos) || !list_ok(out->at) || !aligned(out->slot, 8))
        return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    // every CTA reads all counts, and its tokens' lengths, rows and masks, while others write
    const size_t seqs = (size_t) n_seq * sizeof(int32_t), toks = (size_t) n_tok * sizeof(int32_t);
    const struct { const void * p; size_t n; } in[4] = {{len, seqs}, {add, seqs}, {rows, seqs}, {masks, 2 * toks}},
        to[5] = {{out->first, seqs + sizeof(int32_t)}, {out->row, toks}, {out->pos, toks}, {out->at, toks}, {out->slot, 2 * toks}};
    for (const auto & x : in)
        for (const auto & y : to)
            if (!apart(x.p, x.n, y.p, y.n)) return SJKVARN_ERR_ARG;
    MapParams p = {*c, len, add, rows, masks, n_seq, n_tok, *out};
    const int64_t ctas = ((int64_t) n_tok + NT - 1) / NT;
    return launch(maps_kernel, dim3((unsigned) (ctas < 1 ? 1 : ctas < 148 * 4 ? ctas : 148 * 4)), dim3(NT), (size_t) (n_seq + 1) * sizeof(int32_t), st, p);
}

extern "C" int sjk_kv16_keep(const sjk_kv16 * c, int n_layers, int64_t layer_stride, const int32_t * len, const int32_t * path,
                             const int32_t * count, const int32_t * rows, int width, int n_seq, int32_t * new_len, sjk_stream st) {
    if (!c || sjk_kv16_check(c) || n_layers < 1 || n_layers > 65535 || layer_stride < 0 || width < 1 || width > SJK_KEEP_MAX || n_seq < 0) return SJKVARN_ERR_ARG;
    if ((n_seq && (!len || !path || !count)) || !list_ok(len) || !list_ok(path) || !list_ok(count) || !list_ok(rows) || !list_ok(new_len)) return SJKVARN_ERR_ARG;
    if (!rows && (int64_t) n_seq > (int64_t) c->n_rows) return SJKVARN_ERR_ARG;
    // every CTA of a sequence reads its length, path, count and row (and the rows before it), one writes the new length
    const size_t list = (size_t) n_seq * sizeof(int32_t);
    if (!apart(new_len, list, len, list) || !apart(new_len, list, path, list * width) || !apart(new_len, list, count, list) || !apart(new_len, list, rows, list))
        return SJKVARN_ERR_ARG;
    if (n_seq == 0) return 0;
    const KeepParams p = {*c, layer_stride, len, path, count, rows, n_seq, width, new_len};
    const int64_t strides = c->page_stride | c->slot_stride | c->head_stride | (n_layers > 1 ? layer_stride : 0);
    const bool wide = aligned(c->k, 16) && aligned(c->v, 16) && (strides & 7) == 0 && c->head_dim % 8 == 0;
    const dim3 grid((unsigned) n_seq, (unsigned) n_layers, 2);
    return wide ? launch(keep_kernel<uint4>, grid, dim3(NK), 0, st, p) : launch(keep_kernel<uint16_t>, grid, dim3(NK), 0, st, p);
}

int sjk_step_status_take(void) {
    unsigned v = 0;
    if (sjk_check(cudaMemcpyFromSymbol(&v, g_step_status, sizeof v))) return -1;
    if (v) {
        const unsigned z = 0;
        if (sjk_check(cudaMemcpyToSymbol(g_step_status, &z, sizeof z))) return -1;
    }
    return (int) v;
}
