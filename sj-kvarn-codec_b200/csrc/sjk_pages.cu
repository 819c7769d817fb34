// sjk_pages.cu - who owns the pages of a cache: forks that share pages, copy on write, freeing, compaction, and the
// copies of page contents these need. Integer bookkeeping with a fixed result: where requests meet on one page, counts
// go by atomics (their order does not matter) and every choice - who keeps a page, which id a request takes, in which
// order ids return to the stack - by request and page numbers.
//
// Bound: the contents' copies by HBM (every moved page once in and once out), the bookkeeping by latency: one CTA per
// call, phases in a row, each a few dependent loads. Measured: a beam step of 8 (fork, free, extend with 4 split pages of
// 16 layers) 14.1 us in four launches; 63 copies of an 8.4 MB block, read from L2 after the first, 93 us (5.7 TB/s
// written); 230 MB of pages moved by a compaction about 75 us (6.1 TB/s read and written).
#include "sjk_kv16.cuh"
#include "sjk_internal.h"

namespace {

using namespace sjk16;

constexpr int NT = 256;                     // fork, free, copy
constexpr int NB = 1024;                    // one-CTA bookkeeping
constexpr uint32_t NO_BLOCK = SJKVARN_NO_BLOCK;
__device__ unsigned int g_pages_status;

SJK_DEV void flag() { atomicOr(&g_pages_status, (unsigned) SJK_DEVICE_PAGE); }

// The ledger: the device pool's header and stack (sjk_pool_dev_bytes), then per-page words. Ticket, claims, count, last
// and marks are zero between calls.
struct Ledger {
    uint32_t * head;                        // n_free, n_pages, ticket of sjk_pages_free, copies of the last call
    uint32_t * ids, * shares, * count, * last, * old, * src, * dst, * map, * marks, * claims;
};
SJK_HD Ledger ledger_of(void * base, uint32_t n) {
    Ledger l;
    uint32_t * w = static_cast<uint32_t *>(base);
    l.head = w;      w += 4;
    l.ids = w;       w += n;
    l.shares = w;    w += n;
    l.count = w;     w += n;
    l.last = w;      w += n;
    l.old = w;       w += n;
    l.src = w;       w += n;
    l.dst = w;       w += n;
    l.map = w;       w += n;
    l.marks = w;     w += (n + 31u) / 32u;
    l.claims = w;
    return l;
}

struct Params {
    Ledger l;
    uint32_t * tables;
    uint32_t n_pages, n_rows, stride;
    int page_tokens, n_slabs;
    sjk_slab slabs[SJK_MAX_SLABS];
    const int32_t * a, * b, * c;            // the call's lists
    int n, add_all;
    int32_t * status;
};

// exclusive prefix sum over a CTA of NTHR threads; *total gets the sum. s: NTHR / 32 words
template <int NTHR>
SJK_DEV uint32_t cta_scan(uint32_t v, uint32_t * s, uint32_t * total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = lane < NTHR / 32 ? s[lane] : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, w, o);
            if (lane >= o) w += y;
        }
        if (lane < NTHR / 32) s[lane] = w;
    }
    __syncthreads();
    const uint32_t before = (warp ? s[warp - 1] : 0u) + x - v;
    *total = s[NTHR / 32 - 1];
    __syncthreads();
    return before;
}

// ---- fork: one CTA per request -------------------------------------------------------------------------------
__global__ void __launch_bounds__(NT) pages_fork_kernel(const __grid_constant__ Params p) {
    pdl_wait();
    pdl_release();
    const int i = blockIdx.x;
    const int32_t src = p.a[i], dst = p.b[i];
    int bad = src < 0 || dst < 0 || (uint32_t) src >= p.n_rows || (uint32_t) dst >= p.n_rows ? 1 : 0;
    for (int j = threadIdx.x; j < p.n && !bad; j += NT)
        if (p.a[j] == dst || (j < i && p.b[j] == dst)) bad = 1;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) p.status[i] = SJKVARN_ERR_ARG;
        return;
    }
    const uint32_t * from = p.tables + (size_t) src * p.stride;
    uint32_t * to = p.tables + (size_t) dst * p.stride;
    int full = 0, wrong = 0;
    for (uint32_t g = threadIdx.x; g < p.stride; g += NT) {
        full |= to[g] != NO_BLOCK ? 1 : 0;
        wrong |= from[g] != NO_BLOCK && from[g] >= p.n_pages ? 1 : 0;
    }
    full = __syncthreads_or(full);
    wrong = __syncthreads_or(wrong);
    if (full || wrong) {
        if (threadIdx.x == 0) p.status[i] = full ? SJKVARN_ERR_ARG : SJKVARN_ERR_CORRUPT;
        return;
    }
    for (uint32_t g = threadIdx.x; g < p.stride; g += NT) {
        const uint32_t e = from[g];
        if (e == NO_BLOCK) continue;
        to[g] = e;
        atomicAdd(&p.l.shares[e], 1u);
    }
    if (threadIdx.x == 0) p.status[i] = 0;
}

// ---- free: grid.x requests, grid.y runs of a row; the last CTA pushes what lost its last owner ------------------
__global__ void __launch_bounds__(NT) pages_free_kernel(const __grid_constant__ Params p) {
    __shared__ uint32_t s_scan[NT / 32];
    __shared__ int s_last;
    pdl_wait();
    pdl_release();
    const int i = blockIdx.x;
    const int32_t row = p.a[i];
    if (row < 0 || (uint32_t) row >= p.n_rows) {
        if (threadIdx.x == 0) flag();
    } else {
        const int64_t g0 = p.b && p.b[i] > 0 ? p.b[i] : 0;
        const int64_t g1 = p.c && (uint32_t) p.c[i] < p.stride ? p.c[i] : p.c && p.c[i] < 0 ? 0 : (int64_t) p.stride;
        for (int64_t g = g0 + (int64_t) blockIdx.y * NT + threadIdx.x; g < g1; g += (int64_t) gridDim.y * NT) {
            uint32_t * at = p.tables + (size_t) row * p.stride + g;
            if (*at == NO_BLOCK) continue;
            const uint32_t e = atomicExch(at, NO_BLOCK);    // a row that is named twice gives each entry up once
            if (e == NO_BLOCK) continue;
            if (e >= p.n_pages) { flag(); continue; }
            if (atomicSub(&p.l.shares[e], 1u) == 0u) atomicOr(&p.l.marks[e >> 5], 1u << (e & 31u));
        }
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicAdd(&p.l.head[2], 1u) == gridDim.x * gridDim.y - 1u;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    // marked pages in descending order, from the last word of the bitmap to the first
    const uint32_t words = (p.n_pages + 31u) / 32u;
    uint32_t n_free = p.l.head[0];
    bool torn = n_free > p.n_pages;                         // a stack that is no stack of this pool
    if (torn) n_free = p.n_pages;
    for (uint32_t w0 = 0; w0 < words; w0 += NT) {
        const uint32_t k = w0 + threadIdx.x;
        const bool on = k < words;
        const uint32_t w = on ? words - 1u - k : 0u;
        uint32_t m = on ? __ldcg(&p.l.marks[w]) : 0u;
        if (m) p.l.marks[w] = 0u;
        uint32_t total;
        uint32_t at = n_free + cta_scan<NT>((uint32_t) __popc(m), s_scan, &total);
        while (m) {
            const uint32_t bit = 31u - (uint32_t) __clz(m), id = w * 32u + bit;
            m &= ~(1u << bit);
            if (at < p.n_pages) p.l.ids[at] = id;
            ++at;
            p.l.shares[id] = 0u;
        }
        n_free += total;
        if (n_free > p.n_pages) {                           // more free ids than pages: some were free before
            torn = true;
            n_free = p.n_pages;
        }
    }
    if (torn && threadIdx.x == 0) flag();
    if (threadIdx.x == 0) { p.l.head[0] = n_free; p.l.head[2] = 0u; }
}

// ---- extend: one CTA; an item is an entry (request, page) -----------------------------------------------------------
// NTHR threads, at least a thread per request. Up to NTHR items (a decode step) stay in registers from phase to phase;
// more go round by NTHR.
template <int NTHR>
__global__ void __launch_bounds__(NTHR) pages_extend_kernel(const __grid_constant__ Params p) {
    __shared__ uint32_t s_scan[NTHR / 32];
    __shared__ int32_t s_row[NTHR], s_len[NTHR];
    __shared__ uint32_t s_g0[NTHR], s_off[NTHR];
    pdl_wait();
    pdl_release();
    const int tid = threadIdx.x;
    const uint32_t P = (uint32_t) p.page_tokens, n_free = p.l.head[0];
    // the requests: rows, first pages, and where their items begin
    int bad = 0, much = 0;                                  // much: more entries than there are pages
    uint32_t items = 0;
    if (tid < p.n) {
        const int32_t row = p.a[tid], len = p.b[tid], add = p.c ? p.c[tid] : p.add_all;
        s_row[tid] = row;
        s_len[tid] = len;
        if (row < 0 || (uint32_t) row >= p.n_rows || len < 0 || add < 0 || (add > 0 && ((uint32_t) len + (uint32_t) add - 1u) / P >= p.stride)) bad = 1;
        else if (add > 0) {
            s_g0[tid] = (uint32_t) len / P;
            items = ((uint32_t) len + (uint32_t) add - 1u) / P - s_g0[tid] + 1u;
            much = items > p.n_pages;
        }
    }
    uint32_t n_items;
    const uint32_t off = cta_scan<NTHR>(much || bad ? 0u : items, s_scan, &n_items);
    s_off[tid] = off;
    if (tid < p.n)
        for (int j = 0; j < tid; ++j) bad |= s_row[j] == s_row[tid] ? 1 : 0;
    bad = __syncthreads_or(bad);
    much = __syncthreads_or(much);
    const bool torn = n_free > p.n_pages;                   // a stack that is no stack of this pool
    if (bad || torn || much) {
        if (tid == 0) { p.status[0] = bad ? SJKVARN_ERR_ARG : torn ? SJKVARN_ERR_CORRUPT : SJKVARN_ERR_POOL_FULL; p.l.head[3] = 0u; }
        return;
    }
    const uint32_t top_id = (uint32_t) tid < n_free ? p.l.ids[n_free - 1u - tid] : 0u;
    // an item: its request (the last whose items begin at or before it), table entry, page and how many share that
    struct Item { int r; uint32_t * at; uint32_t e, shares; };
    auto item_of = [&](uint32_t it) {
        Item x = {0, nullptr, NO_BLOCK, 0u};
        if (it >= n_items) return x;
        int lo = 0, hi = p.n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_off[mid] <= it) lo = mid; else hi = mid - 1;
        }
        x.r = lo;
        x.at = p.tables + (size_t) s_row[lo] * p.stride + s_g0[lo] + (it - s_off[lo]);
        x.e = *x.at;
        if (x.e < p.n_pages) x.shares = p.l.shares[x.e];
        return x;
    };
    // a hole, or a shared page that is not kept: the last of a page's owners keeps it when all are in the call
    auto takes = [&](const Item & x) {
        if (!x.at) return false;
        if (x.e == NO_BLOCK) return true;
        return x.shares && !(__ldcg(&p.l.count[x.e]) == x.shares + 1u && __ldcg(&p.l.last[x.e]) == (uint32_t) x.r);
    };
    const bool one = n_items <= (uint32_t) NTHR;
    const Item mine = item_of(tid);
    // who holds the shared pages: how many of the call, and the last of them
    int wrong = 0;
    for (uint32_t it = tid; it < n_items; it += NTHR) {
        const Item x = one ? mine : item_of(it);
        if (x.e != NO_BLOCK && x.e >= p.n_pages) wrong = 1;
        else if (x.shares) { atomicAdd(&p.l.count[x.e], 1u); atomicMax(&p.l.last[x.e], (uint32_t) x.r); }
    }
    wrong = __syncthreads_or(wrong);
    uint32_t need = 0;
    for (uint32_t it = tid; it < n_items; it += NTHR) need += takes(one ? mine : item_of(it)) ? 1u : 0u;
    uint32_t total;
    const uint32_t before_mine = cta_scan<NTHR>(need, s_scan, &total);
    // the ids that will be handed out are pages (this thread's first was asked for above)
    if (!wrong && total <= n_free) {
        int off_pool = (uint32_t) tid < total && top_id >= p.n_pages ? 1 : 0;
        for (uint32_t k = (uint32_t) tid + NTHR; k < total; k += NTHR) off_pool |= p.l.ids[n_free - 1u - k] >= p.n_pages ? 1 : 0;
        wrong = __syncthreads_or(off_pool);
    }
    if (wrong || total > n_free) {                          // nothing is done: only the counts go back
        for (uint32_t it = tid; it < n_items; it += NTHR) {
            const uint32_t e = (one ? mine : item_of(it)).e;
            if (e < p.n_pages) { p.l.count[e] = 0u; p.l.last[e] = 0u; }
        }
        if (tid == 0) { p.status[0] = wrong ? SJKVARN_ERR_CORRUPT : SJKVARN_ERR_POOL_FULL; p.l.head[3] = 0u; }
        return;
    }
    uint32_t taken = 0, copies = 0;
    for (uint32_t it0 = 0; it0 < n_items; it0 += NTHR) {
        const uint32_t it = it0 + tid;
        const Item x = one ? mine : item_of(it);
        const bool take = one ? need != 0u : takes(x);
        const bool keep = take && x.e != NO_BLOCK && (uint64_t) (s_g0[x.r] + (it - s_off[x.r])) * P < (uint64_t) (uint32_t) s_len[x.r];
        uint32_t takes_all = total, keeps_all, before = before_mine;
        if (!one) before = cta_scan<NTHR>(take ? 1u : 0u, s_scan, &takes_all);
        const uint32_t q = cta_scan<NTHR>(keep ? 1u : 0u, s_scan, &keeps_all);
        if (take) {
            const uint32_t k = taken + before, id = p.l.ids[n_free - 1u - k];
            *x.at = id;
            p.l.old[k] = x.e;
            if (keep) {
                p.l.src[copies + q] = x.e;
                p.l.dst[copies + q] = id;
            }
        }
        taken += takes_all;
        copies += keeps_all;
    }
    __syncthreads();
    for (uint32_t k = tid; k < total; k += NTHR) {
        const uint32_t e = p.l.old[k];
        if (e == NO_BLOCK) continue;
        atomicSub(&p.l.shares[e], 1u);
        p.l.count[e] = 0u;
        p.l.last[e] = 0u;
    }
    if (tid == 0) {
        p.l.head[0] = n_free - total;
        p.l.head[3] = copies;
        p.status[0] = 0;
    }
}

// ---- compact: the moves (one CTA, a bitmap of the used pages in shared memory), then tables and contents ---------------
__global__ void __launch_bounds__(NB) pages_plan_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint32_t s_used[];
    __shared__ uint32_t s_scan[NB / 32];
    pdl_wait();
    pdl_release();
    const uint32_t tid = threadIdx.x, n = p.n_pages, words = (n + 31u) / 32u;
    const bool torn = p.l.head[0] > n;                      // a stack that is no stack of this pool: nothing moves
    const uint32_t n_free = torn ? n : p.l.head[0], top = n - n_free;
    for (uint32_t w = tid; w < words; w += NB) s_used[w] = w * 32u + 32u <= n ? 0xFFFFFFFFu : (1u << (n & 31u)) - 1u;
    __syncthreads();
    for (uint32_t i = tid; i < n_free; i += NB) {
        const uint32_t id = p.l.ids[i];
        if (id < n) atomicAnd(&s_used[id >> 5], ~(1u << (id & 31u)));
        else flag();
    }
    __syncthreads();
    uint32_t holes = 0, movers = 0;
    for (uint32_t w0 = 0; w0 < words; w0 += NB) {
        const uint32_t w = w0 + tid;
        uint32_t h = 0, m = 0;
        if (w < words) {
            const uint32_t below = top <= w * 32u ? 0u : top - w * 32u >= 32u ? 0xFFFFFFFFu : (1u << (top - w * 32u)) - 1u;
            h = ~s_used[w] & below;
            m = s_used[w] & ~below;
        }
        uint32_t nh, nm;
        uint32_t ah = holes + cta_scan<NB>((uint32_t) __popc(h), s_scan, &nh);
        uint32_t am = movers + cta_scan<NB>((uint32_t) __popc(m), s_scan, &nm);
        for (; h; h &= h - 1u) p.l.dst[ah++] = w * 32u + (uint32_t) __ffs(h) - 1u;
        for (; m; m &= m - 1u) p.l.src[am++] = w * 32u + (uint32_t) __ffs(m) - 1u;
        holes += nh;
        movers += nm;
    }
    __syncthreads();
    // equal where the stack holds every free id once; a damaged one moves nothing
    const bool sound = holes == movers && !torn;
    const uint32_t moves = sound ? movers : 0u;
    if (!sound && tid == 0) flag();
    for (uint32_t k = tid; k < moves; k += NB) {
        const uint32_t s = p.l.src[k], d = p.l.dst[k];
        p.l.map[s] = k;
        p.l.shares[d] = p.l.shares[s];
        p.l.shares[s] = 0u;
    }
    if (sound)
        for (uint32_t i = tid; i < n_free; i += NB) p.l.ids[i] = n - 1u - i;
    if (tid == 0) {
        p.l.head[3] = moves;
        if (p.status) { p.status[0] = (int32_t) top; p.status[1] = (int32_t) moves; }
    }
}

// Contents of the listed pages in every layer of every slab, in segments of SEG bytes, which the CTAs of a grid that
// fills the GPU claim one by one (SMs are not equally fast: with equal shares the slow ones would end last); remap: the
// tables' entries of moved pages as well. n_fixed < 0: as many as the ledger says.
constexpr uint32_t SEG = 16384;
__global__ void __launch_bounds__(NT) pages_copy_kernel(const __grid_constant__ Params p, const uint32_t * src, const uint32_t * dst, int n_fixed,
                                                        int remap) {
    __shared__ uint32_t s_next[2];
    pdl_wait();
    pdl_release();
    const uint32_t n = n_fixed >= 0 ? (uint32_t) n_fixed : p.l.head[3];
    if (n == 0) return;
    if (remap) {
        const uint32_t top = p.n_pages - p.l.head[0];
        const uint64_t all = (uint64_t) p.n_rows * p.stride;
        for (uint64_t i = (uint64_t) blockIdx.x * NT + threadIdx.x; i < all; i += (uint64_t) gridDim.x * NT) {
            const uint32_t e = p.tables[i];
            if (e < top || e == NO_BLOCK) continue;
            const uint32_t k = e < p.n_pages ? p.l.map[e] : n;
            if (k < n && src[k] == e) p.tables[i] = dst[k];
            else flag();                                    // an entry whose page is not in use
        }
    }
    if (p.n_slabs == 0) return;
    uint64_t u = blockIdx.x;
    for (uint32_t i = 0;; i ^= 1u) {
        uint64_t at = u;
        int s = 0;
        uint32_t segs = 1, layers = 1;
        for (; s < p.n_slabs; ++s) {
            segs = (uint32_t) ((p.slabs[s].page_bytes + SEG - 1) / SEG);
            layers = (uint32_t) p.slabs[s].n_layers;
            const uint64_t units = (uint64_t) n * layers * segs;
            if (at < units) break;
            at -= units;
        }
        if (s == p.n_slabs) break;
        uint32_t claim = 0;
        if (threadIdx.x == 0) claim = atomicAdd(p.l.claims, 1u);            // the next one, while this one is copied
        const sjk_slab & sl = p.slabs[s];
        const uint32_t seg = (uint32_t) (at % segs);
        const uint64_t q = at / segs;
        const uint32_t k = (uint32_t) (q / layers), layer = (uint32_t) (q - (uint64_t) k * layers);
        const uint32_t a = src[k], b = dst[k];
        if (a < p.n_pages && b < p.n_pages) {
            uint8_t * base = static_cast<uint8_t *>(sl.base) + (size_t) layer * sl.layer_stride + (size_t) seg * SEG;
            const uint4 * from = reinterpret_cast<const uint4 *>(base + (size_t) a * sl.page_bytes);
            uint4 * to = reinterpret_cast<uint4 *>(base + (size_t) b * sl.page_bytes);
            const size_t left = sl.page_bytes - (size_t) seg * SEG;
            const uint32_t words = (uint32_t) ((left < SEG ? left : SEG) / 16);
            uint4 x[SEG / 16 / NT];
#pragma unroll
            for (int j = 0; j < (int) (SEG / 16 / NT); ++j)
                if (j * NT + threadIdx.x < words) x[j] = from[j * NT + threadIdx.x];
#pragma unroll
            for (int j = 0; j < (int) (SEG / 16 / NT); ++j)
                if (j * NT + threadIdx.x < words) to[j * NT + threadIdx.x] = x[j];
        } else if (threadIdx.x == 0) flag();
        if (threadIdx.x == 0) s_next[i] = claim;
        __syncthreads();
        u = (uint64_t) gridDim.x + s_next[i];
    }
    // the last CTA leaves the counters as they were
    if (threadIdx.x == 0 && atomicAdd(&p.l.head[2], 1u) == gridDim.x - 1u) {
        p.l.claims[0] = 0u;
        p.l.head[2] = 0u;
    }
}

int params_of(const sjk_pages * g, Params * p, bool tables) {
    if (!g || !g->ledger || !aligned(g->ledger, 16) || g->n_pages < 1 || g->n_pages > SJK_PAGES_MAX) return SJKVARN_ERR_ARG;
    if (tables && (!g->tables || !aligned(g->tables, 4) || g->n_rows < 1 || g->n_rows > 0x7FFFFFFFu || g->table_stride < 1 || g->page_tokens < 1)) return SJKVARN_ERR_ARG;
    if (g->n_slabs < 0 || g->n_slabs > SJK_MAX_SLABS) return SJKVARN_ERR_ARG;
    for (int i = 0; i < g->n_slabs; ++i) {
        const sjk_slab & s = g->slabs[i];
        if (!s.base || !aligned(s.base, 16) || s.page_bytes < 16 || s.page_bytes % 16 || s.layer_stride % 16 || s.n_layers < 1) return SJKVARN_ERR_ARG;
    }
    *p = Params();
    p->l = ledger_of(g->ledger, g->n_pages);
    p->tables = g->tables;
    p->n_pages = g->n_pages; p->n_rows = g->n_rows; p->stride = g->table_stride;
    p->page_tokens = g->page_tokens; p->n_slabs = g->n_slabs;
    for (int i = 0; i < g->n_slabs; ++i) p->slabs[i] = g->slabs[i];
    return 0;
}

__global__ void __launch_bounds__(NT) pages_init_kernel(Ledger l, uint32_t n) {
    pdl_wait();
    pdl_release();
    for (uint32_t i = blockIdx.x * NT + threadIdx.x; i < n; i += gridDim.x * NT) {
        l.ids[i] = n - 1u - i;
        l.shares[i] = l.count[i] = l.last[i] = 0u;
        if (i < (n + 31u) / 32u) l.marks[i] = 0u;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) { l.head[0] = l.head[1] = n; l.head[2] = l.head[3] = l.claims[0] = 0u; }
}

// Whether n copies are more segments than the 32-bit claims can count, with those that the CTAs claim in vain.
bool too_many(const Params & p, uint32_t n) {
    double units = 0.0;
    for (int i = 0; i < p.n_slabs; ++i) units += (double) ((p.slabs[i].page_bytes + SEG - 1) / SEG) * p.slabs[i].n_layers * n;
    return units > 4e9;
}

int copy_launch(const Params & p, const uint32_t * src, const uint32_t * dst, int n, int remap, sjk_stream st) {
    if (p.n_slabs == 0 && !remap) return 0;
    return launch(pages_copy_kernel, dim3(148 * 6), dim3(NT), 0, st, p, src, dst, n, remap);
}

}  // namespace

extern "C" size_t sjk_pages_bytes(uint32_t n) { return 16u + ((size_t) n * 8u + (n + 31u) / 32u + 1u) * sizeof(uint32_t); }

extern "C" int sjk_pages_init(const sjk_pages * g, sjk_stream st) {
    Params p;
    const int rc = params_of(g, &p, false);
    if (rc) return rc;
    const uint32_t ctas = (p.n_pages + NT - 1) / NT;
    return launch(pages_init_kernel, dim3(ctas < 148u ? ctas : 148u), dim3(NT), 0, st, p.l, p.n_pages);
}

extern "C" uint32_t * sjk_pages_shares(const sjk_pages * g) {
    return g && g->ledger ? ledger_of(g->ledger, g->n_pages).shares : nullptr;
}

extern "C" int sjk_pages_fork(const sjk_pages * g, const int32_t * src, const int32_t * dst, int n, int32_t * status, sjk_stream st) {
    Params p;
    const int rc = params_of(g, &p, true);
    if (rc) return rc;
    if (n < 0 || (n && (!src || !dst || !status)) || !list_ok(src) || !list_ok(dst) || !list_ok(status)) return SJKVARN_ERR_ARG;
    if (n == 0) return 0;
    p.a = src; p.b = dst; p.n = n; p.status = status;
    return launch(pages_fork_kernel, dim3((unsigned) n), dim3(NT), 0, st, p);
}

extern "C" int sjk_pages_free(const sjk_pages * g, const int32_t * rows, const int32_t * g0, const int32_t * g1, int n, sjk_stream st) {
    Params p;
    const int rc = params_of(g, &p, true);
    if (rc) return rc;
    if (n < 0 || (n && !rows) || !list_ok(rows) || !list_ok(g0) || !list_ok(g1)) return SJKVARN_ERR_ARG;
    if (n == 0) return 0;
    p.a = rows; p.b = g0; p.c = g1; p.n = n;
    uint32_t runs = (p.stride + 4 * NT - 1) / (4 * NT);     // about four entries a thread, at most a wave over all rows
    const uint32_t most = 148u * 4u / (uint32_t) n + 1u;
    if (runs > most) runs = most;
    return launch(pages_free_kernel, dim3((unsigned) n, runs), dim3(NT), 0, st, p);
}

extern "C" int sjk_pages_extend(const sjk_pages * g, const int32_t * rows, const int32_t * len, const int32_t * add, int add_all, int n,
                                int32_t * status, sjk_stream st) {
    Params p;
    int rc = params_of(g, &p, true);
    if (rc) return rc;
    if (n < 0 || n > SJK_PAGES_MAX_ROWS || (n && (!rows || !len || !status)) || (!add && add_all < 0) || !list_ok(rows) || !list_ok(len) ||
        !list_ok(add) || !list_ok(status))
        return SJKVARN_ERR_ARG;
    if (n == 0) return 0;
    if (too_many(p, (uint32_t) n)) return SJK_ERR_UNSUPPORTED;      // a request copies its first page at most
    p.a = rows; p.b = len; p.c = add; p.add_all = add_all; p.n = n; p.status = status;
    rc = n <= 256 ? launch(pages_extend_kernel<256>, dim3(1), dim3(256), 0, st, p) : launch(pages_extend_kernel<NB>, dim3(1), dim3(NB), 0, st, p);
    if (rc) return rc;
    return copy_launch(p, p.l.src, p.l.dst, -1, 0, st);
}

extern "C" int sjk_pages_compact(const sjk_pages * g, int32_t * info, sjk_stream st) {
    Params p;
    int rc = params_of(g, &p, true);
    if (rc) return rc;
    if (!list_ok(info)) return SJKVARN_ERR_ARG;
    if (too_many(p, p.n_pages / 2)) return SJK_ERR_UNSUPPORTED;     // a move needs a used page and a free one
    p.status = info;
    const size_t smem = (size_t) ((p.n_pages + 31u) / 32u) * sizeof(uint32_t);
    if (smem > 40 * 1024 && smem_limit<pages_plan_kernel>(SJK_PAGES_MAX / 8)) return SJK_ERR_DEVICE;
    rc = launch(pages_plan_kernel, dim3(1), dim3(NB), smem, st, p);
    if (rc) return rc;
    return copy_launch(p, p.l.src, p.l.dst, -1, 1, st);
}

extern "C" int sjk_pages_copy(const sjk_pages * g, const int32_t * src, const int32_t * dst, int n, sjk_stream st) {
    Params p;
    const int rc = params_of(g, &p, false);
    if (rc) return rc;
    if (n < 0 || (n && (!src || !dst)) || !list_ok(src) || !list_ok(dst)) return SJKVARN_ERR_ARG;
    if (n == 0) return 0;
    if (too_many(p, (uint32_t) n)) return SJK_ERR_UNSUPPORTED;
    return copy_launch(p, reinterpret_cast<const uint32_t *>(src), reinterpret_cast<const uint32_t *>(dst), n, 0, st);
}

int sjk_pages_status_take(void) {
    unsigned v = 0;
    if (sjk_check(cudaMemcpyFromSymbol(&v, g_pages_status, sizeof v))) return -1;
    if (v) {
        const unsigned z = 0;
        if (sjk_check(cudaMemcpyToSymbol(g_pages_status, &z, sizeof z))) return -1;
    }
    return (int) v;
}
