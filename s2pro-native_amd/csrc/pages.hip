/* s2pro MI355X — the bookkeeping of paged session caches: room for the next
 * tokens, forks, freeing and compaction.
 *
 * The state is a reference count a page and the sessions' tables; there is no free
 * list, a free page is one whose count is 0.  Freed pages then need no order among
 * each other (counts fall by atomics, in any order), and what a call hands out (the
 * lowest free ids) depends on the counts alone, not on what happened before.  The
 * price is a scan of the counts, 4 bytes a page, by one workgroup.
 * Payload is moved by one launch over (page, layer, 16 KB piece) items, as many as the
 * device's list says; that copy is what bounds a fork's first tokens and a compaction.
 * The others are bound by their chain of loads: launch, count, table, count again.
 *
 * MI355X, pages of 16 slots: 4 forks of 1,000 tokens 3.4 us, the reservation after them 5.9
 * and its copies 2.9; 32 forks of 4,090 tokens at 36 layers 4.8, 7.1 and 14.6 (151 MB, read
 * from cache); 100 of 333 pages kept and moved together: freeing 2.8 us, plan 4.1, moves 3.9;
 * 200 pages of 36 layers (944 MB): 4.6, 5.2 and 195 (4.8 TB/s; a 2 GiB copy runs at 4.9). */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemv_internal.h"
#include "paged_dev.h"

#define PT 1024     /* threads of the workgroup that scans the counts */
#define PT_EACH 8   /* counts a thread takes at a time */
#define PC_PIECE 16384

/* inclusive sum over the 64 lanes, on the vector unit: within rows of 16, then the rows' last
 * lanes to the rows behind */
template <int CTRL, int ROWS>
S2P_DEV uint32_t add_dpp(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
S2P_DEV uint32_t wave_scan(uint32_t v) {
    v = add_dpp<0x111, 0xF>(v); /* row_shr:1 */
    v = add_dpp<0x112, 0xF>(v);
    v = add_dpp<0x114, 0xF>(v);
    v = add_dpp<0x118, 0xF>(v);
    v = add_dpp<0x142, 0xA>(v); /* row_bcast:15 into rows 1, 3 */
    return add_dpp<0x143, 0xC>(v); /* row_bcast:31 into rows 2, 3 */
}
/* inclusive sum over the block; *total for everybody */
S2P_DEV uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads(); /* lds may still be read from the scan before */
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PT / 64; w++) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    *total = all;
    return v + before;
}

/* PT_EACH counts from i on as a mask of those that are free (FREE) or in use */
template <bool FREE>
S2P_DEV unsigned page_mask(const int32_t* ref, int i, int pages) {
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < PT_EACH; k++) {
        const int r = i + k < pages ? ref[i + k] : (FREE ? 1 : 0);
        if (FREE ? r == 0 : r != 0) m |= 1u << k;
    }
    return m;
}

/* work: [0] pairs, [4 ..) sources, then destinations (sessions each), then the free
 * pages in order (those past the first PT_NEAR, which stay in LDS) */
#define PT_NEAR 4096
__global__ __launch_bounds__(PT) void k_pages_reserve(s2p_page_tables t, int pages, int shift,
                                                      const int32_t* __restrict__ want,
                                                      int32_t* __restrict__ granted,
                                                      int32_t* __restrict__ work) {
    __shared__ __align__(16) uint32_t s_scan[PT / 64];
    __shared__ uint32_t s_upto[PT]; /* pages needed by the sessions up to this one */
    __shared__ __align__(16) int s_mine[PT]; /* the session's partly filled page, or -1 */
    __shared__ int s_held[PT], s_len[PT], s_copy[PT], s_rank[PT], s_free[PT_NEAR];
    const int s = threadIdx.x, page = 1 << shift;
    unsigned near = page_mask<true>(t.ref, s * PT_EACH, pages); /* on its way from the start */
    int held = 0, L = 0, more = 0, mine = -1, copy = 0;
    bool fits = false;
    if (s < t.sessions) {
        const int w = want[s];
        L = t.len[s];
        held = t.held[s];
        if (w > 0 && L >= 0 && held >= 0 && held <= t.max_pages &&
            (((int64_t)L + page - 1) >> shift) <= held) {
            const int64_t room = ((int64_t)L + w + page - 1) >> shift;
            fits = room <= t.max_pages;
            if (fits) {
                more = room > held ? (int)room - held : 0;
                if (L & (page - 1)) {
                    mine = t.table[(size_t)s * t.max_pages + (L >> shift)];
                    if ((unsigned)mine >= (unsigned)pages) { /* a table that was not kept here */
                        fits = false;
                        more = 0;
                        mine = -1;
                    }
                }
            }
        }
    }
    const int holders = mine >= 0 ? t.ref[mine] : 0;
    s_mine[s] = mine;
    s_held[s] = held;
    s_len[s] = L;
    __syncthreads();
    if (holders > 1) { /* all but the last of a page's holders copy it */
        int before = 0;
        for (int u = 0; u < s; u += 4) {
            const int4 m = *(const int4*)&s_mine[u];
            before += (m.x == mine) + (u + 1 < s && m.y == mine) + (u + 2 < s && m.z == mine) +
                      (u + 3 < s && m.w == mine);
        }
        copy = before < holders - 1;
    }
    /* 32 bits hold 1,024 sessions' needs, none counted for more than one page over all there are */
    uint32_t total, found = 0;
    const uint32_t need = min((uint32_t)more + (uint32_t)copy, (uint32_t)pages + 1);
    s_upto[s] = block_scan(need, s_scan, &total);
    /* the free pages, in order, until there are enough */
    int32_t* const fre = work + 4 + 2 * t.sessions;
    for (int i0 = 0; i0 < pages && found < total; i0 += PT * PT_EACH) {
        const int i = i0 + s * PT_EACH;
        unsigned m = i0 ? page_mask<true>(t.ref, i, pages) : near;
        const int c = __popc(m);
        uint32_t n, at = found + block_scan(c, s_scan, &n) - c;
        while (m) {
            const int id = i + __ffs(m) - 1;
            if (at < PT_NEAR) s_free[at] = id;
            else fre[at] = id;
            at++;
            m &= m - 1;
        }
        found += n;
        if (pages - i0 <= PT * PT_EACH) break; /* i0 stays in range */
    }
    const bool ok = fits && s_upto[s] <= found;
    if (!ok) copy = 0;
    s_copy[s] = copy;
    uint32_t pairs, give; /* what is granted is a prefix of the needs */
    s_rank[s] = (int)block_scan(copy, s_scan, &pairs) - copy;
    block_scan(ok ? need : 0, s_scan, &give);
    if (s == 0) work[0] = (int)pairs;
    if (granted && s < t.sessions) granted[s] = ok ? 1 : 0;
    if (ok) t.held[s] = held + more;
    __syncthreads();
    for (uint32_t r = s; r < give; r += PT) {
        int lo = 0, hi = t.sessions - 1; /* the first session whose needs reach past r */
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_upto[mid] > r) hi = mid;
            else lo = mid + 1;
        }
        const int k = (int)(r - (lo ? s_upto[lo - 1] : 0)), id = r < PT_NEAR ? s_free[r] : fre[r];
        int32_t* row = t.table + (size_t)lo * t.max_pages;
        t.ref[id] = 1;
        if (k < s_copy[lo]) {
            const int old = s_mine[lo];
            row[s_len[lo] >> shift] = id;
            work[4 + s_rank[lo]] = old;
            work[4 + t.sessions + s_rank[lo]] = id;
            atomicSub(t.ref + old, 1);
        } else {
            row[s_held[lo] + k - s_copy[lo]] = id;
        }
    }
}

struct PgCopy {
    char *kv, *sc;
    size_t kv_page, sc_page;   /* bytes of a page of one layer */
    size_t kv_layer, sc_layer; /* bytes of a layer */
    const int32_t *n, *src, *dst;
    int layers, kv_pieces, pieces;
};

/* A compaction's new ids into the tables: to[id - live] of a page from `live` on. */
struct PgRename {
    s2p_page_tables t;
    const int32_t *live, *to;
    int pages;
};
S2P_DEV void pages_rename(const PgRename& r, int s) {
    const int held = min(r.t.held[s], r.t.max_pages), live = *r.live;
    int32_t* row = r.t.table + (size_t)s * r.t.max_pages;
    for (int j = threadIdx.x; j < held; j += 256) {
        const int id = row[j];
        if (id >= live && id < r.pages) row[j] = r.to[id - live];
    }
}

/* One 16 KB piece of a page of a layer (or of its scales) an item; RENAME: the tables too, a
 * session a block, beside the copy (a launch of its own cost 4 us of 20). */
template <bool RENAME>
__global__ __launch_bounds__(256) void k_pages_copy(PgCopy c, PgRename r) {
    if (RENAME)
        for (int s = blockIdx.x; s < r.t.sessions; s += gridDim.x) pages_rename(r, s);
    const int64_t items = (int64_t)*c.n * c.layers * c.pieces;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int pc = (int)(it % c.pieces);
        const int64_t rest = it / c.pieces;
        const int layer = (int)(rest % c.layers), pair = (int)(rest / c.layers);
        const int from = c.src[pair], to = c.dst[pair];
        const bool kv = pc < c.kv_pieces;
        const size_t bytes = kv ? c.kv_page : c.sc_page;
        char* const base = kv ? c.kv + c.kv_layer * layer : c.sc + c.sc_layer * layer;
        const size_t off = (size_t)(kv ? pc : pc - c.kv_pieces) * PC_PIECE;
        const char* s = base + bytes * from + off;
        char* d = base + bytes * to + off;
        const int n = (int)(bytes - off < PC_PIECE ? bytes - off : PC_PIECE);
        s2p_u32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int o = (k * 256 + threadIdx.x) * 16;
            if (o < n) v[k] = *(const s2p_u32x4*)(s + o);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int o = (k * 256 + threadIdx.x) * 16;
            if (o < n) *(s2p_u32x4*)(d + o) = v[k];
        }
    }
}

/* most: the pairs that there can be */
static hipError_t copy_launch(const s2p_page_pool* p, const int32_t* n, const int32_t* src,
                              const int32_t* dst, int most, const PgRename* r, hipStream_t st) {
    const size_t slots = (size_t)2 * p->kv_heads * p->page;
    PgCopy c = {};
    c.kv = (char*)p->kv;
    c.kv_page = slots * pg_slot_bytes(p->bits);
    c.kv_layer = c.kv_page * p->pages;
    c.kv_pieces = (int)((c.kv_page + PC_PIECE - 1) / PC_PIECE);
    c.pieces = c.kv_pieces;
    if (p->bits != 16) {
        c.sc = (char*)p->scales;
        c.sc_page = slots * 8;
        c.sc_layer = c.sc_page * p->pages;
        c.pieces += (int)((c.sc_page + PC_PIECE - 1) / PC_PIECE);
    }
    c.n = n;
    c.src = src;
    c.dst = dst;
    c.layers = p->layers;
    const int64_t items = (int64_t)most * p->layers * c.pieces;
    const int64_t full = 8 * (int64_t)s2p_cu_count();
    const dim3 grid((unsigned)(items < full ? items : full));
    if (r) hipLaunchKernelGGL((k_pages_copy<true>), grid, dim3(256), 0, st, c, *r);
    else hipLaunchKernelGGL((k_pages_copy<false>), grid, dim3(256), 0, st, c, PgRename{});
    return hipGetLastError();
}

__global__ __launch_bounds__(256) void k_pages_fork(s2p_page_tables t, int pages, int shift,
                                                    const int32_t* __restrict__ src,
                                                    const int32_t* __restrict__ dst, int n,
                                                    int32_t* __restrict__ done) {
    const int i = blockIdx.x, a = src[i], b = dst[i];
    /* what other entries decide is read from the lists alone: no block reads a row
     * that another one writes */
    bool bad = (unsigned)a >= (unsigned)t.sessions || (unsigned)b >= (unsigned)t.sessions;
    for (int k = threadIdx.x; k < n; k += 256)
        bad |= dst[k] == a || src[k] == b || (k < i && dst[k] == b);
    if (!__syncthreads_or(bad)) {
        const int L = t.len[a], held = t.held[a];
        const int64_t cover = ((int64_t)L + (1 << shift) - 1) >> shift;
        bad = t.held[b] != 0 || L <= 0 || cover > held || held > t.max_pages;
        if (!bad) {
            const int32_t* from = t.table + (size_t)a * t.max_pages;
            int32_t* to = t.table + (size_t)b * t.max_pages;
            for (int k = threadIdx.x; k < cover; k += 256) {
                const int id = from[k];
                to[k] = id;
                if ((unsigned)id < (unsigned)pages) atomicAdd(t.ref + id, 1);
            }
            __syncthreads(); /* everybody has read held[b] */
            if (threadIdx.x == 0) {
                t.held[b] = (int)cover;
                t.len[b] = L;
            }
        }
    } else {
        bad = true;
    }
    if (done && threadIdx.x == 0) done[i] = bad ? 0 : 1;
}

__global__ __launch_bounds__(256) void k_pages_free(s2p_page_tables t, int pages, int shift,
                                                    const int32_t* __restrict__ keep) {
    const int s = blockIdx.x, k = keep[s];
    const int L = t.len[s], held = t.held[s];
    if (k < 0 || L < 0 || held < 0 || held > t.max_pages) return;
    const int n = min(k, L);
    const int stay = (int)min((int64_t)held, ((int64_t)n + (1 << shift) - 1) >> shift);
    int32_t* row = t.table + (size_t)s * t.max_pages;
    for (int j = stay + (int)threadIdx.x; j < held; j += 256) {
        const int id = row[j];
        if ((unsigned)id < (unsigned)pages) atomicSub(t.ref + id, 1);
        row[j] = -1;
    }
    __syncthreads(); /* everybody has read the session */
    if (threadIdx.x == 0) {
        t.held[s] = stay;
        t.len[s] = n;
    }
}

/* work: [0] moves, [1] pages in use, [4 ..) sources and destinations (pages / 2 + 1
 * each), then the new id of every page behind the first `live` */
__global__ __launch_bounds__(PT) void k_pages_plan(int32_t* __restrict__ ref, int pages,
                                                   int32_t* __restrict__ n_live,
                                                   int32_t* __restrict__ work) {
    __shared__ __align__(16) uint32_t s_scan[PT / 64];
    const int tid = threadIdx.x;
    uint32_t mine = 0, live;
    for (int64_t i = (int64_t)tid * PT_EACH; i < pages; i += PT * PT_EACH)
        mine += __popc(page_mask<false>(ref, (int)i, pages));
    block_scan(mine, s_scan, &live);
    int32_t *src = work + 4, *dst = src + pages / 2 + 1, *to = dst + pages / 2 + 1;
    uint32_t holes = 0, movers = 0;
    for (int64_t i0 = 0; i0 < pages; i0 += PT * PT_EACH) {
        const int64_t i = i0 + tid * PT_EACH;
        unsigned used = i < pages ? page_mask<false>(ref, (int)i, pages) : 0u;
        unsigned front = 0; /* of this thread's pages, those before `live` */
        for (int k = 0; k < PT_EACH; k++)
            if (i + k < live) front |= 1u << k;
        unsigned h = ~used & front, m = used & ~front;
        /* both counts (8,192 at most) in one scan */
        uint32_t all;
        const uint32_t c = (uint32_t)__popc(h) | ((uint32_t)__popc(m) << 16);
        const uint32_t at = block_scan(c, s_scan, &all) - c;
        uint32_t ah = holes + (at & 0xFFFF), am = movers + (at >> 16);
        while (h) {
            dst[ah++] = (int)(i + __ffs(h) - 1);
            h &= h - 1;
        }
        while (m) {
            src[am++] = (int)(i + __ffs(m) - 1);
            m &= m - 1;
        }
        holes += all & 0xFFFF;
        movers += all >> 16;
    }
    __syncthreads();
    for (uint32_t k = tid; k < movers; k += PT) { /* as many holes as movers */
        const int a = src[k], b = dst[k];
        to[a - live] = b;
        ref[b] = ref[a];
        ref[a] = 0;
    }
    if (tid == 0) {
        work[0] = (int)movers;
        work[1] = (int)live;
        if (n_live) *n_live = (int)live;
    }
}

static bool tables_ok(const s2p_page_pool* p, const s2p_page_tables* t) {
    return pg_pool_ok(p) && t && t->ref && t->table && t->held && t->len && t->sessions > 0 &&
           t->sessions <= S2P_PAGE_MAX_SESSIONS && t->max_pages > 0;
}

extern "C" int64_t s2pk_pages_work_ints(const s2p_page_pool* pool, const s2p_page_tables* tab) {
    if (!pool || !tab || pool->pages <= 0 || tab->sessions <= 0) return 0;
    return 4 + 2 * ((int64_t)pool->pages + 1) + 2 * (int64_t)tab->sessions;
}

extern "C" hipError_t s2pk_pages_reserve(const s2p_page_pool* pool, const s2p_page_tables* tab,
                                         const int32_t* want, int32_t* granted, int32_t* work,
                                         hipStream_t st) {
    if (!tables_ok(pool, tab) || !want || !work) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_pages_reserve, dim3(1), dim3(PT), 0, st, *tab, pool->pages,
                       pg_shift(pool->page), want, granted, work);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return copy_launch(pool, work, work + 4, work + 4 + tab->sessions, tab->sessions, nullptr, st);
}

extern "C" hipError_t s2pk_pages_fork(const s2p_page_pool* pool, const s2p_page_tables* tab,
                                      const int32_t* src, const int32_t* dst, int n, int32_t* done,
                                      hipStream_t st) {
    if (n <= 0) return hipSuccess;
    if (!tables_ok(pool, tab) || !src || !dst) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_pages_fork, dim3((unsigned)n), dim3(256), 0, st, *tab, pool->pages,
                       pg_shift(pool->page), src, dst, n, done);
    return hipGetLastError();
}

extern "C" hipError_t s2pk_pages_free(const s2p_page_pool* pool, const s2p_page_tables* tab,
                                      const int32_t* keep, hipStream_t st) {
    if (!tables_ok(pool, tab) || !keep) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_pages_free, dim3((unsigned)tab->sessions), dim3(256), 0, st, *tab,
                       pool->pages, pg_shift(pool->page), keep);
    return hipGetLastError();
}

extern "C" hipError_t s2pk_pages_compact(const s2p_page_pool* pool, const s2p_page_tables* tab,
                                         int32_t* n_live, int32_t* work, hipStream_t st) {
    if (!tables_ok(pool, tab) || !work) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_pages_plan, dim3(1), dim3(PT), 0, st, tab->ref, pool->pages, n_live, work);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int each = pool->pages / 2 + 1; /* as k_pages_plan lays the workspace out */
    const PgRename r = {*tab, work + 1, work + 4 + 2 * each, pool->pages};
    return copy_launch(pool, work, work + 4, work + 4 + each, each, &r, st);
}
