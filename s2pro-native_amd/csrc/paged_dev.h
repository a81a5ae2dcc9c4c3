/* s2pro MI355X — what the paged-cache kernels share: the descriptors as the
 * kernels take them, their checks, and the addresses of slots. */
#ifndef S2P_PAGED_DEV_H
#define S2P_PAGED_DEV_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "s2pro/paged.h"

#define PG_HD 128

static inline bool pg_pool_ok(const s2p_page_pool* p) {
    if (!p || !p->kv || ((uintptr_t)p->kv & 15)) return false;
    if (p->bits != 16 && p->bits != 8 && p->bits != 4) return false;
    if (p->bits != 16 && (!p->scales || ((uintptr_t)p->scales & 15))) return false;
    if (p->page < 16 || p->page > 256 || (p->page & (p->page - 1))) return false;
    /* pages: 1,024 sessions' needs of them are summed in 32 bits */
    return p->layers > 0 && p->pages > 0 && p->pages <= 1 << 21 && p->kv_heads > 0 &&
           p->kv_heads <= 1024;
}
static inline bool pg_batch_ok(const s2p_page_pool* p, const s2p_page_batch* b) {
    if (!b || !b->table || !b->len || !b->row0) return false;
    if (b->sessions <= 0 || b->sessions > S2P_PAGE_MAX_SESSIONS || b->max_pages <= 0) return false;
    if (b->max_rows <= 0 || b->max_rows > b->max_len || b->max_len > 1 << 30) return false;
    return (int64_t)b->max_len <= (int64_t)b->max_pages * p->page;
}
/* query heads a kv head; 0: a grouping there is none of */
static inline int pg_group(int q_heads, int kv_heads) {
    if (q_heads <= 0 || q_heads % kv_heads) return 0;
    const int g = q_heads / kv_heads;
    return g <= S2P_PAGED_MAX_GROUP ? g : 0;
}
/* bytes of a slot's row in a plane */
static inline int pg_slot_bytes(int bits) { return bits == 16 ? 256 : bits == 8 ? 128 : 64; }
static inline int pg_shift(int page) { return __builtin_ctz((unsigned)page); }

/* one layer of the pool: page id i, plane h at (i * planes + h) * page slots */
struct PgLayer {
    char* kv;
    uint16_t* sc;
    int pages, planes, page, shift;
};
static inline PgLayer pg_layer(const s2p_page_pool* p, int layer) {
    const size_t slots = (size_t)p->pages * 2 * p->kv_heads * p->page * layer;
    PgLayer l;
    l.kv = (char*)p->kv + slots * pg_slot_bytes(p->bits);
    l.sc = p->bits == 16 ? nullptr : (uint16_t*)p->scales + slots * 4;
    l.pages = p->pages;
    l.planes = 2 * p->kv_heads;
    l.page = p->page;
    l.shift = pg_shift(p->page);
    return l;
}

/* the rows of session s, or n = 0 where it is left out */
struct PgSess {
    int r0, n, L;
};
S2P_DEV PgSess pg_session(const s2p_page_batch& b, int s) {
    PgSess o;
    o.r0 = b.row0[s];
    const int r1 = b.row0[s + 1];
    o.L = b.len[s];
    o.n = 0;
    if (o.r0 >= 0 && r1 > o.r0 && r1 <= b.rows && o.L >= 0) {
        const int n = r1 - o.r0;
        if (n <= b.max_rows && o.L <= b.max_len - n) o.n = n;
    }
    return o;
}

#endif
