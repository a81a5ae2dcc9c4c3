/* s2pro MI355X — paged session caches: K/V in pages that sessions take as they
 * grow, share after a fork and give back.
 *
 * The contiguous session cache (verify.h) reserves ctx_len slots a session.  A
 * pool instead holds pages of 16 to 256 slots of every layer; a session is a row
 * of page ids (slot p of the session is place p % page of its page p / page) and
 * a token count.  Within a page the planes are those of the contiguous caches: K
 * heads, then V heads, [page][128] bf16, or the INT8 / INT4 codes and f16 group
 * scales of s2pk_kv_append8 (kernels.cu:510-581), so a page's plane is a piece of
 * a contiguous one, byte for byte.
 *
 * Conventions as in kernels.h: device pointers, asynchronous on `st` (the
 * stream's device must be the current one), no allocation and no host
 * synchronisation (hipGraph-capturable), the HIP error code is returned, bad
 * arguments are hipErrorInvalidValue before anything is launched, rows <= 0 is
 * success.  The structs are read on the host during the call.  A workspace holds
 * nothing between calls; calls that may overlap need one each, as do captured
 * graphs whose replays may. */
#ifndef S2P_PAGED_H
#define S2P_PAGED_H

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#include "s2pro/kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

#define S2P_PAGE_MAX_SESSIONS 1024 /* of a batch, of the tables */
#define S2P_PAGED_MAX_GROUP 16     /* query heads a kv head */

typedef struct {
    void*   kv;       /* [layers][pages][2 * kv_heads][page][128] bf16 (bits 16) or int8
                       * (bits 8), [..][64] bytes of two codes (bits 4: element 2b low);
                       * 16-byte aligned */
    void*   scales;   /* bits 8 / 4: f16 [layers][pages][2 * kv_heads][page][4], 16-byte
                       * aligned; NULL with bits 16 */
    int32_t layers, pages, kv_heads; /* pages <= 2^21, kv_heads <= 1024 */
    int32_t page;     /* slots a page: 16, 32, 64, 128 or 256 */
    int32_t bits;     /* 16, 8 or 4 */
} s2p_page_pool;

/* The rows of one call.  Session s has rows row0[s] .. row0[s + 1] - 1, at slots
 * len[s] + 0, 1, ..; row0 does not decrease.  A session whose rows are none, more
 * than max_rows or behind `rows`, whose len is negative or whose last slot is at or
 * past max_len is left out: nothing is written for its rows.  Rows that belong to
 * no session (the padding of a captured batch) are left as they were.  A table
 * entry outside [0, pages) is a page that is not there: nothing is written to it
 * and its slots are seen by no row. */
typedef struct {
    const int32_t* table;  /* [sessions][max_pages] */
    const int32_t* len;    /* [sessions] tokens before this call's rows */
    const int32_t* row0;   /* [sessions + 1] */
    int32_t sessions;      /* <= S2P_PAGE_MAX_SESSIONS */
    int32_t max_pages;
    int32_t rows;          /* of the row arrays */
    int32_t max_rows;      /* host bound of a session's rows */
    int32_t max_len;       /* host bound of len + rows, <= max_pages * page, <= 2^30 */
} s2p_page_batch;

/* bytes of the pool's kv and scales */
size_t s2p_page_pool_bytes(const s2p_page_pool* pool);
size_t s2p_page_pool_scale_bytes(const s2p_page_pool* pool);

/* The (cos, sin) pairs of positions 0 .. n_pos - 1, [n_pos][64][2] bf16: the values
 * s2pk_rope computes (rounded through bf16), laid out once.  head_dim 128. */
hipError_t s2pk_rope_table(s2p_bf16* tab, int n_pos, int head_dim, float rope_base,
                           hipStream_t st);

/* qk-norm, RoPE, quantisation and append in one pass over the fused qkv rows
 * [rows][(q_heads + 2 kv_heads) * 128]: row r's query heads, normed (qn_w, kn_w
 * [128]; both NULL: no norm) and rotated, to q [rows][q_heads * 128]; its K, normed
 * and rotated, and V to its slot of `layer`.  The bits are those of s2pk_qkv_split,
 * s2pk_qk_norm, s2pk_rope_pos and s2pk_kv_append_ptrs / s2pk_kv_append8_ptrs in turn.
 * rope: an s2pk_rope_table of n_pos positions.  pos: [rows] RoPE positions (a draft
 * tree's depths), or NULL: each row's slot.  A row whose position is outside the
 * table is left out.  The pages that hold the rows' slots must be the session's own
 * (s2pk_pages_reserve sees to it).  q lies apart from qkv. */
hipError_t s2pk_paged_append(const s2p_page_pool* pool, const s2p_page_batch* batch, int layer,
                             const s2p_bf16* qkv, int q_heads, const s2p_bf16* qn_w,
                             const s2p_bf16* kn_w, float eps, const s2p_bf16* rope, int n_pos,
                             const int32_t* pos, s2p_bf16* q, hipStream_t st);

/* GQA attention of every session's rows over its pages, head_dim 128, q_heads =
 * 1 .. 16 x kv_heads; q and out [rows][q_heads * 128].  Row i of a session sees slots
 * [0, len) and, with vis NULL, slots len .. len + i; else slot len + b where bit b of
 * vis[row] is set (max_rows <= 64; s2p_verify's visibility words).  The rows' own K/V
 * are in their slots already.  A row that sees no slot gets zeros.  NaN and infinities
 * in slots that a row does not see do not reach it, and a session's bits do not depend on
 * what lies behind its last slot.  work: s2pk_paged_attention_work_floats floats, 16-byte
 * aligned.  out lies apart from q.  Refused too: sessions x row tiles (max_rows in eights at worst) x 64-slot tiles
 * of max_len past 2^30. */
hipError_t s2pk_paged_attention(const s2p_page_pool* pool, const s2p_page_batch* batch, int layer,
                                const s2p_bf16* q, int q_heads, const uint64_t* vis,
                                s2p_bf16* out, float* work, hipStream_t st);
int64_t s2pk_paged_attention_work_floats(const s2p_page_batch* batch, int q_heads, int kv_heads);

/* The accepted nodes of a verify batch to their final slots, every layer: node
 * path[row0[s] + d - 1] of session s from slot len + node to len + d, d = 1 ..
 * n_acc[s] (path and n_acc as s2p_verify_accept leaves them; nodes increase along a
 * path), then len_out[s] = len[s] + 1 + n_acc[s] (len_out may be the batch's len, or
 * NULL).  A session with n_acc < 0, or left out of the batch, keeps everything; n_acc
 * past the session's rows - 1 counts as rows - 1.  max_rows <= 64. */
hipError_t s2pk_paged_commit(const s2p_page_pool* pool, const s2p_page_batch* batch,
                             const int32_t* path, const int32_t* n_acc, int32_t* len_out,
                             hipStream_t st);

/* The pages' bookkeeping, device resident.  ref counts the sessions that hold a page
 * (0: free); session s holds table[s][0 .. held[s] - 1], which cover its len[s]
 * tokens.  A program starts from zeros in ref, held and len, raises len as it writes
 * tokens into the room it reserved, and lowers it through s2pk_pages_free alone.  Every
 * session that holds pages of the pool is a row here.  Calls on one set of tables are
 * ordered by their stream. */
typedef struct {
    int32_t* ref;    /* [pages] */
    int32_t* table;  /* [sessions][max_pages] */
    int32_t* held;   /* [sessions] */
    int32_t* len;    /* [sessions] */
    int32_t sessions, max_pages; /* sessions <= S2P_PAGE_MAX_SESSIONS */
} s2p_page_tables;

/* int32s of the workspace of s2pk_pages_reserve and s2pk_pages_compact */
int64_t s2pk_pages_work_ints(const s2p_page_pool* pool, const s2p_page_tables* tab);

/* Room for want[s] more tokens (sessions with want <= 0 are passed over): the pages
 * that are missing come from the free ones, lowest ids first, in session order; a
 * partly filled last page that other sessions hold too is replaced by a copy of it
 * (every layer), except for the last of its holders.  granted[s] (may be NULL) is 1
 * if the session has its room; a session that would need more than max_pages pages,
 * or for which, with those before it, too few pages are free, gets nothing and is
 * left as it was.  Deterministic. */
hipError_t s2pk_pages_reserve(const s2p_page_pool* pool, const s2p_page_tables* tab,
                              const int32_t* want, int32_t* granted, int32_t* work,
                              hipStream_t st);

/* Session dst[i] becomes a continuation of session src[i], i < n: it holds the same
 * pages (those of the source's tokens) and as many tokens.  done[i] (may be NULL) is 1,
 * or 0 where nothing was done: an index outside the tables, a source without tokens, a
 * destination that holds pages or that an earlier entry names too, an entry one of whose
 * sessions this call names both as a source and as a destination. */
hipError_t s2pk_pages_fork(const s2p_page_pool* pool, const s2p_page_tables* tab,
                           const int32_t* src, const int32_t* dst, int n, int32_t* done,
                           hipStream_t st);

/* Session s keeps its first keep[s] tokens (at most its len) and the pages that hold
 * them, and gives the others back; keep[s] = 0 ends it, keep[s] < 0 passes it over. */
hipError_t s2pk_pages_free(const s2p_page_pool* pool, const s2p_page_tables* tab,
                           const int32_t* keep, hipStream_t st);

/* Moves the pages in use to ids 0 .. n_live - 1, every layer: the pages behind go, in
 * order, to the free ones before; tables and counts follow.  *n_live (device, may be
 * NULL) is the pages in use. */
hipError_t s2pk_pages_compact(const s2p_page_pool* pool, const s2p_page_tables* tab,
                              int32_t* n_live, int32_t* work, hipStream_t st);

#ifdef __cplusplus
}
#endif
#endif
