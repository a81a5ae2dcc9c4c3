/* s2pro MI355X — appending to paged session caches: qk-norm, RoPE, quantisation
 * and append in one pass, the RoPE table, and the commit of accepted nodes.
 *
 * Append: y = bf16((x inv) w), inv = 1 / sqrt(mean(x^2) + eps) over a head's 128
 * values; the neighbouring pairs of y turned by the position's (cos, sin); K and V
 * into the row's slot, as codes c = clamp(rint(x / s)) with s = f16(absmax / QMAX)
 * a group of 32.  A row is read once and written once, which is what bounds a
 * prompt chunk; a decode tick is bound by the launch and the loads that follow one
 * another (row0, len, table).
 * A wave takes four heads of a row, 16 lanes a head with eight neighbouring
 * elements each: 16-byte loads and stores, a lane's four rotation pairs one 16-byte
 * load, and a scale group is four lanes.  The sum of squares runs over the tree of
 * s2pk_qk_norm (elements 64, 32, 16, 8 apart across lanes, 4, 2, 1 within one), so the
 * bits are those of the separate launchers.
 *
 * MI355X, 32 query and 8 kv heads: 64 decode rows 3.2 us; 7,023 prompt rows into INT8
 * pages 38 us (161 MB read and written, 4.2 TB/s), of which the norm's root and
 * the codes' arithmetic are about 5. */
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "gemv_internal.h"
#include "paged_dev.h"
#include "prims_dev.h"

struct PgAppend {
    PgLayer l;
    s2p_page_batch b;
    const uint16_t *qkv, *qn, *kn;
    const uint32_t* rope; /* [n_pos][64] (cos low, sin high) */
    const int32_t* pos;
    uint16_t* q;
    float eps;
    int n_pos, qh, kvh;
};

S2P_DEV float pa_max4(float v) { /* over the quad */
    v = fmaxf(v, dpp_f<0xB1>(v));
    return fmaxf(v, dpp_f<0x4E>(v));
}

/* two floats as a bf16 pair, one conversion for both */
S2P_DEV uint32_t pa_pk(float a, float b) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f2;
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 b2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
}

/* a wave: IT items (of four heads) of a row */
template <int BW, int IT>
__global__ __launch_bounds__(256) void k_paged_append(PgAppend a) {
#pragma clang fp contract(off)
    const int lane = threadIdx.x & 63, j = lane & 15;
    const int heads = a.qh + 2 * a.kvh, waves = (heads + 4 * IT - 1) / (4 * IT); /* of a row */
    const uint32_t wv = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = __builtin_amdgcn_readfirstlane((int)(wv / (uint32_t)waves));
    if (row >= a.b.rows) return;
    const int head0 = (int)(wv % (uint32_t)waves) * 4 * IT + (lane >> 4);
    s2p_u32x4 xin[IT];
#pragma unroll
    for (int it = 0; it < IT; it++)
        if (head0 + 4 * it < heads)
            xin[it] = *(const s2p_u32x4*)(a.qkv + ((size_t)row * heads + head0 + 4 * it) * PG_HD + 8 * j);
    /* the row's session: as many as end at or before it */
    int s = 0;
    for (int i = 0; i < a.b.sessions; i += 64)
        s += __popcll(__ballot(i + lane < a.b.sessions && a.b.row0[i + lane + 1] <= row));
    if (s >= a.b.sessions) return;
    const PgSess ss = pg_session(a.b, s);
    const int i = row - ss.r0;
    if (i < 0 || i >= ss.n) return;
    const int slot = ss.L + i;
    const int p = a.pos ? a.pos[row] : slot;
    if (p < 0 || p >= a.n_pos) return;
    const int id = a.b.table[(size_t)s * a.b.max_pages + (slot >> a.l.shift)];
    const s2p_u32x4 cs = *(const s2p_u32x4*)(a.rope + (size_t)p * 64 + 4 * j);
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int head = head0 + 4 * it;
        if (head >= heads) return; /* nor the ones behind it */
        const bool is_q = head < a.qh, is_v = head >= a.qh + a.kvh;
        s2p_u32x4 xw = xin[it];
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            x[2 * k] = bf2f_lo(xw[k]);
            x[2 * k + 1] = bf2f_hi(xw[k]);
        }
        if (!is_v) {
            const uint16_t* w = is_q ? a.qn : a.kn;
            if (w) {
                float t[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    t[k] = fmaf(x[k], x[k], 0.f);
                    t[k] += dpp_f<0x128>(t[k]); /* row_ror:8 */
                    t[k] += dpp_f<0x124>(t[k]);
                    t[k] += dpp_f<0x122>(t[k]);
                    t[k] += dpp_f<0x121>(t[k]);
                }
                const float sum = ((t[0] + t[4]) + (t[2] + t[6])) + ((t[1] + t[5]) + (t[3] + t[7]));
                const float inv = rsqrt_rule(sum / 128.0f + a.eps);
                const s2p_u32x4 ww = *(const s2p_u32x4*)(w + 8 * j);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t y = pa_pk(__fmul_rn(__fmul_rn(x[2 * k], inv), bf2f_lo(ww[k])),
                                             __fmul_rn(__fmul_rn(x[2 * k + 1], inv), bf2f_hi(ww[k])));
                    x[2 * k] = bf2f_lo(y);
                    x[2 * k + 1] = bf2f_hi(y);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float c = bf2f_lo(cs[k]), sn = bf2f_hi(cs[k]);
                const float x0 = x[2 * k], x1 = x[2 * k + 1];
                xw[k] = pa_pk(__fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, sn)),
                              __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, sn)));
            }
        }
        if (is_q) {
            *(s2p_u32x4*)(a.q + ((size_t)row * a.qh + head) * PG_HD + 8 * j) = xw;
            continue;
        }
        if ((unsigned)id >= (unsigned)a.l.pages) continue;
        const size_t at = (((size_t)id * a.l.planes + (head - a.qh)) << a.l.shift) +
                          (slot & (a.l.page - 1));
        if constexpr (BW == 16) {
            *(s2p_u32x4*)(a.l.kv + at * 256 + 16 * j) = xw;
        } else {
            constexpr int QMAX = BW == 8 ? 127 : 7;
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[2 * k] = bf2f_lo(xw[k]);
                x[2 * k + 1] = bf2f_hi(xw[k]);
                m = fmaxf(m, fmaxf(fabsf(x[2 * k]), fabsf(x[2 * k + 1])));
            }
            m = pa_max4(m);
            const uint16_t hs = f2h(__fdiv_rn(m, (float)QMAX));
            const float sc = h2f(hs);
            /* rint(x / s) from x (1 / s): the product is within 3.1e-5 of the rounded quotient where that
             * is under 128 (2^-23 of it from the reciprocal, 2^-24 each from product and quotient), so
             * only a value closer than 4e-5 to a half needs the division (2,048 rows over INT8 take
             * 15.2 us so, 16.2 with divisions throughout) */
            const float inv = __builtin_amdgcn_rcpf(sc);
            float c8[8], far = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float y = __fmul_rn(x[k], inv);
                c8[k] = rintf(y);
                far = fmaxf(far, fabsf(__fsub_rn(y, c8[k])));
            }
            if (__any(far > 0.5f - 4e-5f)) {
#pragma unroll
                for (int k = 0; k < 8; k++) c8[k] = rintf(__fdiv_rn(x[k], sc));
            }
            uint32_t w[2] = {0u, 0u};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                int c = sc > 0.f ? (int)c8[k] : 0;
                c = max(-QMAX, min(QMAX, c));
                if (BW == 8) w[k >> 2] |= (uint32_t)(c & 0xFF) << (8 * (k & 3));
                else w[0] |= (uint32_t)(c & 0xF) << (4 * k);
            }
            if constexpr (BW == 8) *(s2p_u32x2*)(a.l.kv + at * 128 + 8 * j) = (s2p_u32x2){w[0], w[1]};
            else *(uint32_t*)(a.l.kv + at * 64 + 4 * j) = w[0];
            if ((j & 3) == 0) a.l.sc[at * 4 + (j >> 2)] = hs;
        }
    }
}

template <int IT>
static hipError_t pa_launch(const PgAppend& a, int bits, hipStream_t st) {
    const int64_t waves = (int64_t)a.b.rows * ((a.qh + 2 * a.kvh + 4 * IT - 1) / (4 * IT));
    if (waves > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((waves + 3) / 4));
    if (bits == 16) hipLaunchKernelGGL((k_paged_append<16, IT>), grid, dim3(256), 0, st, a);
    else if (bits == 8) hipLaunchKernelGGL((k_paged_append<8, IT>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_paged_append<4, IT>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

extern "C" hipError_t s2pk_paged_append(const s2p_page_pool* pool, const s2p_page_batch* batch,
                                        int layer, const s2p_bf16* qkv, int q_heads,
                                        const s2p_bf16* qn_w, const s2p_bf16* kn_w, float eps,
                                        const s2p_bf16* rope, int n_pos, const int32_t* pos,
                                        s2p_bf16* q, hipStream_t st) {
    if (batch && batch->rows <= 0) return hipSuccess;
    if (!pg_pool_ok(pool) || !pg_batch_ok(pool, batch) || layer < 0 || layer >= pool->layers ||
        !pg_group(q_heads, pool->kv_heads) || !qkv || !rope || !q || n_pos <= 0 ||
        (!qn_w) != (!kn_w) || (const void*)qkv == (void*)q ||
        (((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)rope | (uintptr_t)qn_w | (uintptr_t)kn_w) & 15))
        return hipErrorInvalidValue;
    PgAppend a = {};
    a.l = pg_layer(pool, layer);
    a.b = *batch;
    a.qkv = (const uint16_t*)qkv;
    a.qn = (const uint16_t*)qn_w;
    a.kn = (const uint16_t*)kn_w;
    a.rope = (const uint32_t*)rope;
    a.pos = pos;
    a.q = (uint16_t*)q;
    a.eps = eps;
    a.n_pos = n_pos;
    a.qh = q_heads;
    a.kvh = pool->kv_heads;
    /* three items a wave share the row's lookups; one each where the chip is not full anyway */
    return (int64_t)batch->rows * (q_heads + 2 * pool->kv_heads) > 128 * (int64_t)s2p_cu_count()
               ? pa_launch<3>(a, pool->bits, st) : pa_launch<1>(a, pool->bits, st);
}

/* ------------------------------------------------------------ RoPE table */

__global__ __launch_bounds__(256) void k_rope_table(uint32_t* tab, int n_pos, float base) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)n_pos * 64) return;
    float c, s;
    rope_cs((int)(i >> 6), (int)(i & 63), PG_HD, base, &c, &s);
    tab[i] = (uint32_t)f2bf(c) | ((uint32_t)f2bf(s) << 16);
}

extern "C" hipError_t s2pk_rope_table(s2p_bf16* tab, int n_pos, int head_dim, float rope_base,
                                      hipStream_t st) {
    if (n_pos <= 0) return hipSuccess;
    if (!tab || ((uintptr_t)tab & 15) || head_dim != PG_HD || n_pos > (1 << 28) ||
        !(rope_base > 0.f))
        return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_rope_table, dim3((unsigned)(((int64_t)n_pos * 64 + 255) / 256)), dim3(256),
                       0, st, (uint32_t*)tab, n_pos, rope_base);
    return hipGetLastError();
}

/* ---------------------------------------------------------------- commit */

/* One wave a (session, layer, plane); a lane moves the same bytes of every slot, so
 * the moves of a path follow one another within the lane. */
__global__ __launch_bounds__(64) void k_paged_commit(PgLayer l, size_t layer_bytes,
                                                     size_t layer_scales, int slot_bytes,
                                                     s2p_page_batch b,
                                                     const int32_t* __restrict__ path,
                                                     const int32_t* __restrict__ n_acc) {
    const int s = blockIdx.x, plane = blockIdx.y, layer = blockIdx.z, lane = threadIdx.x;
    const PgSess ss = pg_session(b, s);
    const int n = min(n_acc[s], ss.n - 1);
    char* kv = l.kv + layer_bytes * layer;
    uint16_t* sc = l.sc ? l.sc + layer_scales * layer : nullptr;
    const int32_t* row = b.table + (size_t)s * b.max_pages;
    for (int d = 1; d <= n; d++) {
        const int node = path[ss.r0 + d - 1];
        if (node <= d || node >= ss.n) continue; /* in place, or no node behind it */
        const int from = ss.L + node, to = ss.L + d;
        const int pf = row[from >> l.shift], pt = row[to >> l.shift];
        if ((unsigned)pf >= (unsigned)l.pages || (unsigned)pt >= (unsigned)l.pages) continue;
        const size_t f = (((size_t)pf * l.planes + plane) << l.shift) + (from & (l.page - 1));
        const size_t t = (((size_t)pt * l.planes + plane) << l.shift) + (to & (l.page - 1));
        if (lane * 4 < slot_bytes)
            ((uint32_t*)(kv + t * slot_bytes))[lane] = ((const uint32_t*)(kv + f * slot_bytes))[lane];
        if (sc && lane < 4) sc[t * 4 + lane] = sc[f * 4 + lane];
    }
}

__global__ __launch_bounds__(256) void k_paged_advance(s2p_page_batch b, const int32_t* n_acc,
                                                       int32_t* len_out) {
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s >= b.sessions) return;
    const PgSess ss = pg_session(b, s);
    const int n = min(n_acc[s], ss.n - 1);
    len_out[s] = ss.n > 0 && n >= 0 ? ss.L + 1 + n : ss.L;
}

extern "C" hipError_t s2pk_paged_commit(const s2p_page_pool* pool, const s2p_page_batch* batch,
                                        const int32_t* path, const int32_t* n_acc,
                                        int32_t* len_out, hipStream_t st) {
    if (batch && batch->rows <= 0) return hipSuccess;
    if (!pg_pool_ok(pool) || !pg_batch_ok(pool, batch) || batch->max_rows > 64 || !path || !n_acc ||
        pool->layers > 65535)
        return hipErrorInvalidValue;
    const size_t slots = (size_t)pool->pages * 2 * pool->kv_heads * pool->page;
    const int sb = pg_slot_bytes(pool->bits);
    if (batch->max_rows > 2) { /* with two rows the only node is in its place */
        hipLaunchKernelGGL(k_paged_commit,
                           dim3((unsigned)batch->sessions, (unsigned)(2 * pool->kv_heads),
                                (unsigned)pool->layers),
                           dim3(64), 0, st, pg_layer(pool, 0), slots * sb, slots * 4, sb, *batch,
                           path, n_acc);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (!len_out) return hipSuccess;
    hipLaunchKernelGGL(k_paged_advance, dim3((unsigned)((batch->sessions + 255) / 256)), dim3(256),
                       0, st, *batch, n_acc, len_out);
    return hipGetLastError();
}

extern "C" size_t s2p_page_pool_bytes(const s2p_page_pool* p) {
    if (!p) return 0;
    return (size_t)p->layers * p->pages * 2 * p->kv_heads * p->page * pg_slot_bytes(p->bits);
}
extern "C" size_t s2p_page_pool_scale_bytes(const s2p_page_pool* p) {
    if (!p || p->bits == 16) return 0;
    return (size_t)p->layers * p->pages * 2 * p->kv_heads * p->page * 8;
}
