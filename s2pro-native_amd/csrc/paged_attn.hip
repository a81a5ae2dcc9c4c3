/* s2pro MI355X — attention over paged session caches.
 *
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(128) - m)
 *
 * over the slots j that the row sees.  One workgroup of 128 threads a (row, query
 * head): tiles of 128 slots, a slot a thread for the scores and a dim a thread for
 * P V, f32 throughout, slots that are not seen never read into a sum. */
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "paged_dev.h"
#include "prims_dev.h"

struct PgAttn {
    PgLayer l;
    s2p_page_batch b;
    const uint16_t* q;
    const uint64_t* vis;
    uint16_t* out;
    float* work;
    int qh, kvh, g;
};

template <int BW>
S2P_DEV float pg_value(const char* row, const uint16_t* sc, int d) {
    if constexpr (BW == 16) return bf2f(((const uint16_t*)row)[d]);
    else if constexpr (BW == 8) return (float)((const int8_t*)row)[d] * h2f(sc[d >> 5]);
    else {
        const int n = (((const uint8_t*)row)[d >> 1] >> (4 * (d & 1))) & 0xF;
        return (float)(n >= 8 ? n - 16 : n) * h2f(sc[d >> 5]);
    }
}

template <int BW>
__global__ __launch_bounds__(128) void k_paged_attn(PgAttn a) {
    constexpr int EL = BW == 16 ? 256 : BW == 8 ? 128 : 64;
    __shared__ float s_q[128], s_p[128], s_red[2];
    __shared__ int64_t s_at[128];
    const int row = blockIdx.x, head = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int s = 0;
    for (int i = 0; i < a.b.sessions; i += 64)
        s += __popcll(__ballot(i + lane < a.b.sessions && a.b.row0[i + lane + 1] <= row));
    if (s >= a.b.sessions) return;
    const PgSess ss = pg_session(a.b, s);
    const int i = row - ss.r0;
    if (i < 0 || i >= ss.n) return;
    const int kvh = head / a.g;
    const uint64_t vis = a.vis ? a.vis[row] : 0ull;
    const int32_t* tab = a.b.table + (size_t)s * a.b.max_pages;
    s_q[t] = bf2f(a.q[((size_t)row * a.qh + head) * PG_HD + t]) * 0.08838834764831845f;
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc = 0.f;
    bool any = false;
    for (int t0 = 0; t0 < ss.L + ss.n; t0 += 128) {
        const int j = t0 + t, b = j - ss.L;
        bool seen = j < ss.L + ss.n && (b < 0 || (a.vis ? ((vis >> (b & 63)) & 1) : b <= i));
        int64_t at = -1;
        float x = -INFINITY;
        if (seen) {
            const int id = tab[j >> a.l.shift];
            if ((unsigned)id < (unsigned)a.l.pages) {
                at = (((int64_t)id * a.l.planes + kvh) << a.l.shift) + (j & (a.l.page - 1));
                const char* k = a.l.kv + at * EL;
                x = 0.f;
                for (int d = 0; d < 128; d++)
                    x = fmaf(s_q[d], pg_value<BW>(k, a.l.sc ? a.l.sc + at * 4 : nullptr, d), x);
            }
        }
        s_at[t] = at;
        float tm = wave_max(x);
        if (__syncthreads_or(x != x)) tm = NAN;
        if (lane == 0) s_red[wave] = tm;
        any |= __syncthreads_or(at >= 0) != 0;
        const float mn = fmaxf(m, fmaxf(s_red[0], s_red[1]));
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float corr = expf(m - ms);
        s_p[t] = at >= 0 ? expf(x - ms) : 0.f;
        __syncthreads();
        l *= corr;
        acc *= corr;
        for (int u = 0; u < 128; u++) {
            const int64_t v = s_at[u];
            if (v < 0) continue;
            const int64_t vat = v + ((int64_t)a.kvh << a.l.shift);
            l += s_p[u];
            acc = fmaf(s_p[u],
                       pg_value<BW>(a.l.kv + vat * EL, a.l.sc ? a.l.sc + vat * 4 : nullptr, t), acc);
        }
        m = mn;
        __syncthreads();
    }
    a.out[((size_t)row * a.qh + head) * PG_HD + t] = f2bf(any ? acc / l : 0.f);
}

extern "C" int64_t s2pk_paged_attention_work_floats(const s2p_page_batch* batch, int q_heads,
                                                    int kv_heads) {
    if (!batch || batch->sessions <= 0 || batch->rows <= 0 || kv_heads <= 0 ||
        !pg_group(q_heads, kv_heads))
        return 0;
    return 4;
}

extern "C" hipError_t s2pk_paged_attention(const s2p_page_pool* pool, const s2p_page_batch* batch,
                                           int layer, const s2p_bf16* q, int q_heads,
                                           const uint64_t* vis, s2p_bf16* out, float* work,
                                           hipStream_t st) {
    if (batch && batch->rows <= 0) return hipSuccess;
    if (!pg_pool_ok(pool) || !pg_batch_ok(pool, batch) || layer < 0 || layer >= pool->layers ||
        !pg_group(q_heads, pool->kv_heads) || !q || !out || !work ||
        (((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) || ((uintptr_t)vis & 7) ||
        (vis && batch->max_rows > 64))
        return hipErrorInvalidValue;
    PgAttn a = {};
    a.l = pg_layer(pool, layer);
    a.b = *batch;
    a.q = (const uint16_t*)q;
    a.vis = vis;
    a.out = (uint16_t*)out;
    a.work = work;
    a.qh = q_heads;
    a.kvh = pool->kv_heads;
    a.g = pg_group(q_heads, pool->kv_heads);
    const dim3 grid((unsigned)batch->rows, (unsigned)q_heads);
    if (pool->bits == 16) hipLaunchKernelGGL(k_paged_attn<16>, grid, dim3(128), 0, st, a);
    else if (pool->bits == 8) hipLaunchKernelGGL(k_paged_attn<8>, grid, dim3(128), 0, st, a);
    else hipLaunchKernelGGL(k_paged_attn<4>, grid, dim3(128), 0, st, a);
    return hipGetLastError();
}
