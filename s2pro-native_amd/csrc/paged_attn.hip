/* s2pro MI355X — attention over paged session caches.
 *
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(128) - m)
 *
 * over the slots j that the row sees, in one pass with the running maximum m.
 *
 * Up to 32 query vectors (rows x heads a kv head) a session, k_paged_dec: bound by the
 * K/V stream.  A block is a kv head's share of the rounds (four waves x a tile of 32
 * bf16 or 64 coded slots) of all sessions, each block the same number of rounds, so
 * ragged lengths need no bound on the host and no session waits for the longest:
 *   - S^T = K Q^T on the matrix cores, K straight from HBM into the operand; the lane
 *     that has a vector's scores has them for the slots whose V^T operand it needs next,
 *     so P goes from the softmax into O^T = V^T P^T without leaving its registers;
 *   - V goes from HBM to LDS without registers (global_load_lds) and is transposed by
 *     the reads (ds_read_tr of 16, 8 or 4 bits);
 *   - INT8 codes convert exactly to bf16, INT4 codes to 1.5 + c / 16; a group's K scale
 *     multiplies its 32-dim partial score in f32, its V scale p before p's rounding;
 *   - p is rounded to bf16 (2^-9 of it, as the output is), the sums stay in f32.
 * A session that several blocks worked on is merged from their partials by k_paged_merge. */
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "attn_dev.h"
#include "gemv_dev.h"
#include "paged_dev.h"

struct PgAttn {
    PgLayer l;
    s2p_page_batch b;
    const uint16_t* q;
    const uint64_t* vis;
    uint16_t* out;
    float* work;
    int qh, kvh, g;
    int nb; /* blocks a kv head that share the rounds */
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


#define PD_WAVES 4
#define PD_SCALE (0.08838834764831845f * 1.4426950408889634f) /* log2(e) / sqrt(128) */

typedef __attribute__((address_space(1))) void PgGlb;
typedef __attribute__((address_space(3))) void PgLds;

S2P_DEV void pd_swap32(uint32_t& a, uint32_t& b) { /* a's upper half wave <-> b's lower */
    auto s = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = s[0];
    b = s[1];
}
S2P_DEV float pd_half(uint32_t w, int hi) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w & 0xFFFFu));
}
/* transposing reads: in a 16-lane group lane 2 r + h gives the address of 8 bytes, row r,
 * columns 8 h .. + 7, and lane i gets column i of rows 0 .. 7 (4 bits: lane r gives row r's 16
 * columns, lane i gets column i of rows 0 .. 15, row 0 in the lowest nibble) */
S2P_DEV s2p_u32x2 pd_tr8(const LDS(unsigned char)* p) {
    typedef __attribute__((__vector_size__(2 * sizeof(int)))) int i2;
    return __builtin_bit_cast(s2p_u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((LDS(i2)*)p));
}
S2P_DEV s2p_u32x2 pd_tr4(const LDS(unsigned char)* p) {
    typedef __attribute__((__vector_size__(2 * sizeof(int)))) int i2;
    return __builtin_bit_cast(s2p_u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32((LDS(i2)*)p));
}
/* the loads of the tile before the last N have arrived */
template <int N>
S2P_DEV void pd_wait() {
    static_assert(N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
/* the slots of a tile that a row sees, as bits: `before` of them lie in the prefix (all seen),
 * then come the nodes of the row's word */
S2P_DEV uint64_t pd_mask(uint64_t word, int before) {
    if (before >= 64) return ~0ull;
    if (before > 0) return ~(~0ull << before) | (word << before);
    return before > -64 ? word >> -before : 0ull;
}
S2P_DEV uint64_t pd_ones(int n) { return n >= 64 ? ~0ull : ~(~0ull << n); }
/* the 16-slot groups of a tile that are there, as slots */
S2P_DEV uint64_t pd_groups(int bad) {
    uint64_t m = 0;
#pragma unroll
    for (int g = 0; g < 4; g++)
        if (!((bad >> g) & 1)) m |= 0xFFFFull << (16 * g);
    return m;
}
/* the waves' O in LDS: 16-byte pieces of a vector's row permuted (rows lie a bank apart) */
S2P_DEV int pd_oidx(int vec, int d) { return vec * PG_HD + ((((d >> 2) ^ vec) & 15) << 2) + (d & 64) + (d & 3); }

/* rounds of `rnd` slots of the sessions, summed up to each in s_pre; returns all.  Every thread
 * of the block (of 256 or more) calls it. */
S2P_DEV int pd_rounds(const PgAttn& a, int rnd, int* s_pre, int* s_w) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int E = S2P_PAGE_MAX_SESSIONS / 256; /* neighbouring sessions a thread */
    int v[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int s = tid * E + e;
        if (s < a.b.sessions) {
            const PgSess ss = pg_session(a.b, s);
            if (ss.n > 0) sum += (ss.L + ss.n + rnd - 1) / rnd;
        }
        v[e] = sum;
    }
    int up = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(up, o, 64);
        if (lane >= o) up += t;
    }
    if (lane == 63) s_w[wave] = up;
    __syncthreads();
    up -= sum;
    for (int w = 0; w < wave; w++) up += s_w[w];
#pragma unroll
    for (int e = 0; e < E; e++)
        if (tid < 256) s_pre[tid * E + e] = up + v[e];
    __syncthreads();
    return s_pre[a.b.sessions - 1];
}

/* A bf16 tile that not every row sees whole: V rows that are not there become zeros (what lies
 * behind a session may be NaN, and 0 x NaN is NaN), and a node's V row with a NaN or infinity
 * is added on its own to the vectors that see it, then zeroed for the matrix product. */
template <int MQT>
S2P_DEV void pd_tail(const PgSess& ss, LDS(unsigned char)* vb, int tb, int bad,
                     const uint64_t (&seen)[MQT], const float (&x)[MQT][2][4],
                     s2p_f32x4 (&o)[MQT][8]) {
    const int lane = threadIdx.x & 63, qq = lane >> 4, c = lane & 15;
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int t = 4 * i + qq, j = tb + t;
        LDS(s2p_u32x4)* const p = (LDS(s2p_u32x4)*)(vb + i * 1024 + lane * 16);
        bool nf = false;
        if (j >= ss.L + ss.n || ((bad >> (t >> 4)) & 1)) {
            *p = (s2p_u32x4){0u, 0u, 0u, 0u};
        } else if (j >= ss.L) {
            const s2p_u32x4 w = *p;
#pragma unroll
            for (int e = 0; e < 4; e++)
                nf |= (w[e] & 0x7F80u) == 0x7F80u || (w[e] & 0x7F800000u) == 0x7F800000u;
        }
        const uint64_t b = __ballot(nf);
#pragma unroll
        for (int r = 0; r < 4; r++)
            if ((b >> (16 * r)) & 0xFFFFu) odd |= 1u << (4 * i + r);
    }
    wave_lds_sync();
    while (odd) {
        const int t = __ffs(odd) - 1;
        odd &= odd - 1;
        s2p_u32x2 v[8];
#pragma unroll
        for (int dt = 0; dt < 8; dt++) {
            const int d = 16 * dt + 4 * qq;
            v[dt] = *(const LDS(s2p_u32x2)*)(vb + t * 256 + (((d >> 3) ^ ((t & 7) << 1)) << 4) +
                                             2 * (d & 7));
        }
#pragma unroll
        for (int qt = 0; qt < MQT; qt++) {
            float p = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) p = (t >> 4) == h && (t & 3) == e ? x[qt][h][e] : p;
            p = __shfl(p, ((t >> 2) & 3) * 16 + c, 64);
            if ((seen[qt] >> t) & 1) {
#pragma unroll
                for (int dt = 0; dt < 8; dt++) {
                    o[qt][dt][0] = fmaf(p, bf2f_lo(v[dt].x), o[qt][dt][0]);
                    o[qt][dt][1] = fmaf(p, bf2f_hi(v[dt].x), o[qt][dt][1]);
                    o[qt][dt][2] = fmaf(p, bf2f_lo(v[dt].y), o[qt][dt][2]);
                    o[qt][dt][3] = fmaf(p, bf2f_hi(v[dt].y), o[qt][dt][3]);
                }
            }
        }
        wave_lds_sync();
        if (lane < 16) *(LDS(s2p_u32x4)*)(vb + t * 256 + 16 * lane) = (s2p_u32x4){0u, 0u, 0u, 0u};
        wave_lds_sync();
    }
}

/* ------------------------------------------------------------ few rows a session */

/* tile and LDS of a wave: TS slots; V as it lies in the page, rows of EL bytes whose
 * 16-byte chunks are permuted so that the transposing reads spread over the banks */
template <int BW>
struct PdTile {
    static constexpr int TS = BW == 16 ? 32 : 64, NG = TS / 16;
    static constexpr int EL = BW == 16 ? 256 : BW == 8 ? 128 : 64;
    static constexpr int NP = TS / 16;                          /* MFMAs of 16 slots */
    static constexpr int NK = BW == 16 ? 4 : BW == 8 ? 2 : 1;   /* 16-byte K loads a 16 slots */
    static constexpr int NV = TS * EL / 1024;                   /* 1 KB V loads */
    static constexpr int VB = TS * EL + (BW == 16 ? 0 : 1024);  /* a buffer: V, then K and V scales */
    s2p_u32x4 k[NP][NK];
};

template <int BW>
S2P_DEV int pd_swz(int t) {
    if constexpr (BW == 16) return (t & 7) << 1;
    else if constexpr (BW == 8) return ((t >> 1) & 3) | (((t >> 4) & 1) << 2);
    else return (t >> 4) & 3;
}

template <int BW, int MQT>
__global__ __launch_bounds__(64 * PD_WAVES, 2) void k_paged_dec(PgAttn a) {
#pragma clang fp contract(off)
    typedef PdTile<BW> Tile;
    constexpr int TS = Tile::TS, NG = Tile::NG, NP = Tile::NP, EL = Tile::EL, VB = Tile::VB;
    constexpr int RND = TS * PD_WAVES;
    constexpr int OB = PD_WAVES * 16 * MQT * PG_HD * 4;
    constexpr int VBUF = PD_WAVES * 2 * VB;
    __shared__ __align__(16) unsigned char s_buf[VBUF > OB ? VBUF : OB];
    __shared__ float s_ml[PD_WAVES][16 * MQT][2];
    __shared__ int s_pre[S2P_PAGE_MAX_SESSIONS], s_w[PD_WAVES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qq = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x % a.kvh, blk = blockIdx.x / a.kvh;
    LDS(unsigned char)* const vbuf = (LDS(unsigned char)*)s_buf + wave * 2 * VB;

    /* the block's share of the rounds of all sessions */
    const int total = pd_rounds(a, RND, s_pre, s_w);
    const int nb = min(a.nb, total); /* every one of them has a round */
    if (blk >= nb) return;
    const int begin = (int)((int64_t)blk * total / nb);
    const int end = (int)((int64_t)(blk + 1) * total / nb);
    int vrow[MQT], vhead[MQT];
#pragma unroll
    for (int qt = 0; qt < MQT; qt++) {
        vrow[qt] = (16 * qt + c) / a.g;
        vhead[qt] = kvh * a.g + (16 * qt + c) % a.g;
    }

    for (int cur = begin; cur < end;) {
        /* the session of round cur: the first whose rounds reach past it */
        int s = 0, hi = a.b.sessions - 1;
        while (s < hi) {
            const int mid = (s + hi) >> 1;
            if (s_pre[mid] > cur) hi = mid;
            else s = mid + 1;
        }
        s = __builtin_amdgcn_readfirstlane(s);
        const int first = __builtin_amdgcn_readfirstlane(s ? s_pre[s - 1] : 0);
        const int last = __builtin_amdgcn_readfirstlane(s_pre[s]);
        const PgSess ss = pg_session(a.b, s);
        const int span = ss.L + ss.n;
        const int stop = min(end, last);
        const int p0 = (cur - first) * RND, p1 = min((stop - first) * RND, span);
        const int32_t* tab = a.b.table + (size_t)s * a.b.max_pages;

        s2p_u32x4 qb[MQT][4];
        uint64_t word[MQT];
#pragma unroll
        for (int qt = 0; qt < MQT; qt++) {
            const bool live = vrow[qt] < ss.n;
            const uint16_t* qr =
                a.q + ((size_t)(ss.r0 + (live ? vrow[qt] : 0)) * a.qh + vhead[qt]) * PG_HD;
            word[qt] = 0ull; /* the row's nodes; causal: those up to its own */
            if (live) word[qt] = (a.vis ? a.vis[ss.r0 + vrow[qt]] : pd_ones(vrow[qt] + 1)) & pd_ones(ss.n);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                /* the dims that the lane's K bytes of MFMA g hold; INT8: after the exchange of
                 * half waves quarters 0, 1 have the low 8 of 16-dim pieces 2 g, 2 g + 1 */
                const int d = BW == 8 ? 32 * g + 16 * (qq & 1) + 8 * (qq >> 1) : 32 * g + 8 * qq;
                s2p_u32x4 w = *(const s2p_u32x4*)(qr + d);
                if (BW == 4) w = int4_order(w); /* the k order of deq_int4 */
                qb[qt][g] = live ? w : (s2p_u32x4){0u, 0u, 0u, 0u};
            }
        }
        /* deq_int4 gives 1.5 + code / 16: a second product takes the 1.5 off (in registers of
         * their own its sums would cost 16 a vector tile) */
        const s2p_u32x4 k15 = {0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u};
        (void)k15;
        /* m (in units of log2), l (this lane's slots), o: O^T, dims 16 dt + 4 qq + v of
         * vector 16 qt + c */
        float m[MQT], l[MQT];
        bool any[MQT];
        s2p_f32x4 o[MQT][8];
#pragma unroll
        for (int qt = 0; qt < MQT; qt++) {
            m[qt] = -INFINITY;
            l[qt] = 0.f;
            any[qt] = false;
#pragma unroll
            for (int dt = 0; dt < 8; dt++) o[qt][dt] = (s2p_f32x4){0.f, 0.f, 0.f, 0.f};
        }

        const int tb0 = p0 + wave * TS;
        const int n = tb0 < p1 ? (p1 - tb0 + RND - 1) / RND : 0;
        int ids = 0; /* lane x: the page of the wave's 16-slot group x (of 64 / NG tiles), or -1 */
        auto page_ids = [&](int k) __attribute__((always_inline)) {
            const int slot = tb0 + (k + lane / NG) * RND + 16 * (lane % NG);
            int id = -1;
            if (slot < p1) {
                id = tab[slot >> a.l.shift];
                if ((unsigned)id >= (unsigned)a.l.pages) id = -1;
            }
            ids = id;
        };
        /* tile k: K to registers, V (and scales) to buffer k & 1.  A group that is not there
         * reads page 0 and is masked. */
        auto issue = [&](Tile& t, int k) __attribute__((always_inline)) {
            if ((k & (64 / NG - 1)) == 0) page_ids(k);
            int lane = threadIdx.x & 63; /* offsets made here, not kept through the loop */
            asm volatile("" : "+v"(lane));
            const int c = lane & 15, qq = lane >> 4;
            const int tb = tb0 + k * RND, x0 = (k & (64 / NG - 1)) * NG;
            LDS(unsigned char)* const vb = vbuf + (k & 1) * VB;
            uint64_t at[NG];
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const int id = max(__builtin_amdgcn_readlane(ids, x0 + g), 0);
                at[g] = (((uint64_t)(uint32_t)id * (uint32_t)a.l.planes + (uint32_t)kvh) << a.l.shift) +
                        (uint32_t)((tb + 16 * g) & (a.l.page - 1));
            }
            const uint64_t vplane = (uint64_t)(uint32_t)a.kvh << a.l.shift;
            if constexpr (BW != 16) {
                /* lanes 0..31: two slots' K scales each, 32..63: their V scales */
                const int g = (lane >> 3) & 3;
                const uint64_t sa = (g & 2 ? (g & 1 ? at[3] : at[2]) : (g & 1 ? at[1] : at[0])) +
                                    (lane & 32 ? vplane : 0);
                __builtin_amdgcn_global_load_lds(
                    (PgGlb*)((GblPtr)(uint64_t)a.l.sc + sa * 8 + 16 * (lane & 7)),
                    (PgLds*)(vb + TS * EL), 16, 0, 0);
            }
#pragma unroll
            for (int p = 0; p < NP; p++) {
                const GblPtr kb = gbl_base(a.l.kv, at[p] * EL);
#pragma unroll
                for (int i = 0; i < Tile::NK; i++)
                    t.k[p][i] = gbl_at<s2p_u32x4, true>(kb + 64 * i, (uint32_t)(c * EL + 16 * qq));
            }
#pragma unroll
            for (int i = 0; i < Tile::NV; i++) {
                const int g = i * (1024 / EL) / 16; /* the load's rows lie in one group */
                const int t0 = i * (1024 / EL) % 16, tl = lane / (EL / 16);
                const GblPtr vp = gbl_base(a.l.kv, (at[g] + vplane) * EL);
                const int ch = (lane % (EL / 16)) ^ pd_swz<BW>(i * (1024 / EL) + tl);
                __builtin_amdgcn_global_load_lds(
                    (PgGlb*)(vp + (uint32_t)((t0 + tl) * EL + 16 * ch)),
                    (PgLds*)(vb + i * 1024), 16, 0, 2 /* nontemporal */);
            }
        };
        constexpr int OPS = NP * Tile::NK + Tile::NV + (BW == 16 ? 0 : 1); /* loads of a tile */

        auto bad_of = [&](int k) __attribute__((always_inline)) {
            /* the tile's groups that are not there */
            const uint64_t b = __ballot(ids < 0);
            return (int)((b >> ((k & (64 / NG - 1)) * NG)) & ((1u << NG) - 1));
        };
        auto step = [&](Tile& t, int k, int bad) __attribute__((always_inline)) {
            int lane = threadIdx.x & 63;
            asm volatile("" : "+v"(lane));
            const int c = lane & 15, qq = lane >> 4;
            const int tb = tb0 + k * RND;
            const LDS(unsigned char)* vb = vbuf + (k & 1) * VB;
            if constexpr (BW != 16) pd_wait<Tile::NV>(); /* the scales, issued before K and V */
            /* scores of slots tb + 16 p + 4 qq + v, vector 16 qt + c */
            float x[MQT][NP][4];
#pragma unroll
            for (int p = 0; p < NP; p++) {
                if constexpr (BW == 16) {
#pragma unroll
                    for (int qt = 0; qt < MQT; qt++) {
                        s2p_f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int g = 0; g < 4; g++) sc = mfma16x16x32(t.k[p][g], qb[qt][g], sc);
#pragma unroll
                        for (int v = 0; v < 4; v++) x[qt][p][v] = sc[v];
                    }
                } else {
                    uint32_t kd[4][2];
                    if constexpr (BW == 8) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            uint32_t d0 = t.k[p][i].x, d1 = t.k[p][i].y, d2 = t.k[p][i].z,
                                     d3 = t.k[p][i].w;
                            pd_swap32(d0, d2);
                            pd_swap32(d1, d3);
                            kd[2 * i][0] = d0;
                            kd[2 * i][1] = d1;
                            kd[2 * i + 1][0] = d2;
                            kd[2 * i + 1][1] = d3;
                        }
                    } else {
                        uint32_t d0 = t.k[p][0].x, d1 = t.k[p][0].y, d2 = t.k[p][0].z,
                                 d3 = t.k[p][0].w;
                        xpose4(d0, d1, d2, d3);
                        kd[0][0] = d0;
                        kd[1][0] = d1;
                        kd[2][0] = d2;
                        kd[3][0] = d3;
                    }
                    uint32_t mask = 0x00780078u, one = 0x3F803F80u;
                    asm volatile("" : "+v"(mask), "+v"(one));
                    /* K scales of slots 16 p + 4 qq + 0 .. 3, four groups each */
                    const LDS(s2p_u32x4)* kp =
                        (const LDS(s2p_u32x4)*)(vb + TS * EL + 8 * (16 * p + 4 * qq));
                    const s2p_u32x4 ks[2] = {kp[0], kp[1]};
#pragma unroll
                    for (int qt = 0; qt < MQT; qt++)
#pragma unroll
                        for (int v = 0; v < 4; v++) x[qt][p][v] = 0.f;
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        s2p_u32x4 ka;
                        if constexpr (BW == 8) {
                            const s2p_u32x2 u = deq_s8(kd[g][0]), w = deq_s8(kd[g][1]);
                            ka = (s2p_u32x4){u.x, u.y, w.x, w.y};
                        } else {
                            ka = deq_int4(kd[g][0], mask, one);
                        }
#pragma unroll
                        for (int qt = 0; qt < MQT; qt++) {
                            s2p_f32x4 raw = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (BW == 4) raw = mfma16x16x32(k15, qb[qt][g], raw);
                            raw = mfma16x16x32(ka, qb[qt][g], raw);
#pragma unroll
                            for (int v = 0; v < 4; v++)
                                x[qt][p][v] = fmaf(pd_half(ks[v >> 1][2 * (v & 1) + (g >> 1)], g & 1),
                                                   raw[v], x[qt][p][v]);
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0); /* the next 16 slots' operands wait */
            }
            /* the next tile's loads fly from here to its scores; this tile's V is there when
             * no more than they are out */
            int next = 0;
            if (k + 1 < n) {
                issue(t, k + 1);
                next = bad_of(k + 1);
                pd_wait<OPS>();
            } else {
                pd_wait<0>();
            }
            /* online softmax; slots that are not seen weigh exp2(-inf) = 0 */
            const bool open = tb + TS <= ss.L && bad == 0;
            uint64_t seen[MQT];
#pragma unroll
            for (int qt = 0; qt < MQT; qt++) {
                float tm = -INFINITY;
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        x[qt][p][v] *= (BW == 4 ? 16.0f : 1.0f) * PD_SCALE;
                uint64_t see = ~0ull;
                if (!open) {
                    see = pd_mask(word[qt], ss.L - tb) & pd_groups(bad);
                    if (TS == 32) see &= 0xFFFFFFFFull;
                    seen[qt] = see;
                    const uint32_t w[2] = {(uint32_t)see >> (4 * qq), (uint32_t)(see >> 32) >> (4 * qq)};
#pragma unroll
                    for (int p = 0; p < NP; p++)
#pragma unroll
                        for (int v = 0; v < 4; v++)
                            if (!((w[p >> 1] >> (16 * (p & 1) + v)) & 1)) x[qt][p][v] = -INFINITY;
                }
                any[qt] |= see != 0;
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int v = 0; v < 4; v++) tm = fmaxf(tm, x[qt][p][v]);
                tm = xg_max(tm);
                const float mn = fmaxf(m[qt], tm);
                const float ms = mn == -INFINITY ? 0.f : mn;
                const float corr = __builtin_amdgcn_exp2f(m[qt] - ms);
                float ls = 0.f;
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const float e = __builtin_amdgcn_exp2f(x[qt][p][v] - ms);
                        ls += e;
                        x[qt][p][v] = e;
                    }
                l[qt] = fmaf(l[qt], corr, ls);
                m[qt] = mn;
                if (__any(corr != 1.0f)) {
#pragma unroll
                    for (int dt = 0; dt < 8; dt++) o[qt][dt] *= corr;
                }
            }
            if constexpr (BW == 16) {
                s2p_u32x4 pw[MQT];
                if (!open) pd_tail<MQT>(ss, (LDS(unsigned char)*)vb, tb, bad, seen, x, o);
#pragma unroll
                for (int qt = 0; qt < MQT; qt++)
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        pw[qt][2 * p] = pk_bf(x[qt][p][0], x[qt][p][1]);
                        pw[qt][2 * p + 1] = pk_bf(x[qt][p][2], x[qt][p][3]);
                    }
#pragma unroll
                for (int dt = 0; dt < 8; dt++) {
                    const int k4 = c >> 2, m4 = c & 3;
                    s2p_u32x2 b[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int r = 16 * h + 4 * qq + k4, d = 16 * dt + 4 * m4;
                        b[h] = ds_read_tr16((const LDS(uint16_t)*)(vb + r * 256 +
                                                                   (((d >> 3) ^ pd_swz<16>(r)) << 4) +
                                                                   2 * (d & 7)));
                    }
                    const s2p_u32x4 va = {b[0].x, b[0].y, b[1].x, b[1].y};
#pragma unroll
                    for (int qt = 0; qt < MQT; qt++)
                        o[qt][dt] = mfma16x16x32(va, pw[qt], o[qt][dt]);
                    if (dt & 1) __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                uint32_t mask = 0x00780078u, one = 0x3F803F80u;
                asm volatile("" : "+v"(mask), "+v"(one));
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    /* V scales of the lane's slots, groups g and g ^ 1 */
                    uint32_t vs[NP][4];
#pragma unroll
                    for (int p = 0; p < NP; p++)
#pragma unroll
                        for (int v = 0; v < 4; v++)
                            vs[p][v] = *(const LDS(uint32_t)*)(vb + TS * EL + 512 +
                                                               8 * (16 * p + 4 * qq + v) + 4 * (g >> 1));
                    /* the group's weights p vs, in bf16, halves h of 32 slots */
                    s2p_u32x4 w[MQT][2];
#pragma unroll
                    for (int qt = 0; qt < MQT; qt++) {
                        float y[NP][4];
#pragma unroll
                        for (int p = 0; p < NP; p++)
#pragma unroll
                            for (int v = 0; v < 4; v++)
                                y[p][v] = x[qt][p][v] * pd_half(vs[p][v], g & 1);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            __builtin_amdgcn_sched_barrier(0);
                            if constexpr (BW == 8)
                                w[qt][h] = (s2p_u32x4){pk_bf(y[2 * h][0], y[2 * h][1]),
                                                       pk_bf(y[2 * h][2], y[2 * h][3]),
                                                       pk_bf(y[2 * h + 1][0], y[2 * h + 1][1]),
                                                       pk_bf(y[2 * h + 1][2], y[2 * h + 1][3])};
                            else
                                w[qt][h] = (s2p_u32x4){pk_bf(y[2 * h][0], y[2 * h + 1][0]),
                                                       pk_bf(y[2 * h][1], y[2 * h + 1][1]),
                                                       pk_bf(y[2 * h][2], y[2 * h + 1][2]),
                                                       pk_bf(y[2 * h][3], y[2 * h + 1][3])};
                            if (!open) { /* a scale may be NaN where the slot is not seen */
#pragma unroll
                            for (int h = 0; h < 2; h++)
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    /* the word's two slots of the lane */
                                    const int s0 = BW == 8 ? 32 * h + 16 * (k >> 1) + 2 * (k & 1) : 32 * h + k;
                                    const int s1 = BW == 8 ? s0 + 1 : s0 + 16;
                                    const uint64_t z = seen[qt] >> (4 * qq);
                                    w[qt][h][k] &= ((z >> s0) & 1 ? 0xFFFFu : 0u) |
                                                   ((z >> s1) & 1 ? 0xFFFF0000u : 0u);
                                }
                        }
                    }
                    }
#pragma unroll
                    for (int d2 = 0; d2 < 2; d2++) {
                        const int dt = 2 * g + d2;
                        s2p_u32x4 va[2];
                        if constexpr (BW == 8) {
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const int r = c >> 1, t8 = 32 * h + 16 * (r >> 2) + 4 * qq + (r & 3);
                                const s2p_u32x2 d = pd_tr8(vb + t8 * 128 +
                                                           ((dt ^ pd_swz<8>(t8)) << 4) + 8 * (c & 1));
                                const s2p_u32x2 u = deq_s8(d.x), z = deq_s8(d.y);
                                va[h] = (s2p_u32x4){u.x, u.y, z.x, z.y};
                            }
                        } else {
                            const int t4 = 16 * (c >> 2) + 4 * qq + (c & 3);
                            const s2p_u32x2 d = pd_tr4(vb + t4 * 64 +
                                                       (((dt >> 1) ^ pd_swz<4>(t4)) << 4) + 8 * (dt & 1));
                            va[0] = deq_int4(d.x, mask, one);
                            va[1] = deq_int4(d.y, mask, one);
                        }
#pragma unroll
                        for (int qt = 0; qt < MQT; qt++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                if constexpr (BW == 4) o[qt][dt] = mfma16x16x32(k15, w[qt][h], o[qt][dt]);
                                o[qt][dt] = mfma16x16x32(va[h], w[qt][h], o[qt][dt]);
                            }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            return next;
        };
        Tile t;
        int bad = 0;
        if (n > 0) {
            issue(t, 0);
            bad = bad_of(0);
        }
        for (int k = 0; k < n; k++) bad = step(t, k, bad);
        /* the wave's state to LDS */
        __syncthreads(); /* the V buffers are free */
        LDS(float)* const so = (LDS(float)*)s_buf;
#pragma unroll
        for (int qt = 0; qt < MQT; qt++) {
            float lt = xg_sum(l[qt]);
            /* rows whose every score is -inf are told from rows that see nothing */
            if (m[qt] == -INFINITY && any[qt]) lt = 1.f;
            if (qq == 0) {
                s_ml[wave][16 * qt + c][0] = m[qt];
                s_ml[wave][16 * qt + c][1] = lt;
            }
#pragma unroll
            for (int dt = 0; dt < 8; dt++) {
                s2p_f32x4 z = o[qt][dt];
                if constexpr (BW == 4) z *= 16.0f;
                *(LDS(s2p_f32x4)*)(so + pd_oidx(wave * 16 * MQT + 16 * qt + c, 16 * dt + 4 * qq)) = z;
            }
        }
        __syncthreads();
        /* merge the waves: vector by vector, a dim a thread */
        const bool whole = cur == first && stop == last;
        const int nvec = min(16 * MQT, ss.n * a.g);
        float* const po = a.work + ((size_t)(kvh * a.nb + blk) * 2 + (cur == first ? 1 : 0)) *
                                       (16 * MQT * (PG_HD + 2));
        for (int i = tid; i < nvec * PG_HD; i += 64 * PD_WAVES) {
            const int vec = i >> 7, d = i & 127;
            float M = s_ml[0][vec][0];
#pragma unroll
            for (int w = 1; w < PD_WAVES; w++) M = fmaxf(M, s_ml[w][vec][0]);
            const float Ms = M == -INFINITY ? 0.f : M;
            float lt = 0.f, z = 0.f, mark = 0.f;
#pragma unroll
            for (int w = 0; w < PD_WAVES; w++) {
                const float e = __builtin_amdgcn_exp2f(s_ml[w][vec][0] - Ms);
                lt = fmaf(s_ml[w][vec][1], e, lt);
                mark = fmaxf(mark, s_ml[w][vec][1]);
                z = fmaf(so[pd_oidx(w * 16 * MQT + vec, d)], e, z);
            }
            if (whole) {
                a.out[((size_t)(ss.r0 + vec / a.g) * a.qh + kvh * a.g + vec % a.g) * PG_HD + d] =
                    f2bf(M == -INFINITY && mark == 0.f ? 0.f : z / lt);
            } else {
                po[16 * MQT * 2 + i] = z;
                if (d == 0) {
                    po[2 * vec] = M;
                    po[2 * vec + 1] = M == -INFINITY ? mark : lt;
                }
            }
        }
        cur = stop;
        if (cur < end) __syncthreads(); /* LDS is rewritten */
    }
}

/* Sessions that several blocks worked on: their partials, in the order of the blocks.
 * A block a (vector, kv head, session): four quarters of the blocks, a dim a thread. */
__global__ __launch_bounds__(512) void k_paged_merge(PgAttn a, int rnd, int nvec_max) {
    __shared__ int s_pre[S2P_PAGE_MAX_SESSIONS], s_w[8];
    __shared__ float s_m[4], s_l[4], s_k[4], s_z[4][PG_HD];
    const int vec = blockIdx.x, kvh = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, d = tid & 127, part = tid >> 7;
    const PgSess ss = pg_session(a.b, s);
    if (vec >= ss.n * a.g) return;
    const int total = pd_rounds(a, rnd, s_pre, s_w);
    const int first = s ? s_pre[s - 1] : 0, last = s_pre[s];
    /* block of a round: the last j whose first round, j total / nb, is not behind it */
    const int nb = min(a.nb, total);
    const int j0 = (int)((((int64_t)first + 1) * nb - 1) / total);
    const int j1 = (int)(((int64_t)last * nb - 1) / total);
    if (j0 == j1) return; /* one block had all of it */
    const size_t stride = (size_t)nvec_max * (PG_HD + 2);
    const float* const base = a.work + (size_t)kvh * a.nb * 2 * stride;
    const int each = (j1 - j0 + 4) >> 2;
    const int from = j0 + part * each, to = min(from + each, j1 + 1);
    float M = -INFINITY, lt = 0.f, z = 0.f, mark = 0.f;
    for (int j = from; j < to; j++) {
        const float* p = base + ((size_t)j * 2 + (j == j0 ? 1 : 0)) * stride;
        const float pm = p[2 * vec], pl = p[2 * vec + 1];
        const float pz = p[2 * nvec_max + vec * PG_HD + d];
        const float mn = fmaxf(M, pm), ms = mn == -INFINITY ? 0.f : mn;
        const float e0 = __builtin_amdgcn_exp2f(M - ms), e1 = __builtin_amdgcn_exp2f(pm - ms);
        mark = fmaxf(mark, pl);
        lt = fmaf(lt, e0, pl * e1);
        z = fmaf(z, e0, pz * e1);
        M = mn;
    }
    if (d == 0) {
        s_m[part] = M;
        s_l[part] = lt;
        s_k[part] = mark;
    }
    s_z[part][d] = z;
    __syncthreads();
    if (part) return;
    M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const float Ms = M == -INFINITY ? 0.f : M;
    lt = z = mark = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float e = __builtin_amdgcn_exp2f(s_m[i] - Ms);
        lt = fmaf(s_l[i], e, lt);
        z = fmaf(s_z[i][d], e, z);
        mark = fmaxf(mark, s_k[i]);
    }
    a.out[((size_t)(ss.r0 + vec / a.g) * a.qh + kvh * a.g + vec % a.g) * PG_HD + d] =
        f2bf(M == -INFINITY && mark == 0.f ? 0.f : z / lt);
}

/* blocks a kv head: two a CU fit, and no more than there are rounds of `rnd` slots */
static int64_t pd_blocks(const s2p_page_batch* b, int kv_heads, int rnd) {
    const int64_t most = (int64_t)b->sessions * ((b->max_len + rnd - 1) / rnd);
    int64_t nb = 2 * s2p_cu_count() / kv_heads;
    if (nb < 1) nb = 1;
    return nb < most ? nb : most;
}

template <int BW, int MQT>
static hipError_t pd_launch(PgAttn a, hipStream_t st) {
    const int rnd = PdTile<BW>::TS * PD_WAVES;
    a.nb = (int)pd_blocks(&a.b, a.kvh, rnd);
    hipLaunchKernelGGL((k_paged_dec<BW, MQT>), dim3((unsigned)(a.nb * a.kvh)), dim3(64 * PD_WAVES),
                       0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nb == 1 || a.b.max_len <= rnd) return e; /* no session is shared */
    hipLaunchKernelGGL(k_paged_merge, dim3((unsigned)(a.b.max_rows * a.g), (unsigned)a.kvh,
                                           (unsigned)a.b.sessions),
                       dim3(512), 0, st, a, rnd, 16 * MQT);
    return hipGetLastError();
}

extern "C" int64_t s2pk_paged_attention_work_floats(const s2p_page_batch* batch, int q_heads,
                                                    int kv_heads) {
    if (!batch || batch->sessions <= 0 || batch->rows <= 0 || kv_heads <= 0 ||
        !pg_group(q_heads, kv_heads))
        return 0;
    const int vecs = batch->max_rows * pg_group(q_heads, kv_heads);
    if (vecs > 32) return 4;
    return kv_heads * pd_blocks(batch, kv_heads, 128) * 2 * (vecs > 16 ? 32 : 16) * (PG_HD + 2) + 4;
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
    const int vecs = batch->max_rows * a.g;
    if (vecs <= 16)
        return pool->bits == 16 ? pd_launch<16, 1>(a, st)
               : pool->bits == 8 ? pd_launch<8, 1>(a, st) : pd_launch<4, 1>(a, st);
    if (vecs <= 32)
        return pool->bits == 16 ? pd_launch<16, 2>(a, st)
               : pool->bits == 8 ? pd_launch<8, 2>(a, st) : pd_launch<4, 2>(a, st);
    const dim3 grid((unsigned)batch->rows, (unsigned)q_heads);
    if (pool->bits == 16) hipLaunchKernelGGL(k_paged_attn<16>, grid, dim3(128), 0, st, a);
    else if (pool->bits == 8) hipLaunchKernelGGL(k_paged_attn<8>, grid, dim3(128), 0, st, a);
    else hipLaunchKernelGGL(k_paged_attn<4>, grid, dim3(128), 0, st, a);
    return hipGetLastError();
}
