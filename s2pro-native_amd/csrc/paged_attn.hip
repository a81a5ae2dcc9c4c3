/* s2pro MI355X — attention over paged session caches.
 *
 *   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(q . k_j / sqrt(128) - m)
 *
 * over the slots j that the row sees, in one pass with the running maximum m.
 *
 * Up to 32 query vectors (rows x heads a kv head) a session, k_paged_dec: bound by the
 * K/V stream (over codes by their conversion).  A block is a kv head's share of the rounds (four waves x a tile of 32
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
 * A session that several blocks worked on is merged from their partials by k_paged_merge.
 *
 * More query vectors, k_paged_rows: bound by the matrix cores and the softmax between
 * their products.  A row tile is 256 vectors; a wave takes 32 of them through every
 * 64-slot tile of K and V, which the block shares in LDS (128, and two waves for 32
 * vectors, each with half of a tile's slots, when no session has more):
 *   - S^T = K Q^T and O^T = V^T P^T with 32 x 32 x 16 products, P in registers as above;
 *   - one tile is worked on, one lies converted in LDS, one is on its way in registers,
 *     so there is one barrier a tile;
 *   - O follows a new maximum only when p would pass 2^8 (f32 has the room; p's and the
 *     sums' relative precision do not depend on the maximum);
 *   - codes become value x scale in f16 (11 bits), and q, which a wave scales by a power
 *     of two, f16 without loss; p is f16 too, at 2^7 of itself (what is lost lies 2^-31
 *     under the largest);
 *   - the tiles of slots that all row tiles need are dealt out evenly over one round of
 *     blocks, a row tile that several worked on is merged by k_paged_rows_merge.
 *
 * MI355X, 32 heads on 8 kv heads, in a stream of calls: 16 sessions x 8,192 tokens, one row
 * each, bf16 87 us (6.2 TB/s); 32 over INT4 codes at 512 .. 4,096 tokens 30 us; one at 100
 * tokens 5.8 us in a graph; 2 x 2,048 rows, half of them behind 2,048 tokens, 220 us
 * (770 TFLOP/s; 190 with the softmax taken out); 4 x 17 rows at 8,192 tokens 41 us.  Over INT8 codes the prompt rows take 1.15 times as long
 * (1.5 with the codes exact and p times a group's scale as its weight), the trees 45 us. */
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
    int* sums; /* [sessions] rounds up to each (the merge's view of the schedule) */
    int qh, kvh, g;
    int rt; /* rows a tile of k_paged_rows */
    int nb, nvt; /* blocks a kv head that share the rounds, for each tile of query vectors */
};

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
/* two floats as a bf16 pair, one conversion for both */
S2P_DEV uint32_t pd_pk(float a, float b) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f2;
    typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 b2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
}
/* four INT4 codes a word to bf16 1.5 + c / 16: the code's bits into the mantissa, exponent and the
 * sign bit's flip in one constant */
S2P_DEV s2p_u32x4 pd_deq4(uint32_t d, uint32_t mask, uint32_t k) {
    return (s2p_u32x4){((d << 3) & mask) ^ k, ((d >> 1) & mask) ^ k, ((d >> 5) & mask) ^ k,
                       ((d >> 9) & mask) ^ k};
}
/* LDS reads of what global_load_lds wrote.  In C++ each would wait for every load in flight, the
 * next tile's too (the compiler does not tell the buffers apart), so they are written out, each
 * block with its own wait; what they read has arrived by pd_wait. */
S2P_DEV uint32_t pd_lds(const LDS(unsigned char)* p) { return (uint32_t)(uintptr_t)p; }
/* the transposing ones: in a 16-lane group lane 4 r + h gives the address of 8 bytes, row r,
 * columns 4 h .. + 3, and lane i gets column i of rows 0 .. 3 (16 bits); 8 bits: lane 2 r + h,
 * columns 8 h .. + 7, rows 0 .. 7; 4 bits: lane r, 16 columns, rows 0 .. 15, row 0 lowest */
template <int O>
S2P_DEV void pd_tr16(uint32_t a, uint32_t b, s2p_u32x2& x0, s2p_u32x2& x1, s2p_u32x2& y0,
                     s2p_u32x2& y1) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n"
        "ds_read_b64_tr_b16 %1, %4 offset:%6\n"
        "ds_read_b64_tr_b16 %2, %5\n"
        "ds_read_b64_tr_b16 %3, %5 offset:%6\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x0), "=&v"(x1), "=&v"(y0), "=&v"(y1) : "v"(a), "v"(b), "n"(O) : "memory");
}
S2P_DEV void pd_tr4(uint32_t a, s2p_u32x2& x, s2p_u32x2& y) {
    asm volatile(
        "ds_read_b64_tr_b4 %0, %2\n"
        "ds_read_b64_tr_b4 %1, %2 offset:8\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x), "=&v"(y) : "v"(a) : "memory");
}
/* 32 bytes: four slots' scales */
template <int O>
S2P_DEV void pd_scales4(uint32_t a, s2p_u32x4& x, s2p_u32x4& y) {
    asm volatile(
        "ds_read_b128 %0, %2 offset:%3\n"
        "ds_read_b128 %1, %2 offset:%4\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x), "=&v"(y) : "v"(a), "n"(O), "n"(O + 16) : "memory");
}
/* of slots 0 .. 3 and 16 .. 19 the scales of two groups (a dword): x[p][0, 1], x[p][2, 3] */
template <int G>
S2P_DEV void pd_scales8(uint32_t a, s2p_u32x2 (&x)[2][2]) {
    asm volatile(
        "ds_read2_b32 %0, %4 offset0:%5 offset1:%5+2\n"
        "ds_read2_b32 %1, %4 offset0:%5+4 offset1:%5+6\n"
        "ds_read2_b32 %2, %4 offset0:%5+32 offset1:%5+34\n"
        "ds_read2_b32 %3, %4 offset0:%5+36 offset1:%5+38\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1])
        : "v"(a), "n"(G) : "memory");
}
S2P_DEV void pd_tr8(uint32_t a, uint32_t b, s2p_u32x2& x, s2p_u32x2& y) {
    asm volatile(
        "ds_read_b64_tr_b8 %0, %2\n"
        "ds_read_b64_tr_b8 %1, %3\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x), "=&v"(y) : "v"(a), "v"(b) : "memory");
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

/* The batch as a block keeps it in LDS: a session's rounds summed up with those before it, its
 * first row, length and rows. */
struct PdBatch {
    int pre[S2P_PAGE_MAX_SESSIONS], r0[S2P_PAGE_MAX_SESSIONS], len[S2P_PAGE_MAX_SESSIONS];
    uint8_t n[S2P_PAGE_MAX_SESSIONS]; /* max_rows is at most 32 here */
    int w[PD_WAVES];
};
/* Fills it (256 threads); returns all rounds of `rnd` slots. */
S2P_DEV int pd_batch(const PgAttn& a, int rnd, PdBatch& b) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int before = 0;
    for (int base = 0; base < a.b.sessions; base += 64 * PD_WAVES) {
        const int s = base + tid;
        int v = 0;
        if (s < a.b.sessions) {
            const PgSess ss = pg_session(a.b, s);
            if (ss.n > 0) v = (ss.L + ss.n + rnd - 1) / rnd;
            b.r0[s] = ss.r0;
            b.len[s] = ss.L;
            b.n[s] = (uint8_t)ss.n;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(v, o, 64);
            if (lane >= o) v += t;
        }
        if (base) __syncthreads(); /* w is read no more */
        if (lane == 63) b.w[wave] = v;
        __syncthreads();
        int all = before;
#pragma unroll
        for (int w = 0; w < PD_WAVES; w++) {
            if (w < wave) v += b.w[w];
            all += b.w[w];
        }
        if (s < a.b.sessions) b.pre[s] = before + v;
        before = all;
    }
    __syncthreads();
    return before;
}

/* A bf16 tile that not every row sees whole: V rows of pages that are not there become zeros, and
 * a node's V row with a NaN or infinity is added on its own to the vectors that see it, then zeroed
 * for the matrix product. */
template <int MQT>
S2P_DEV void pd_tail(const PgSess& ss, LDS(unsigned char)* vb, int tb, int bad,
                     const uint64_t (&seen)[MQT], const float (&x)[MQT][2][4],
                     s2p_f32x4 (&o)[MQT][8]) {
    const int lane = threadIdx.x & 63, qq = lane >> 4, c = lane & 15;
    uint32_t nf = 0, odd = 0; /* nf: of this lane's 16 bytes of rows 4 i + qq */
#pragma unroll
    for (int i = 0; i < 8; i++) {
        LDS(s2p_u32x4)* const p = (LDS(s2p_u32x4)*)(vb + i * 1024 + lane * 16);
        if ((bad >> (i >> 2)) & 1) { /* uniform */
            *p = (s2p_u32x4){0u, 0u, 0u, 0u};
        } else if (tb + 4 * i + 3 >= ss.L) { /* behind the nodes lies the last one again */
            const s2p_u32x4 w = *p;
            bool x = false;
#pragma unroll
            for (int e = 0; e < 4; e++)
                x |= (w[e] & 0x7F80u) == 0x7F80u || (w[e] & 0x7F800000u) == 0x7F800000u;
            nf |= (uint32_t)(x && tb + 4 * i + qq >= ss.L) << i;
        }
    }
    if (__any(nf)) { /* rare */
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint64_t b = __ballot((nf >> i) & 1);
#pragma unroll
            for (int r = 0; r < 4; r++)
                if ((b >> (16 * r)) & 0xFFFFu) odd |= 1u << (4 * i + r);
        }
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
    static constexpr int TS = BW == 4 ? 64 : 32, NG = TS / 16;
    static constexpr int EL = BW == 16 ? 256 : BW == 8 ? 128 : 64;
    static constexpr int NP = TS / 16;                          /* MFMAs of 16 slots */
    static constexpr int NK = BW == 16 ? 4 : BW == 8 ? 2 : 1;   /* 16-byte K loads a 16 slots */
    static constexpr int NV = TS * EL / 1024;                   /* 1 KB V loads */
    static constexpr int VB = TS * EL + (BW == 16 ? 0 : 16 * TS);  /* a buffer: V, then K and V scales */
    s2p_u32x4 k[NP][NK];
};

template <int BW>
S2P_DEV unsigned pd_swz(unsigned t) {
    if constexpr (BW == 16) return (t & 7) << 1;
    else if constexpr (BW == 8) return ((t >> 1) & 3) | (((t >> 4) & 1) << 2);
    else return (t >> 4) & 3;
}

/* four dims of a session's query vector; a vector that saw no slot (no mark) gets zeros, one whose
 * every score is -inf NaN */
S2P_DEV void pd_out(const PgAttn& a, int r0, int kvh, int vec, int d, s2p_f32x4 z, float M, float lt,
                    float mark) {
    const float inv = M == -INFINITY ? (mark > 0.f ? NAN : 0.f) : 1.f / lt;
    *(s2p_u32x2*)(a.out + ((size_t)(r0 + vec / a.g) * a.qh + kvh * a.g + vec % a.g) * PG_HD + d) =
        (s2p_u32x2){pd_pk(z[0] * inv, z[1] * inv), pd_pk(z[2] * inv, z[3] * inv)};
}

template <int BW, int MQT>
__global__ __launch_bounds__(64 * PD_WAVES, BW == 8 && MQT == 1 ? 3 : 2) void k_paged_dec(PgAttn a) {
#pragma clang fp contract(off)
    typedef PdTile<BW> Tile;
    constexpr int TS = Tile::TS, NG = Tile::NG, NP = Tile::NP, EL = Tile::EL, VB = Tile::VB;
    constexpr int RND = TS * PD_WAVES;
    constexpr int OB = PD_WAVES * 16 * MQT * PG_HD * 4;
    constexpr int VBUF = PD_WAVES * 2 * VB;
    __shared__ __align__(256) unsigned char s_buf[VBUF > OB ? VBUF : OB];
    __shared__ float s_ml[PD_WAVES][16 * MQT][2];
    __shared__ PdBatch s_b;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int qq = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x % a.kvh, vt = blockIdx.x / a.kvh % a.nvt;
    const int blk = blockIdx.x / a.kvh / a.nvt, v0 = 16 * MQT * vt; /* vectors from v0 on */
    LDS(unsigned char)* const vbuf = (LDS(unsigned char)*)s_buf + wave * 2 * VB;

    /* the block's share of the rounds of all sessions */
    const int total = pd_batch(a, RND, s_b);
    if (blockIdx.x == 0) /* for the merge */
        for (int i = tid; i < a.b.sessions; i += 64 * PD_WAVES) a.sums[i] = s_b.pre[i];
    const int nb = min(a.nb, total); /* every one of them has a round */
    if (blk >= nb) return;
    const int begin = (int)((int64_t)blk * total / nb);
    const int end = (int)((int64_t)(blk + 1) * total / nb);
    int vrow[MQT], vhead[MQT];
#pragma unroll
    for (int qt = 0; qt < MQT; qt++) {
        vrow[qt] = (v0 + 16 * qt + c) / a.g;
        vhead[qt] = kvh * a.g + (v0 + 16 * qt + c) % a.g;
    }

    for (int cur = begin; cur < end;) {
        /* the session of round cur: the first whose rounds reach past it */
        int s = 0, hi = a.b.sessions - 1;
        while (s < hi) {
            const int mid = (s + hi) >> 1;
            if (s_b.pre[mid] > cur) hi = mid;
            else s = mid + 1;
        }
        s = __builtin_amdgcn_readfirstlane(s);
        const int first = __builtin_amdgcn_readfirstlane(s ? s_b.pre[s - 1] : 0);
        const int last = __builtin_amdgcn_readfirstlane(s_b.pre[s]);
        PgSess ss;
        ss.r0 = __builtin_amdgcn_readfirstlane(s_b.r0[s]);
        ss.n = __builtin_amdgcn_readfirstlane((int)s_b.n[s]);
        ss.L = __builtin_amdgcn_readfirstlane(s_b.len[s]);
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
        s2p_u32x4 k15 = {0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u};
        if (BW == 4) asm volatile("" : "+v"(k15)); /* kept, not made again for every product */
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

        const int nvec = min(16 * MQT, ss.n * a.g - v0); /* of this tile; may be none */
        const int tb0 = p0 + wave * TS;
        const int n = nvec > 0 && tb0 < p1 ? (p1 - tb0 + RND - 1) / RND : 0;
        int ids = 0; /* lane x: the page of the wave's 16-slot group x (of 64 / NG tiles), or -1 */
        auto page_ids = [&](int k) __attribute__((always_inline)) {
            const int slot = min(tb0 + (k + lane / NG) * RND + 16 * (lane % NG), p1 - 1);
            const int id = tab[slot >> a.l.shift];
            ids = (unsigned)id < (unsigned)a.l.pages ? id : -1;
        };
        /* tile k: K to registers, V (and scales) to buffer k & 1.  A page that is not there reads page
         * 0 and is masked; behind the last slot the last one is read again (what lies there may be
         * NaN, and 0 x NaN is NaN). */
        auto issue = [&](Tile& t, int k) __attribute__((always_inline)) {
            if ((k & (64 / NG - 1)) == 0) page_ids(k);
            unsigned lane = threadIdx.x & 63; /* offsets made here, not kept through the loop */
            asm volatile("" : "+v"(lane));
            const unsigned c = lane & 15, qq = lane >> 4;
            const int tb = tb0 + k * RND, x0 = (k & (64 / NG - 1)) * NG;
            LDS(unsigned char)* const vb = vbuf + (k & 1) * VB;
            uint64_t at[NG];
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const int id = max(__builtin_amdgcn_readlane(ids, x0 + g), 0);
                at[g] = (((uint64_t)(uint32_t)id * (uint32_t)a.l.planes + (uint32_t)kvh) << a.l.shift) +
                        (uint32_t)(min(tb + 16 * g, (p1 - 1) & ~15) & (a.l.page - 1));
            }
            const uint64_t vplane = (uint64_t)(uint32_t)a.kvh << a.l.shift;
            if constexpr (BW != 16) {
                /* two slots' scales a lane: K's in the first TS / 2 lanes, then V's */
                const int g = (lane >> 3) & (NG - 1);
                uint64_t sa = g & 1 ? at[1] : at[0];
                if (NG == 4) sa = g & 2 ? (g & 1 ? at[NG - 1] : at[NG - 2]) : sa;
                if (lane & (TS / 2)) sa += vplane;
                if (TS == 64 || lane < TS)
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
                const unsigned t0 = i * (1024 / EL) % 16, tl = lane / (EL / 16);
                const GblPtr vp = gbl_base(a.l.kv, (at[g] + vplane) * EL);
                const unsigned ch = (lane % (EL / 16)) ^ pd_swz<BW>(i * (1024 / EL) + tl);
                unsigned row = t0 + tl;
                if constexpr (BW == 16) row = tb + 16 * g + 16 <= p1 ? row : min(row, (unsigned)(p1 - 1) & 15u);
                __builtin_amdgcn_global_load_lds(
                    (PgGlb*)(vp + (uint32_t)(row * EL + 16 * ch)),
                    (PgLds*)(vb + i * 1024), 16, 0, 2 /* nontemporal */);
            }
        };
        constexpr int OPS = NP * Tile::NK + Tile::NV + (BW == 16 ? 0 : 1); /* loads of a tile */

        auto bad_of = [&](int k) __attribute__((always_inline)) {
            /* the tile's groups that are not there */
            const uint64_t b = __ballot(ids < 0);
            return (int)((b >> ((k & (64 / NG - 1)) * NG)) & ((1u << NG) - 1));
        };
        /* O^T += V^T P^T over codes: p times a group's V scale is the weight of its 32 dims */
        [[maybe_unused]] auto codes_pv = [&](const LDS(unsigned char)* vb, float (&x)[MQT][NP][4],
                                             const uint64_t (&seen)[MQT], auto open)
                                             __attribute__((always_inline)) {
            constexpr int NH = NP / 2; /* products of 32 slots */
            int lane = threadIdx.x & 63;
            asm volatile("" : "+v"(lane));
            const int c = lane & 15, qq = lane >> 4;
            uint32_t mask = 0x00780078u, one = 0x3FC03FC0u;
            asm volatile("" : "+v"(mask), "+v"(one));
            const uint32_t v0 = pd_lds(vb), s0 = v0 + TS * EL + 8 * TS + 32 * qq;
            /* the row that the lane's address of a transposing read stands for */
            const int r = BW == 8 ? 16 * (c >> 3) + 4 * qq + ((c >> 1) & 3)
                                  : 16 * (c >> 2) + 4 * qq + (c & 3);
            const uint32_t va0 = v0 + r * EL + (pd_swz<BW>(r) << 4) + (BW == 8 ? 8 * (c & 1) : 0);
            s2p_u32x2 vs[NH][2][2];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                /* V scales of the lane's slots, groups g and g ^ 1 */
                if (g == 0) {
                    pd_scales8<0>(s0, vs[0]);
                    if constexpr (NH > 1) pd_scales8<64>(s0, vs[NH - 1]);
                } else if (g == 2) {
                    pd_scales8<1>(s0, vs[0]);
                    if constexpr (NH > 1) pd_scales8<65>(s0, vs[NH - 1]);
                }
                s2p_u32x2 b[2]; /* V codes: dims 32 g + c, 32 g + 16 + c */
                if constexpr (BW == 8) pd_tr8(va0 ^ (g << 5), va0 ^ (g << 5) ^ 16, b[0], b[1]);
                else pd_tr4(va0 ^ (g << 4), b[0], b[1]);
                s2p_u32x4 w[MQT][NH]; /* the group's weights p vs in bf16 */
#pragma unroll
                for (int qt = 0; qt < MQT; qt++)
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        float y[2][4];
#pragma unroll
                        for (int p = 0; p < 2; p++)
#pragma unroll
                            for (int v = 0; v < 4; v++)
                                y[p][v] = fmaf(pd_half(vs[h][p][v >> 1][v & 1], g & 1),
                                               x[qt][2 * h + p][v], 0.f);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            /* word k: INT8 slots in order, INT4 the order of deq_int4 */
                            const int p0 = BW == 8 ? k >> 1 : 0, e0 = BW == 8 ? 2 * (k & 1) : k;
                            const int p1 = BW == 8 ? p0 : 1, e1 = BW == 8 ? e0 + 1 : k;
                            w[qt][h][k] = pd_pk(y[p0][e0], y[p1][e1]);
                            if constexpr (!decltype(open)::value) {
                                /* a scale may be NaN where the slot is not seen */
                                const uint64_t z = seen[qt] >> (4 * qq + 32 * h);
                                w[qt][h][k] &= ((z >> (16 * p0 + e0)) & 1 ? 0xFFFFu : 0u) |
                                               ((z >> (16 * p1 + e1)) & 1 ? 0xFFFF0000u : 0u);
                            }
                        }
                    }
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    s2p_u32x4 va[NH];
                    if constexpr (BW == 8) {
                        const s2p_u32x2 u = deq_s8(b[d].x), z = deq_s8(b[d].y);
                        va[0] = (s2p_u32x4){u.x, u.y, z.x, z.y};
                    } else {
                        va[0] = pd_deq4(b[d].x, mask, one);
                        va[NH - 1] = pd_deq4(b[d].y, mask, one);
                    }
#pragma unroll
                    for (int qt = 0; qt < MQT; qt++)
#pragma unroll
                        for (int h = 0; h < NH; h++) {
                            if constexpr (BW == 4)
                                o[qt][2 * g + d] = mfma16x16x32(k15, w[qt][h], o[qt][2 * g + d]);
                            o[qt][2 * g + d] = mfma16x16x32(va[h], w[qt][h], o[qt][2 * g + d]);
                        }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto step = [&](Tile& t, int k, int bad) __attribute__((always_inline)) {
            int lane = threadIdx.x & 63;
            asm volatile("" : "+v"(lane));
            const int c = lane & 15, qq = lane >> 4;
            const int tb = tb0 + k * RND;
            const LDS(unsigned char)* vb = vbuf + (k & 1) * VB;
            if constexpr (BW != 16) pd_wait<Tile::NV>(); /* K and the scales, issued before V */
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
                    uint32_t mask = 0x00780078u, one = 0x3FC03FC0u;
                    asm volatile("" : "+v"(mask), "+v"(one));
                    /* K scales of slots 16 p + 4 qq + 0 .. 3, four groups each */
                    s2p_u32x4 ks[2];
                    const uint32_t sa = pd_lds(vb) + TS * EL + 32 * qq;
                    if (p == 0) pd_scales4<0>(sa, ks[0], ks[1]);
                    else if (p == 1) pd_scales4<128>(sa, ks[0], ks[1]);
                    else if (p == 2) pd_scales4<256>(sa, ks[0], ks[1]);
                    else pd_scales4<384>(sa, ks[0], ks[1]);
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
                            ka = pd_deq4(kd[g][0], mask, one);
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
                uint64_t see = ~0ull;
                if (!open) {
                    see = pd_mask(word[qt], ss.L - tb) & pd_groups(bad);
                    if (TS == 32) see &= 0xFFFFFFFFull; /* what lies behind the tile */
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
                constexpr float SC = (BW == 4 ? 16.0f : 1.0f) * PD_SCALE;
                tm = xg_max(tm) * SC;
                const float mn = fmaxf(m[qt], tm);
                const float ms = mn == -INFINITY ? 0.f : mn;
                const float corr = __builtin_amdgcn_exp2f(m[qt] - ms);
                float ls = 0.f;
#pragma unroll
                for (int p = 0; p < NP; p++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(x[qt][p][v], SC, -ms));
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
                if ((ss.n > 1 || a.vis || bad) && !open)
                    pd_tail<MQT>(ss, (LDS(unsigned char)*)vb, tb, bad, seen, x, o);
#pragma unroll
                for (int qt = 0; qt < MQT; qt++)
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        pw[qt][2 * p] = pd_pk(x[qt][p][0], x[qt][p][1]);
                        pw[qt][2 * p + 1] = pd_pk(x[qt][p][2], x[qt][p][3]);
                    }
                /* rows 4 qq + c / 4 (and + 16), dims 16 dt + 4 (c % 4) */
                const int r = 4 * qq + (c >> 2);
                const uint32_t va0 = pd_lds(vb) + r * 256 + ((((c >> 1) & 1) ^ pd_swz<16>(r)) << 4) +
                                     8 * (c & 1);
#pragma unroll
                for (int d2 = 0; d2 < 4; d2++) {
                    s2p_u32x2 b[4];
                    pd_tr16<4096>(va0 ^ (d2 << 6), va0 ^ (d2 << 6) ^ 32, b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const s2p_u32x4 va = {b[2 * e].x, b[2 * e].y, b[2 * e + 1].x, b[2 * e + 1].y};
#pragma unroll
                        for (int qt = 0; qt < MQT; qt++)
                            o[qt][2 * d2 + e] = mfma16x16x32(va, pw[qt], o[qt][2 * d2 + e]);
                    }
                }
            } else {
                if (open) codes_pv(vb, x, seen, std::true_type());
                else codes_pv(vb, x, seen, std::false_type());
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
        /* merge the waves, four dims of a vector a thread */
        const bool whole = cur == first && stop == last;
        float* const po = a.work + (((size_t)(kvh * a.nb + blk) * 2 + (cur == first ? 1 : 0)) * a.nvt + vt) *
                                       (16 * MQT * (PG_HD + 2));
        for (int i = tid; i < nvec * (PG_HD / 4); i += 64 * PD_WAVES) {
            const int vec = i >> 5, d = 4 * (i & 31);
            float pm[PD_WAVES], pl[PD_WAVES], M = -INFINITY;
            s2p_f32x4 pz[PD_WAVES];
#pragma unroll
            for (int w = 0; w < PD_WAVES; w++) {
                pm[w] = s_ml[w][vec][0];
                pl[w] = s_ml[w][vec][1];
                pz[w] = *(const LDS(s2p_f32x4)*)(so + pd_oidx(w * 16 * MQT + vec, d));
            }
#pragma unroll
            for (int w = 0; w < PD_WAVES; w++) M = fmaxf(M, pm[w]);
            const float Ms = M == -INFINITY ? 0.f : M;
            float lt = 0.f, mark = 0.f;
            s2p_f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < PD_WAVES; w++) {
                const float e = __builtin_amdgcn_exp2f(pm[w] - Ms);
                lt = fmaf(pl[w], e, lt);
                mark = fmaxf(mark, pl[w]);
#pragma unroll
                for (int v = 0; v < 4; v++) z[v] = fmaf(pz[w][v], e, z[v]);
            }
            if (whole) {
                pd_out(a, ss.r0, kvh, v0 + vec, d, z, M, lt, mark);
            } else {
                *(s2p_f32x4*)(po + 16 * MQT * 2 + 4 * i) = z;
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

/* partials joined: running maximum, sum, mark (> 0: a slot was seen) and four dims of O */
struct PgSum {
    float M = -INFINITY, lt = 0.f, mark = 0.f;
    s2p_f32x4 z = {0.f, 0.f, 0.f, 0.f};
};
S2P_DEV void pd_add(PgSum& o, float m, float l, s2p_f32x4 z, float mark) {
    const float mn = fmaxf(o.M, m), ms = mn == -INFINITY ? 0.f : mn;
    const float e0 = __builtin_amdgcn_exp2f(o.M - ms), e1 = __builtin_amdgcn_exp2f(m - ms);
    o.mark = fmaxf(o.mark, mark);
    o.lt = fmaf(o.lt, e0, l * e1);
#pragma unroll
    for (int e = 0; e < 4; e++) o.z[e] = fmaf(o.z[e], e0, z[e] * e1);
    o.M = mn;
}
/* Partial j of a run j0 .. j1 that blocks of a kv head left lies at (2 j + (j == j0)) strides from
 * `base`: vec's (m, l) at 2 vec, its O at 2 tile + 128 vec.  PARTS threads of 32 apart share the run
 * (part j - j0 mod PARTS), four dims each. */
template <int PARTS>
S2P_DEV PgSum pd_gather(const float* base, size_t stride, int tile, int j0, int j1, int vec, int part,
                        int d) {
    PgSum o;
    for (int jj = j0 + part; jj <= j1; jj += 4 * PARTS) { /* four partials' loads at a time */
        float pm[4], pl[4];
        s2p_f32x4 pz[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int j = min(jj + u * PARTS, j1);
            const float* p = base + ((size_t)j * 2 + (j == j0 ? 1 : 0)) * stride;
            pm[u] = p[2 * vec];
            pl[u] = p[2 * vec + 1];
            pz[u] = *(const s2p_f32x4*)(p + 2 * tile + vec * PG_HD + d);
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (jj + u * PARTS <= j1) pd_add(o, pm[u], pl[u], pz[u], pl[u]);
    }
    return o;
}

/* Sessions that several blocks worked on: their partials.  A block: 8 / PM_PARTS vectors of a kv
 * head and session, PM_PARTS threads of 32 apart share a vector's partials. */
#define PM_PARTS 4
#define PM_VECS (8 / PM_PARTS)
__global__ __launch_bounds__(256) void k_paged_merge(PgAttn a, int tile) {
    __shared__ float s_m[PM_VECS][PM_PARTS][3];
    __shared__ s2p_f32x4 s_z[PM_VECS][PM_PARTS][32];
    const int kvh = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, x = tid & 31, part = (tid >> 5) % PM_PARTS, u = (tid >> 5) / PM_PARTS;
    const int vec = blockIdx.x * PM_VECS + u;
    const int total = a.sums[a.b.sessions - 1], last = a.sums[s], first = s ? a.sums[s - 1] : 0;
    const PgSess ss = pg_session(a.b, s);
    if ((int)blockIdx.x * PM_VECS >= ss.n * a.g) return;
    /* block of a round: the last j whose first round, j total / nb, is not behind it */
    const int nb = min(a.nb, total);
    const int j0 = (int)((((int64_t)first + 1) * nb - 1) / total);
    const int j1 = (int)(((int64_t)last * nb - 1) / total);
    if (j0 == j1) return; /* one block had all of it */
    const bool live = vec < ss.n * a.g;
    const size_t stride = (size_t)tile * (PG_HD + 2); /* of a tile's partial */
    PgSum o;
    if (live)
        o = pd_gather<PM_PARTS>(a.work + ((size_t)kvh * a.nb * 2 * a.nvt + vec / tile) * stride,
                                a.nvt * stride, tile, j0, j1, vec % tile, part, 4 * x);
    if (x == 0) {
        s_m[u][part][0] = o.M;
        s_m[u][part][1] = o.lt;
        s_m[u][part][2] = o.mark;
    }
    s_z[u][part][x] = o.z;
    __syncthreads();
    if (part || !live) return;
#pragma unroll
    for (int i = 1; i < PM_PARTS; i++)
        pd_add(o, s_m[u][i][0], s_m[u][i][1], s_z[u][i][x], s_m[u][i][2]);
    pd_out(a, ss.r0, kvh, vec, 4 * x, o.z, o.M, o.lt, o.mark);
}

/* ------------------------------------------------------------ many rows a session */

#define PR_W 8                 /* waves of a block */
#define PR_TS 64               /* slots of a tile */
/* A row tile's start (q, the first loads with nothing to hide them) and end, in rounds of the
 * schedule: without them 2,048 rows of one session from position 0 take 108 us, with three 82;
 * 2 x 2,048 behind 2,048 tokens, whose tiles are long, 257 and 259. */
#define PR_BEGIN 3
#define PR_LAZY 8.0f           /* the running maximum follows when p would pass 2^8 */

typedef __attribute__((ext_vector_type(16))) float pr_f32x16;
S2P_DEV pr_f32x16 mfma32x32x16(s2p_u32x4 a, s2p_u32x4 b, pr_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
S2P_DEV pr_f32x16 mfma32x32x16_f16(s2p_u32x4 a, s2p_u32x4 b, pr_f32x16 c) {
    typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
S2P_DEV uint32_t pr_pk_f16(float a, float b) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f2;
    typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 h2;
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, h2));
}
/* a K row's 16-byte chunks permuted, and a V row's (for the transposing reads), in elements */
S2P_DEV int pr_koff(int t, int ch) { return t * PG_HD + ((ch ^ (t & 15)) << 3); }
S2P_DEV int pr_voff(int t, int ch) { return t * PG_HD + ((ch ^ ((t & 7) << 1)) << 3); }
S2P_DEV float pr_swap_max(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
S2P_DEV float pr_swap_sum(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
S2P_DEV bool pr_odd(s2p_u32x4 w) { /* eight bf16, one of them NaN or infinite */
    bool o = false;
#pragma unroll
    for (int e = 0; e < 4; e++)
        o |= (w[e] & 0x7F80u) == 0x7F80u || (w[e] & 0x7F800000u) == 0x7F800000u;
    return o;
}
/* rounds that row tile r of a session costs: its tiles of slots, and PR_BEGIN before them */
S2P_DEV int pr_rounds(const PgAttn& a, const PgSess& s, int r) {
    const int span = s.L + (a.vis ? s.n : min(s.n, (r + 1) * a.rt));
    return PR_BEGIN + (span + PR_TS - 1) / PR_TS;
}
/* a code pair's element of a word: INT8 word q / 2 of the chunk, INT4 the chunk's one word */
template <int BW>
S2P_DEV float pr_code(uint32_t w, int q, int e) {
    if constexpr (BW == 8) return (float)(int8_t)(w >> (8 * (2 * (q & 1) + e)));
    else return (float)((int32_t)(w << (28 - 4 * (2 * q + e))) >> 28);
}

/* what a thread brings of a tile's K or V: 16-byte pieces and their scales */
template <int BW>
struct PrStage {
    static constexpr int EL = BW == 16 ? 256 : BW == 8 ? 128 : 64;
    static constexpr int NP = PR_TS * EL / 16;                       /* pieces of a tile's K or V */
    static constexpr int NL = (NP + 64 * PR_W - 1) / (64 * PR_W);
    s2p_u32x4 w[NL];
    uint16_t s[NL];
};

template <int BW, int SP>
__global__ __launch_bounds__(64 * PR_W, 2) void k_paged_rows(PgAttn a) {
#pragma clang fp contract(off)
    typedef PrStage<BW> Stage;
    /* codes: p goes in f16, from 2^15 down to 2^-24 */
    constexpr float SHIFT = BW == 16 ? 0.f : 7.f;
    constexpr int VEC = 32 * PR_W / SP; /* query vectors of a row tile */
    constexpr int EL = Stage::EL, NL = Stage::NL, CR = EL / 16; /* pieces of a row */
    constexpr int NC = BW == 16 ? 1 : BW == 8 ? 2 : 4;         /* 8-dim chunks of a piece */
    __shared__ __align__(256) uint16_t s_k[2][PR_TS * PG_HD], s_v[2][PR_TS * PG_HD];
    __shared__ float s_ml[SP == 2 ? VEC : 1][2];
    __shared__ int s_pre[S2P_PAGE_MAX_SESSIONS], s_w[PR_W];
    /* of a tile: nodes whose V holds a NaN or infinity; codes: a scale over 512 */
    __shared__ unsigned long long s_odd[3];
    __shared__ int s_big[3];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, col = lane & 31;
    const int kvh = blockIdx.x % a.kvh, blk = blockIdx.x / a.kvh;

    /* the block's share of the rounds of all row tiles */
    int total = 0;
    for (int base = 0; base < a.b.sessions; base += 64 * PR_W) {
        int v = 0;
        if (base + tid < a.b.sessions) {
            const PgSess ss = pg_session(a.b, base + tid);
            for (int r = 0; r * a.rt < ss.n; r++) v += pr_rounds(a, ss, r);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(v, o, 64);
            if (lane >= o) v += t;
        }
        if (base) __syncthreads();
        if (lane == 63) s_w[wave] = v;
        __syncthreads();
        int all = total;
#pragma unroll
        for (int w = 0; w < PR_W; w++) {
            if (w < wave) v += s_w[w];
            all += s_w[w];
        }
        if (base + tid < a.b.sessions) s_pre[base + tid] = total + v;
        total = all;
    }
    if (tid < 3) s_odd[tid] = s_big[tid] = 0;
    __syncthreads();
    const int nb = min(a.nb, total);
    if (blk >= nb) {
        if (kvh == 0 && blk < a.nb && tid == 0) a.sums[4 * blk + 1] = 0;
        return;
    }
    const int begin = (int)((int64_t)blk * total / nb);
    const int end = (int)((int64_t)(blk + 1) * total / nb);

    /* SP = 2: two waves have the same vectors, each half of a tile's slots */
    const int vw = wave / SP, part = wave % SP;
    const int vec = 32 * vw + col; /* this lane's query vector of a row tile */
    const int vi = vec / a.g, vhead = kvh * a.g + vec % a.g;
    int nvec_out = 0; /* of the row tile that the block leaves to another one */
    int seq = 0;      /* tiles so far, mod 3 */

    for (int cur = begin; cur < end;) {
        int s = 0, hi = a.b.sessions - 1;
        while (s < hi) {
            const int mid = (s + hi) >> 1;
            if (s_pre[mid] > cur) hi = mid;
            else s = mid + 1;
        }
        s = __builtin_amdgcn_readfirstlane(s);
        const PgSess ss = pg_session(a.b, s);
        int first = __builtin_amdgcn_readfirstlane(s ? s_pre[s - 1] : 0), r = 0, cnt;
        while (first + (cnt = pr_rounds(a, ss, r)) <= cur) { /* ends: the session reaches past cur */
            first += cnt;
            r++;
        }
        const int last = first + cnt, stop = min(end, last);
        const int k0 = max(0, cur - first - PR_BEGIN), k1 = stop - first - PR_BEGIN;
        cur = stop;
        if (k1 <= 0) break; /* the block ends in the tile's first rounds: the next one begins it */
        const int i0 = r * a.rt, rows = min(a.rt, ss.n - i0); /* the tile's rows */
        const int span = ss.L + (a.vis ? ss.n : i0 + rows);   /* slots that one of them may see */
        const int32_t* tab = a.b.table + (size_t)s * a.b.max_pages;
        const int nvec = rows * a.g;
        const bool live = vec < nvec;
        const bool busy = 32 * vw < nvec; /* the wave has a vector */
        const int row = ss.r0 + i0 + (live ? vi : 0);
        /* the row's nodes as a word, or (causal) how many slots it sees */
        const uint64_t word = a.vis && live ? a.vis[row] & pd_ones(ss.n) : 0ull;
        const int sees = live ? ss.L + i0 + vi + 1 : 0;
        /* no row of the wave sees a slot from here on; every one sees those before `open` */
        const int wend = a.vis ? span : min(span, ss.L + i0 + (min(32 * vw + 31, nvec - 1) / a.g) + 1);
        const int open_end = a.vis ? ss.L : ss.L + i0 + 32 * vw / a.g + 1;

        s2p_u32x4 qb[8];
        float scale = PD_SCALE;
        {
            const uint16_t* qr = a.q + ((size_t)row * a.qh + (live ? vhead : 0)) * PG_HD + 8 * half;
#pragma unroll
            for (int ks = 0; ks < 8; ks++)
                qb[ks] = live ? *(const s2p_u32x4*)(qr + 16 * ks) : (s2p_u32x4){0u, 0u, 0u, 0u};
            if constexpr (BW != 16) {
                /* q in f16 as a multiple of a power of two (which goes into the scale): its largest
                 * value at 2^14, all of its 8 bits down to 2^-28 of that */
                uint32_t top = 0;
#pragma unroll
                for (int ks = 0; ks < 8; ks++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        top = max(top, max(qb[ks][e] & 0x7FFFu, (qb[ks][e] >> 16) & 0x7FFFu));
                top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
                const int up = min(max((int)(top >> 7) - (127 + 14), -112), 112);
                const float down = __uint_as_float((uint32_t)(127 - up) << 23);
                scale *= __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
                for (int ks = 0; ks < 8; ks++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        qb[ks][e] = pr_pk_f16(bf2f_lo(qb[ks][e]) * down, bf2f_hi(qb[ks][e]) * down);
            }
        }
        float m = -INFINITY, l = 0.f;
        bool any = false;
        pr_f32x16 o[4];
#pragma unroll
        for (int dt = 0; dt < 4; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[dt][i] = 0.f;

        int ids = 0; /* of 16 tiles, 64 groups of 16 slots: lane x has group x's page, or -1 */
        auto page_ids = [&](int k) __attribute__((always_inline)) {
            if (((k - k0) & 15) == 0) {
                const int slot = (k + (lane >> 2)) * PR_TS + 16 * (lane & 3);
                int id = -1;
                if (slot < span && k + (lane >> 2) < k1) {
                    id = tab[slot >> a.l.shift];
                    if ((unsigned)id >= (unsigned)a.l.pages) id = -1;
                }
                ids = id;
            }
        };
        /* tile k's K (is_v: V) into registers */
        auto issue = [&](Stage& t, int k, bool is_v) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int i = tid + 64 * PR_W * j, trow = i / CR, ch = i % CR;
                if (Stage::NP % (64 * PR_W) && i >= Stage::NP) break; /* whole waves */
                const int g = __builtin_amdgcn_readfirstlane(trow >> 4); /* one group a wave */
                const int id = max(__builtin_amdgcn_readlane(ids, ((k - k0) & 15) * 4 + g), 0);
                const uint64_t at = (((uint64_t)(uint32_t)id * (uint32_t)a.l.planes +
                                      (uint32_t)(is_v ? a.kvh + kvh : kvh)) << a.l.shift) +
                                    (uint32_t)((k * PR_TS + 16 * g) & (a.l.page - 1));
                t.w[j] = gbl_at<s2p_u32x4>(gbl_base(a.l.kv, at * EL), (uint32_t)((trow & 15) * EL + 16 * ch));
                if constexpr (BW != 16)
                    t.s[j] = gbl_at<uint16_t>(gbl_base(a.l.sc, at * 8),
                                              (uint32_t)((trow & 15) * 8 + 2 * (BW == 8 ? ch >> 1 : ch)));
            }
        };
        /* groups of tile k that are not there (of the ids at hand) */
        auto bad_of = [&](int k) __attribute__((always_inline)) {
            return (int)((__ballot(ids < 0) >> (((k - k0) & 15) * 4)) & 15);
        };
        /* Tile k to LDS.  Codes: value x scale in f16 (2^-12 off; a tile with a scale over 512 is
         * marked and brought again as 2^-7 of itself, which stays in range).  V rows that are not
         * there become zeros (what lies there may be NaN, and 0 x NaN is NaN), and so do pieces of a
         * node's V with a NaN or infinity, which the rows that see the node add by themselves. */
        auto put = [&](s2p_u32x4 w16, float sc, LDS(uint16_t)* to, int trow, int ch, bool is_v)
                       __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < NC; e++) {
                s2p_u32x4 w = w16;
                if constexpr (BW != 16) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const uint32_t x = BW == 8 ? w16[2 * e + (q >> 1)] : w16[e];
                        w[q] = pr_pk_f16(pr_code<BW>(x, q, 0) * sc, pr_code<BW>(x, q, 1) * sc);
                    }
                }
                *(LDS(s2p_u32x4)*)(to + (is_v ? pr_voff(trow, NC * ch + e) : pr_koff(trow, NC * ch + e))) = w;
            }
        };
        auto big = [&](uint16_t sc) { return sc > 0x6000u && sc < 0x7C00u; }; /* 512 < sc < inf */
        auto store_k = [&](Stage& t, int k, int buf, int bad, int slot3) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int i = tid + 64 * PR_W * j, trow = i / CR, ch = i % CR;
                if (Stage::NP % (64 * PR_W) && i >= Stage::NP) break;
                if constexpr (BW != 16) /* in a slot that is there */
                    if (big(t.s[j]) && k * PR_TS + trow < span && !((bad >> (trow >> 4)) & 1))
                        s_big[slot3] = 1;
                put(t.w[j], BW == 16 ? 1.f : h2f(t.s[j]), (LDS(uint16_t)*)s_k[buf], trow, ch, false);
            }
        };
        auto store_v = [&](Stage& t, int k, int buf, int bad, int slot3) __attribute__((always_inline)) {
            const bool whole = k * PR_TS + PR_TS <= ss.L && bad == 0;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int i = tid + 64 * PR_W * j, trow = i / CR, ch = i % CR;
                if (Stage::NP % (64 * PR_W) && i >= Stage::NP) break;
                if (!whole) {
                    const int slot = k * PR_TS + trow;
                    const bool gone = slot >= ss.L + ss.n || ((bad >> (trow >> 4)) & 1);
                    const bool odd = !gone && slot >= ss.L &&
                                     (BW == 16 ? pr_odd(t.w[j]) : (t.s[j] & 0x7C00u) == 0x7C00u);
                    if (gone || odd) {
                        t.w[j] = (s2p_u32x4){0u, 0u, 0u, 0u};
                        if constexpr (BW != 16) t.s[j] = 0;
                    }
                    if (odd) atomicOr(&s_odd[slot3], 1ull << trow);
                }
                if constexpr (BW != 16)
                    if (big(t.s[j]) && k * PR_TS + trow < span) s_big[slot3] = 1;
                put(t.w[j], BW == 16 ? 1.f : h2f(t.s[j]), (LDS(uint16_t)*)s_v[buf], trow, ch, true);
            }
        };

        /* the next tile is on its way while one is worked on */
        Stage sk, sv;
        page_ids(k0);
        issue(sk, k0, false);
        issue(sv, k0, true);
        int bad = bad_of(k0), next = 0;
        store_k(sk, k0, 0, bad, seq);
        store_v(sv, k0, 0, bad, seq);
        if (k0 + 1 < k1) {
            issue(sk, k0 + 1, false);
            issue(sv, k0 + 1, true);
            next = bad_of(k0 + 1);
        }
        __syncthreads();
        for (int k = k0; k < k1; k++) {
            const int buf = (k - k0) & 1, tb = k * PR_TS;
            const LDS(uint16_t)* kt = (const LDS(uint16_t)*)s_k[buf];
            const LDS(uint16_t)* vt = (const LDS(uint16_t)*)s_v[buf];
            const int after = seq == 2 ? 0 : seq + 1;
            const unsigned long long odd = s_odd[seq];
            bool down = false; /* the tile's K and V are 2^-7 of themselves */
            float tscale = scale;
            if constexpr (BW != 16) {
                down = s_big[seq] != 0;
                if (down) { /* uniform and rare */
                    for (int i = tid; i < Stage::NP; i += 64 * PR_W) {
                        const int trow = i / CR, ch = i % CR, slot = min(tb + trow, span - 1);
                        int id = tab[slot >> a.l.shift];
                        const bool there = tb + trow < span && (unsigned)id < (unsigned)a.l.pages;
                        if (!there) id = 0; /* masked */
                        const size_t at = (((size_t)id * a.l.planes + kvh) << a.l.shift) +
                                          (slot & (a.l.page - 1));
                        const size_t av = at + ((size_t)a.kvh << a.l.shift);
                        const int gp = BW == 8 ? ch >> 1 : ch;
                        put(*(const s2p_u32x4*)(a.l.kv + at * EL + 16 * ch),
                            h2f(a.l.sc[at * 4 + gp]) * 0.0078125f, (LDS(uint16_t)*)s_k[buf], trow, ch, false);
                        uint16_t vs = a.l.sc[av * 4 + gp];
                        if (!there || (slot >= ss.L && (vs & 0x7C00u) == 0x7C00u)) vs = 0;
                        put(*(const s2p_u32x4*)(a.l.kv + av * EL + 16 * ch), h2f(vs) * 0.0078125f,
                            (LDS(uint16_t)*)s_v[buf], trow, ch, true);
                    }
                    tscale = scale * 128.0f;
                    __syncthreads();
                }
            }
            /* the marks of the tile before: everybody has read them, nobody has set them again */
            if (tid == 0) s_odd[seq ? seq - 1 : 2] = s_big[seq ? seq - 1 : 2] = 0;
            const bool work = busy && tb < wend;
            const bool open = tb + PR_TS <= open_end && bad == 0;
            uint64_t seen = ~0ull;
            if (!open) {
                seen = (a.vis ? pd_mask(word, ss.L - tb) : pd_ones(max(0, sees - tb))) & pd_groups(bad);
                if (!live) seen = 0;
            }
            any |= work && seen != 0;
            /* byte addresses in LDS: the permuted chunk is the row's own, xor the operand's number
             * (made here for every tile: kept, they would cost a register a read) */
            uint32_t ka = pd_lds((const LDS(unsigned char)*)kt) + col * 256 + ((half ^ (col & 15)) << 4);
            uint32_t va;
            {
                const int r = 4 * half + ((lane >> 2) & 3);
                va = pd_lds((const LDS(unsigned char)*)vt) + r * 256 +
                     (((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ (r << 1)) << 4) + 8 * (lane & 1);
            }
            asm volatile("" : "+v"(ka), "+v"(va));
            s2p_u32x4 kr[8];
            auto read_k = [&](int h) __attribute__((always_inline)) { /* slots 32 h + col */
#pragma unroll
                for (int ks = 0; ks < 8; ks++)
                    kr[ks] = *(const LDS(s2p_u32x4)*)((const LDS(unsigned char)*)(uintptr_t)(ka ^ (ks << 5)) +
                                                      8192 * h);
                __builtin_amdgcn_sched_barrier(0); /* the reads are out before what follows */
            };
            /* V^T operand of dims 32 dt .., slots 16 kb + 4 half + 0 .. 3 and + 8: lane 4 r + c
             * gives row r, dims 4 c .. */
            auto read_v = [&](int kb, int dt) __attribute__((always_inline)) {
                const LDS(unsigned char)* p =
                    (const LDS(unsigned char)*)(uintptr_t)(va ^ (dt << 6)) + 4096 * kb;
                const s2p_u32x2 b0 = ds_read_tr16((const LDS(uint16_t)*)p);
                const s2p_u32x2 b1 = ds_read_tr16((const LDS(uint16_t)*)(p + 2048));
                return (s2p_u32x4){b0.x, b0.y, b1.x, b1.y};
            };
            if (work) {
                read_k(part);
#pragma unroll
                for (int hh = 0; hh < 2 / SP; hh++) { /* halves of 32 slots */
                    const int h = SP == 2 ? part : hh;
                    pr_f32x16 sc;
#pragma unroll
                    for (int i = 0; i < 16; i++) sc[i] = 0.f;
                    /* the products go first: while a wave has them another one's softmax fills
                     * the vector unit (2 x 2,048 rows 252 us, 259 without; around O's too: 261) */
                    __builtin_amdgcn_s_setprio(1);
#pragma unroll
                    for (int ks = 0; ks < 8; ks++)
                        sc = BW == 16 ? mfma32x32x16(kr[ks], qb[ks], sc) : mfma32x32x16_f16(kr[ks], qb[ks], sc);
                    __builtin_amdgcn_s_setprio(0);
                    __builtin_amdgcn_sched_barrier(0);
                    /* the next operands are read while the softmax runs */
                    s2p_u32x4 vr[2][4];
#pragma unroll
                    for (int dt = 0; dt < 4; dt++) vr[0][dt] = read_v(2 * h, dt);
                    __builtin_amdgcn_sched_barrier(0);
                    if (SP == 1 && h == 0) read_k(1);
                    /* x[i]: slot 32 h + 8 (i / 4) + 4 half + i % 4 of this lane's vector */
                    float x[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) x[i] = sc[i];
                    const uint32_t mine = (uint32_t)(seen >> (32 * h)) >> (4 * half);
                    if (!open) {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (!((mine >> (8 * (i >> 2) + (i & 3))) & 1)) x[i] = -INFINITY;
                    }
                    float tm = x[0];
#pragma unroll
                    for (int i = 1; i < 16; i++) tm = fmaxf(tm, x[i]);
                    tm = pr_swap_max(tm) * tscale;
                    if (__any(tm > m + PR_LAZY)) {
                        const float mn = tm > m + PR_LAZY ? tm : m;
                        const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                        l *= corr;
#pragma unroll
                        for (int dt = 0; dt < 4; dt++) o[dt] *= corr;
                        m = mn;
                    }
                    const float ms = m == -INFINITY ? 0.f : m - SHIFT;
                    float ls = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], tscale, -ms));
                        ls += x[i];
                    }
                    l += ls;
                    if (odd) { /* uniform and rare: what store_v left out, from the page */
                        for (uint32_t w = (uint32_t)(odd >> (32 * h)); w; w &= w - 1) {
                            const int t = __ffs(w) - 1, slot = tb + 32 * h + t;
                            float p = 0.f;
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                p = (t >> 3) == (i >> 2) && (t & 3) == (i & 3) ? x[i] : p;
                            p = __shfl(p, ((t >> 2) & 1) * 32 + col, 64);
                            if ((seen >> (32 * h + t)) & 1) {
                                const int id = tab[slot >> a.l.shift]; /* there: its bit is set */
                                const size_t at = (((size_t)id * a.l.planes + a.kvh + kvh) << a.l.shift) +
                                                  (slot & (a.l.page - 1));
                                const char* vp = a.l.kv + at * EL;
#pragma unroll
                                for (int i = 0; i < 16; i++) { /* o[i / 4], dims 8 (i % 4) + 4 half .. */
                                    float v[4];
                                    if constexpr (BW == 16) {
                                        const s2p_u32x4 w8 =
                                            *(const s2p_u32x4*)(vp + 64 * (i >> 2) + 16 * (i & 3));
                                        if (!pr_odd(w8)) continue;
#pragma unroll
                                        for (int e = 0; e < 4; e++) {
                                            const uint32_t d = half ? w8[2 + (e >> 1)] : w8[e >> 1];
                                            v[e] = e & 1 ? bf2f_hi(d) : bf2f_lo(d);
                                        }
                                    } else {
                                        const uint16_t vs = a.l.sc[at * 4 + (i >> 2)];
                                        if ((vs & 0x7C00u) != 0x7C00u) continue;
                                        const int d = 32 * (i >> 2) + 8 * (i & 3) + 4 * half;
#pragma unroll
                                        for (int e = 0; e < 4; e++) {
                                            const int byte = (int8_t)vp[BW == 8 ? d + e : (d + e) >> 1];
                                            const int c = BW == 8 ? byte
                                                          : e & 1 ? byte >> 4 : (int)((uint32_t)byte << 28) >> 28;
                                            v[e] = (float)c * h2f(vs);
                                        }
                                    }
#pragma unroll
                                    for (int e = 0; e < 4; e++)
                                        o[i >> 2][4 * (i & 3) + e] =
                                            fmaf(p, v[e], o[i >> 2][4 * (i & 3) + e]);
                                }
                            }
                        }
                    }
                    if (BW != 16 && down) {
#pragma unroll
                        for (int dt = 0; dt < 4; dt++) o[dt] *= 0.0078125f;
                    }
#pragma unroll
                    for (int dt = 0; dt < 4; dt++) vr[1][dt] = read_v(2 * h + 1, dt);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        s2p_u32x4 pw;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            pw[e] = BW == 16 ? pd_pk(x[8 * b + 2 * e], x[8 * b + 2 * e + 1])
                                             : pr_pk_f16(x[8 * b + 2 * e], x[8 * b + 2 * e + 1]);
#pragma unroll
                        for (int dt = 0; dt < 4; dt++)
                            o[dt] = BW == 16 ? mfma32x32x16(vr[b][dt], pw, o[dt])
                                             : mfma32x32x16_f16(vr[b][dt], pw, o[dt]);
                    }
                    if (BW != 16 && down) {
#pragma unroll
                        for (int dt = 0; dt < 4; dt++) o[dt] *= 128.0f;
                    }
                }
            }
            bad = next;
            if (k + 1 < k1) {
                store_k(sk, k + 1, buf ^ 1, bad, after);
                store_v(sv, k + 1, buf ^ 1, bad, after);
                if (k + 2 < k1) {
                    page_ids(k + 2);
                    issue(sk, k + 2, false);
                    issue(sv, k + 2, true);
                    next = bad_of(k + 2);
                }
            }
            seq = after;
            __syncthreads();
        }
        /* out, or the partial of a tile that other blocks work on too */
        float lt0 = pr_swap_sum(l);
        if constexpr (SP == 2) { /* the second wave's state to the first, through the tiles' LDS */
            LDS(s2p_f32x4)* const x01 = (LDS(s2p_f32x4)*)s_k + 512 * vw + lane;
            LDS(s2p_f32x4)* const x23 = (LDS(s2p_f32x4)*)s_v + 512 * vw + lane;
            if (part == 1 && busy) {
                if (half == 0) {
                    s_ml[vec][0] = m;
                    s_ml[vec][1] = lt0;
                }
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        (dt < 2 ? x01 : x23)[64 * (4 * (dt & 1) + q)] =
                            (s2p_f32x4){o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
            }
            __syncthreads();
            if (part == 0 && busy) {
                const float m1 = s_ml[vec][0], l1 = s_ml[vec][1];
                const float mn = fmaxf(m, m1), ms = mn == -INFINITY ? 0.f : mn;
                const float e0 = __builtin_amdgcn_exp2f(m - ms), e1 = __builtin_amdgcn_exp2f(m1 - ms);
                lt0 = fmaf(lt0, e0, l1 * e1);
                m = mn;
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const s2p_f32x4 z = (dt < 2 ? x01 : x23)[64 * (4 * (dt & 1) + q)];
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            o[dt][4 * q + e] = fmaf(o[dt][4 * q + e], e0, z[e] * e1);
                    }
            }
            __syncthreads(); /* the next row tile's loads go there */
        }
        const bool leave = live && part == 0;
        const float lt = m == -INFINITY ? (any ? 1.f : 0.f) : lt0; /* -inf everywhere, not nothing */
        if (k0 == 0 && stop == last) {
            const float inv = m == -INFINITY ? (any ? NAN : 0.f) : 1.f / lt;
            if (leave) {
                uint16_t* out = a.out + ((size_t)row * a.qh + vhead) * PG_HD + 4 * half;
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        *(s2p_u32x2*)(out + 32 * dt + 8 * q) =
                            (s2p_u32x2){pd_pk(o[dt][4 * q] * inv, o[dt][4 * q + 1] * inv),
                                        pd_pk(o[dt][4 * q + 2] * inv, o[dt][4 * q + 3] * inv)};
            }
        } else {
            float* const po = a.work + ((size_t)(kvh * a.nb + blk) * 2 + (k0 == 0 ? 1 : 0)) *
                                           ((size_t)VEC * (PG_HD + 2));
            if (leave) {
                if (half == 0) {
                    po[2 * vec] = m;
                    po[2 * vec + 1] = lt;
                }
                float* const pz = po + 2 * VEC + vec * PG_HD + 4 * half;
#pragma unroll
                for (int dt = 0; dt < 4; dt++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        *(s2p_f32x4*)(pz + 32 * dt + 8 * q) =
                            (s2p_f32x4){o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
            }
            if (k0 == 0 && kvh == 0 && tid == 0) { /* what begins here and ends elsewhere */
                a.sums[4 * blk] = ss.r0 + i0;
                a.sums[4 * blk + 2] = (int)(((int64_t)last * nb - 1) / total); /* its last block */
            }
            if (k0 == 0) nvec_out = nvec;
        }
    }
    if (kvh == 0 && tid == 0) a.sums[4 * blk + 1] = nvec_out;
}

/* Row tiles that several blocks worked on, from their partials: a block a (block where the tile
 * begins, kv head, 8 / PARTS vectors), as in k_paged_merge. */
template <int PARTS>
__global__ __launch_bounds__(256) void k_paged_rows_merge(PgAttn a, int tile) {
    constexpr int VECS = 8 / PARTS;
    __shared__ float s_m[VECS][PARTS][3];
    __shared__ s2p_f32x4 s_z[VECS][PARTS][32];
    const int j0 = blockIdx.z, kvh = blockIdx.y;
    const int tid = threadIdx.x, x = tid & 31, part = (tid >> 5) % PARTS, u = (tid >> 5) / PARTS;
    const int vec = blockIdx.x * VECS + u;
    const int row0 = a.sums[4 * j0], nvec = a.sums[4 * j0 + 1], j1 = a.sums[4 * j0 + 2];
    if ((int)blockIdx.x * VECS >= nvec) return;
    const bool live = vec < nvec;
    const size_t stride = (size_t)tile * (PG_HD + 2);
    PgSum o;
    if (live)
        o = pd_gather<PARTS>(a.work + (size_t)kvh * a.nb * 2 * stride, stride, tile, j0, j1, vec,
                                part, 4 * x);
    if (x == 0) {
        s_m[u][part][0] = o.M;
        s_m[u][part][1] = o.lt;
        s_m[u][part][2] = o.mark;
    }
    s_z[u][part][x] = o.z;
    __syncthreads();
    if (part || !live) return;
#pragma unroll
    for (int i = 1; i < PARTS; i++)
        pd_add(o, s_m[u][i][0], s_m[u][i][1], s_z[u][i][x], s_m[u][i][2]);
    pd_out(a, row0, kvh, vec, 4 * x, o.z, o.M, o.lt, o.mark);
}

/* blocks a kv head and tile of query vectors: as many as fit at once, `each` a CU, and no more
 * than there are rounds of `rnd` slots */
static int64_t pd_blocks(const s2p_page_batch* b, int tiles, int rnd, int each) {
    const int64_t most = (int64_t)b->sessions * ((b->max_len + rnd - 1) / rnd);
    int64_t nb = each * s2p_cu_count() / tiles;
    if (nb < 1) nb = 1;
    return nb < most ? nb : most;
}

template <int BW, int MQT>
static hipError_t pd_launch(PgAttn a, hipStream_t st) {
    const int rnd = PdTile<BW>::TS * PD_WAVES;
    a.nvt = (a.b.max_rows * a.g + 16 * MQT - 1) / (16 * MQT);
    a.nb = (int)pd_blocks(&a.b, a.kvh * a.nvt, rnd, BW == 8 && MQT == 1 ? 3 : 2);
    hipLaunchKernelGGL((k_paged_dec<BW, MQT>), dim3((unsigned)(a.nb * a.nvt * a.kvh)),
                       dim3(64 * PD_WAVES), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nb == 1 || a.b.max_len <= rnd) return e; /* no session is shared */
    hipLaunchKernelGGL(k_paged_merge, dim3((unsigned)((a.b.max_rows * a.g + PM_VECS - 1) / PM_VECS),
                                           (unsigned)a.kvh, (unsigned)a.b.sessions),
                       dim3(256), 0, st, a, 16 * MQT);
    return hipGetLastError();
}

template <int BW, int SP>
static hipError_t pr_launch(PgAttn a, hipStream_t st) {
    hipLaunchKernelGGL((k_paged_rows<BW, SP>), dim3((unsigned)(a.nb * a.kvh)), dim3(64 * PR_W), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nb == 1) return e;
    /* a row tile's partials: many where there are few row tiles (one session of 8,192 tokens and 17
     * rows takes 24 us with four threads on a vector's, 31 with one; 2 x 2,048 rows, of mostly two
     * partials, 266 and 256) */
    constexpr int tile = 32 * PR_W / SP;
    const int64_t tiles = (int64_t)a.b.sessions * ((a.b.max_rows + a.rt - 1) / a.rt);
    if (a.nb > 4 * tiles)
        hipLaunchKernelGGL((k_paged_rows_merge<4>), dim3(tile / 2, (unsigned)a.kvh, (unsigned)a.nb),
                           dim3(256), 0, st, a, tile);
    else
        hipLaunchKernelGGL((k_paged_rows_merge<1>), dim3(tile / 8, (unsigned)a.kvh, (unsigned)a.nb),
                           dim3(256), 0, st, a, tile);
    return hipGetLastError();
}
/* Waves that share 32 of a row tile's vectors, each with half of a tile's slots: two where no
 * session has more than 128 vectors, whose tiles would leave waves idle (32 sessions x 16 rows x 4
 * heads a kv head at 300 tokens 18.3 us, 21.5 with one) */
static int pr_split(int64_t vecs) { return vecs <= 32 * PR_W / 2 ? 2 : 1; }
/* blocks a kv head over row tiles of rt rows: one a CU, no more than there are rounds */
static int64_t pr_blocks(const s2p_page_batch* b, int kv_heads, int rt) {
    const int64_t most = (int64_t)b->sessions * ((b->max_rows + rt - 1) / rt) *
                         (PR_BEGIN + (b->max_len + PR_TS - 1) / PR_TS);
    int64_t nb = s2p_cu_count() / kv_heads;
    if (nb < 1) nb = 1;
    return nb < most ? nb : most;
}

extern "C" int64_t s2pk_paged_attention_work_floats(const s2p_page_batch* batch, int q_heads,
                                                    int kv_heads) {
    if (!batch || batch->sessions <= 0 || batch->rows <= 0 || kv_heads <= 0 ||
        !pg_group(q_heads, kv_heads))
        return 0;
    const int64_t vecs = (int64_t)batch->max_rows * pg_group(q_heads, kv_heads);
    if (vecs > 32) {
        const int tile = 32 * PR_W / pr_split(vecs);
        const int64_t nb = pr_blocks(batch, kv_heads, tile / pg_group(q_heads, kv_heads));
        return 4 * nb + kv_heads * nb * 2 * tile * (PG_HD + 2);
    }
    const int64_t sums = (batch->sessions + 3) & ~3;
    return sums + kv_heads * pd_blocks(batch, kv_heads, 128, 3) * 2 * (vecs > 16 ? 32 : 16) * (PG_HD + 2);
}

extern "C" hipError_t s2pk_paged_attention(const s2p_page_pool* pool, const s2p_page_batch* batch,
                                           int layer, const s2p_bf16* q, int q_heads,
                                           const uint64_t* vis, s2p_bf16* out, float* work,
                                           hipStream_t st) {
    if (batch && batch->rows <= 0) return hipSuccess;
    if (!pg_pool_ok(pool) || !pg_batch_ok(pool, batch) || layer < 0 || layer >= pool->layers ||
        !pg_group(q_heads, pool->kv_heads) || !q || !out || !work || (const void*)q == (void*)out ||
        (((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) || ((uintptr_t)vis & 7) ||
        (vis && batch->max_rows > 64))
        return hipErrorInvalidValue;
    PgAttn a = {};
    a.l = pg_layer(pool, layer);
    a.b = *batch;
    a.q = (const uint16_t*)q;
    a.vis = vis;
    a.out = (uint16_t*)out;
    a.sums = (int*)work;
    a.qh = q_heads;
    a.kvh = pool->kv_heads;
    a.g = pg_group(q_heads, pool->kv_heads);
    const int64_t vecs = (int64_t)batch->max_rows * a.g;
    const bool split = pr_split(vecs) == 2;
    a.rt = 32 * PR_W / pr_split(vecs) / a.g;
    /* rounds are counted in 32 bits */
    if ((int64_t)batch->sessions * ((batch->max_rows + a.rt - 1) / a.rt) *
            (PR_BEGIN + (batch->max_len + PR_TS - 1) / PR_TS) > 1 << 30)
        return hipErrorInvalidValue;
    if (vecs > 32) {
        a.nb = (int)pr_blocks(batch, a.kvh, a.rt);
        a.work = work + 4 * (int64_t)a.nb;
        if (split) return pool->bits == 16 ? pr_launch<16, 2>(a, st)
                          : pool->bits == 8 ? pr_launch<8, 2>(a, st) : pr_launch<4, 2>(a, st);
        return pool->bits == 16 ? pr_launch<16, 1>(a, st)
               : pool->bits == 8 ? pr_launch<8, 1>(a, st) : pr_launch<4, 1>(a, st);
    }
    a.work = work + ((batch->sessions + 3) & ~3);
    /* 17 to 32 vectors: two tiles of them in a wave where its registers hold them.  INT4's do not
     * (64-slot tiles; 16 sessions x 5 rows at 8,192 tokens take 145 us so, 72 with a block for each
     * tile); INT8's spill a little, which pays from about six rounds a block on (8 sessions x 5 rows
     * at 8,000 tokens 44 and 54 us; at 250 tokens 14 and 13, of 256 to 4,096 tokens 29 and 26). */
    const bool two = vecs > 16 && (pool->bits == 16 || (pool->bits == 8 &&
                     (int64_t)batch->sessions * ((batch->max_len + 127) / 128) * a.kvh >=
                         6 * 2 * (int64_t)s2p_cu_count()));
    if (two) return pool->bits == 16 ? pd_launch<16, 2>(a, st) : pd_launch<8, 2>(a, st);
    return pool->bits == 16 ? pd_launch<16, 1>(a, st)
           : pool->bits == 8 ? pd_launch<8, 1>(a, st) : pd_launch<4, 1>(a, st);
}
