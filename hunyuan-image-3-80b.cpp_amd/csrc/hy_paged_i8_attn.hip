// hy_paged_i8_attn.hip -- attention of ragged batches over a paged cache of 8-bit integers
// (hy_paged_attention_i8): out = sum_j softmax_j(scale q . k_j) v_j, k_j and v_j codes times the scale of
// their block.
//
// paged_i8_few_kernel: requests of few rows (single tokens, drafts).  A stream over the codes, as
// paged_few_kernel's (hy_paged_attn.hip): one wave works for itself on L rows (token x query head of a
// kv head; 16, or 32) and goes over its keys 64 (32 rows: 32) at a time, from memory into registers, as
// f16 into the operands of L x L MFMAs, without LDS and barriers:
//  * a code is exact in f16: the byte, its sign flipped, behind 0x64 is 1024 + 128 + code, less 1152;
//  * S^T = K Q^T: lane l = L g + i holds a key's dims, 16 bytes at a time, two steps of 8;
//  * which key a row of K's operand is is free: rows are dealt so that lane l's 16 scores are 16 neighbouring
//    keys, 16 g .. + 15 of the turn -- two halves of 8, each in one page and one block, with one scale;
//  * they are the B operand of O^T = V^T W^T as they stand; V's lane holds HD / L dims of those keys,
//    put in pairs by byte permutes.
// f32 accuracy: q and the weights are two f16 pieces each (22 bits, q scaled per row by a power of two).
// K's scale joins the scores.  V's, 2^e m with 1 <= m < 2, joins the weights: with R the running maximum of
// t_j = s_j + e_j (base 2), w_j = 2^(t_j - R) m_j goes into the products and l sums 2^(t_j - R) 2^-e_j, so
// out = O / l whatever R; e is kept in -60 .. 34, so that no weight that counts in l underflows
// (hy_paged_many.hip).  e - R comes before s is added, so that nothing is rounded at the size of e.
// Keys that a row does not see get a score of -inf, and factors that leave them a weight of 0; codes are
// finite, whatever lies in memory.
//
// 32 heads over 8 kv heads of 128.  64 requests of one token behind up to 8000 keys: 127 us, 5.2 TB/s, the memory's
// rate.  32 of six tokens behind up to 2900 keys (32 rows): 39 us, 3.4 TB/s; about 20 of them are a worker's start
// and end (finding its piece, q, the block table, the first keys; partial results), the rest is held up by what a
// turn does in a row (turning codes into f16, products, maximum, exponentials, pieces).  One token behind 1000 keys:
// 8.2 us of latency, and 3.5 for the join.
#include "hy_device.hpp"
#include "hy_int8.hpp"
#include "hy_lds.hpp"
#include "hy_paged_part.hpp"
#include "hy_paged_split.hpp"

namespace hy {

template <int L>
struct I8Acc {
    typedef v4f_t type;
};
template <>
struct I8Acc<32> {
    typedef v16f_t type;
};
// row of an L x L result's register v of lane group g
template <int L>
__device__ __forceinline__ int acc_row(int v, int g) {
    return L == 16 ? 4 * g + v : 8 * (v / 4) + 4 * g + v % 4;
}
// over the lanes of a row
template <int L>
__device__ __forceinline__ float row_max(float v) {
    return fmax_half(L == 16 ? fmax_row(v) : v);
}
template <int L>
__device__ __forceinline__ float row_sum(float v) {
    return fadd_half(L == 16 ? fadd_row(v) : v);
}

template <int HD, int L>
__global__ __launch_bounds__(WAVE * PF_WAVES, 2) void paged_i8_few_kernel(PagedAttnArgs a, PartShape ps, float per_item) {
    using P = PaType<_Float16>;
    typedef typename I8Acc<L>::type acc_t;
    constexpr int GQ = WAVE / L;             // lanes of a row
    constexpr int KT = L == 16 ? 4 : 1;      // K tiles per turn
    constexpr int KB = KT * L;               // keys per turn
    constexpr int NL = HD / (16 * GQ);       // 16-byte loads of a key per lane
    constexpr int VD = HD / L;               // dims of a value row per lane, tiles of the output
    constexpr int VW = VD == 8 ? 2 : 1;      // dwords of them
    constexpr int SR = L * L / WAVE;         // scores of a tile per lane
    static_assert(KT * SR == 16 && KB == 16 * GQ, "16 neighbouring keys per lane");
    __shared__ PartSums<WAVE * PF_WAVES> sums;
    const int lane = threadIdx.x % WAVE, i = lane % L, g = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int64_t total = part_sums(a, ps, sums);
    // Pieces of few keys cost more in the join than they spare here: of an item of n keys sqrt(4 n) or more (one
    // request of 4 tokens behind 4000 keys 21 us, so 19, behind 1000 15.4 and 13.6)
    const int64_t least = uniform((int)__builtin_amdgcn_sqrtf((float)total * per_item));
    const int64_t stretch = max(part_stretch(ps, total), least);
    const int worker = blockIdx.x * PF_WAVES + wave;
    int64_t x = worker * stretch;
    const int64_t x_end = min(x + stretch, total);
    const int G = ps.G, pmask = (1 << a.c.shift) - 1;
    // the key of a turn that row i of K's tile u is, less 4 u (16 rows)
    const int k_key = L == 16 ? 16 * (i / 4) + i % 4 : 16 * (i / 4 % 2) + 4 * (i / 8) + i % 4;

    PartJob job{};
    while (x < x_end) {
        const PartItem it = part_find(a, ps, sums, x);
        int p0, p1;
        if (!part_piece(ps, it, x, x_end, p0, p1)) continue;

        // this lane's row; rows past the last repeat it and are not stored
        const int n_live = min(it.q.n * G - it.tile * L, L);
        const int rho0 = it.tile * L, tok0 = part_quotient(rho0, G);
        const int rho = rho0 + min(i, n_live - 1) - tok0 * G, tok1 = part_div(rho, G), tok = tok0 + tok1;
        const int row = it.q.start + tok, head = it.g * G + rho - tok1 * G;
        const int end = a.seen ? min(a.seen[row], it.q.kv) : it.q.kv - it.q.n + tok + 1;
        int last = end, first = end;  // the most and the fewest keys that a row sees
        if (a.seen) {
#pragma unroll
            for (int d = 1; d < L; d <<= 1) {
                last = max(last, shfl_xor(last, d));
                first = min(first, shfl_xor(first, d));
            }
        } else {  // the last row's, the first row's
            last = __builtin_amdgcn_readlane(end, L - 1);
        }
        last = max(uniform(last), 0);
        first = uniform(first);
        const int blocks = (last + KB - 1) / KB;
        const int t0 = part_block(p0, it.len, blocks), t1 = part_block(p1, it.len, blocks);

        job = part_job(ps, it, p0, p1, stretch, n_live);
        const int slot_id = p0 == 0 && p1 == it.len ? -1 : 2 * worker + (p0 == 0 ? 1 : 0);  // -1: all of it is here

        // block table: 64 entries in the lanes, the next 64 on their way
        const int* const trow = a.table + (int64_t)it.r * a.max_pages;
        const int n_tab = (it.q.kv + pmask) >> a.c.shift;
        auto entries = [&](int seg) {
            const int p = seg * 64 + lane;
            const int e = p < n_tab ? trow[p] : -1;
            return e >= 0 && e < a.c.n_pages ? e : -1;
        };
        int seg = (t0 * KB) >> (a.c.shift + 6);
        int tab = entries(seg), tab2 = entries(seg + 1);
        // q: scaled by scale * log2(e) and by a power of two that brings the row's largest to [2^13, 2^14)
        const float* const qp = a.q + ((int64_t)row * a.nh + head) * HD;
        v4i_t qf[2 * NL][2];
        float unscale;
        v4f_t q[2 * NL][2];
#pragma unroll
        for (int s = 0; s < 2 * NL; s++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                q[s][u] = *reinterpret_cast<const v4f_t*>(qp + 16 * GQ * (s / 2) + 16 * g + 8 * (s % 2) + 4 * u);
        const int8_t* const kbase = static_cast<const int8_t*>(a.c.k) + it.g * a.c.head_stride + 16 * g;
        const int8_t* const vbase = static_cast<const int8_t*>(a.c.v) + it.g * a.c.head_stride + VD * i;

        v4i_t kx[KT][NL];
        uint32_t vx[16][VW];
        float ks_next[2], vs_next[2];  // of the halves of this lane's 16 keys
        int vpage[2];                  // their pages, -1: none
        auto page_of = [&](int key) { return __shfl(tab, (key >> a.c.shift) & 63, WAVE); };
        // loads of a turn; keys without a page read page 0
        auto load_k = [&](int t) {
            const int s = (t * KB) >> (a.c.shift + 6);
            if (s != seg) {  // wave-uniform; turns come in order
                seg = s;
                tab = tab2;
                tab2 = entries(seg + 1);
            }
            int page = 0;
#pragma unroll
            for (int u = 0; u < KT; u++) {
                const int key = t * KB + k_key + 4 * u;
                if (u % 2 == 0) page = max(page_of(key), 0);  // two tiles lie in 8 neighbouring keys
                const int8_t* const kp = kbase + page * a.c.page_stride + (key & pmask) * a.c.token_stride;
#pragma unroll
                for (int n = 0; n < NL; n++) kx[u][n] = *reinterpret_cast<const v4i_t*>(kp + 16 * GQ * n);
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int key = t * KB + 16 * g + 8 * h, page = max(page_of(key), 0);
                const int64_t b = (((int64_t)page * a.c.nkv + it.g) << (a.c.shift - a.bshift)) + ((key & pmask) >> a.bshift);
                ks_next[h] = a.ks[b];
                vs_next[h] = a.vs[b];
            }
        };
        auto load_v = [&](int t) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int key = t * KB + 16 * g + 8 * h;
                vpage[h] = page_of(key);
                const int8_t* const vp = vbase + max(vpage[h], 0) * a.c.page_stride + (key & pmask) * a.c.token_stride;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int8_t* const src = vp + j * a.c.token_stride;
                    if constexpr (VD == 8) {
                        const uint2 w = *reinterpret_cast<const uint2*>(src);
                        vx[8 * h + j][0] = w.x;
                        vx[8 * h + j][1] = w.y;
                    } else if constexpr (VD == 4) {
                        vx[8 * h + j][0] = *reinterpret_cast<const uint32_t*>(src);
                    } else {
                        vx[8 * h + j][0] = *reinterpret_cast<const uint16_t*>(src);
                    }
                }
            }
        };

        __builtin_amdgcn_sched_barrier(0);
        {
            const float qscale = a.scale * 1.4426950408889634f;
            float big = 0.0f;
#pragma unroll
            for (int s = 0; s < 2 * NL; s++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    q[s][u] *= qscale;
#pragma unroll
                    for (int j = 0; j < 4; j++) big = fmaxf(big, fabsf(q[s][u][j]));
                }
            big = row_max<L>(big);
            const int e = min(max((int)((__float_as_uint(big) >> 23) & 255) - 127, -100), 127);
            const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
            unscale = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll
            for (int s = 0; s < 2 * NL; s++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t hi, lo;
                    split_f16(q[s][j / 2][2 * (j % 2)] * up, q[s][j / 2][2 * (j % 2) + 1] * up, hi, lo);
                    qf[s][0][j] = (int)hi;
                    qf[s][1][j] = (int)lo;
                }
        }

        acc_t o[VD];
#pragma unroll
        for (int d = 0; d < VD; d++) o[d] = acc_t{};
        float m_run = -INFINITY, l_run = 0.0f;
        if (t0 < t1) {
            load_k(t0);
            load_v(t0);
        }
        for (int t = t0; t < t1; t++) {
            // K's registers are free after the scores, V's after its products: the next turn's
            // loads go out there and run under the rest, and under the other wave of the SIMD
            float s[16];
#pragma unroll
            for (int u = 0; u < KT; u++) {
                acc_t acc = acc_t{};
#pragma unroll
                for (int n = 0; n < 2 * NL; n++) {
                    v4i_t kf;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        uint32_t w0, w1;
                        i8_to_f16((uint32_t)kx[u][n / 2][2 * (n % 2) + j], w0, w1);
                        kf[2 * j] = (int)w0;
                        kf[2 * j + 1] = (int)w1;
                    }
                    acc = P::mfma(kf, qf[n][1], acc);
                    acc = P::mfma(kf, qf[n][0], acc);
                }
#pragma unroll
                for (int v = 0; v < SR; v++) s[SR * u + v] = acc[v];
            }
            float fac[2], ex[2], inv[2], mant[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const I8Scale v = i8_scale(vs_next[h]);
                fac[h] = fmaf(ks_next[h], 0.0f, ks_next[h]) * unscale;  // an infinity becomes NaN
                ex[h] = v.ex;
                inv[h] = v.inv;
                mant[h] = v.mant;
            }
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) load_k(t + 1);
            __builtin_amdgcn_sched_barrier(0);
            const int key0 = t * KB + 16 * g;
            if ((t + 1) * KB > first || __any((vpage[0] | vpage[1]) < 0)) {  // wave-uniform
                asm volatile("");
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (key0 + v >= end || vpage[v / 8] < 0) s[v] = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    // eight keys of one block: what its scales are where this row sees none of them does not matter,
                    // and a NaN is the row's where it sees one; -inf times a scale of 0 would be NaN
                    const bool sees = key0 + 8 * h < end && vpage[h] >= 0;
                    fac[h] = !sees || fac[h] < 0x1p-126f ? 0x1p-126f : fac[h];
                    mant[h] = sees ? mant[h] : 0.0f;
                }
            }
            // scales are not negative: a half's largest score has its largest t
            float big = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float m = s[8 * h];
#pragma unroll
                for (int v = 1; v < 8; v++) m = fmaxf(m, s[8 * h + v]);
                big = fmaxf(big, fmaf(m, fac[h], ex[h]));
            }
            if (__any(big > m_run + PA_LAG)) {
                big = row_max<L>(big);
                const float m = big > m_run + PA_LAG ? big : m_run;
                const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m);
                m_run = m;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < VD; d++) o[d] *= alpha;
            }
            const float ref = (m_run == -INFINITY ? 0.0f : m_run) - 6.0f;  // weights are 2^6 times as large: PF_PSCALE
#pragma unroll
            for (int h = 0; h < 2; h++) ex[h] -= ref;
#pragma unroll
            for (int v = 0; v < 16; v++) {
                s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], fac[v / 8], ex[v / 8]));
                l_run = fmaf(s[v], inv[v / 8], l_run);  // of this lane's keys; joined behind the loop
                s[v] *= mant[v / 8];
            }
            v4i_t pf[2][2];
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t hi, lo;
                    split_f16(s[8 * c + 2 * j], s[8 * c + 2 * j + 1], hi, lo);
                    pf[c][0][j] = (int)hi;
                    pf[c][1][j] = (int)lo;
                }
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int d = 0; d < VD; d++) {
                    v4i_t vf;  // dim VD i + d of the lane's keys 8 c .. + 7
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        vf[j] = (int)i8_pair(vx[8 * c + 2 * j][d / 4], vx[8 * c + 2 * j + 1][d / 4], d % 4);
                    o[d] = P::mfma(vf, pf[c][1], o[d]);
                    o[d] = P::mfma(vf, pf[c][0], o[d]);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) load_v(t + 1);
        }

        l_run = row_sum<L>(l_run);
        if (i < n_live) {
            float* dst;
            float f = 1.0f;
            if (slot_id < 0) {
                dst = a.out + ((int64_t)row * a.nh + head) * HD;
                f = l_run == 0.0f ? 0.0f : 1.0f / l_run;
            } else {
                float* const slot = a.ws + ps.ws + (size_t)slot_id * part_slot_floats(L, HD);
                dst = slot + i * HD;
                if (g == 0) {
                    slot[L * HD + i] = m_run;
                    slot[L * (HD + 1) + i] = l_run;
                }
            }
            // dims VD row + d are in a row for d = 0 .. VD - 1
            constexpr int STEP = VD >= 4 ? 1 : 4 / VD;
#pragma unroll
            for (int v = 0; v < SR; v += STEP)
#pragma unroll
                for (int d = 0; d < VD; d += 4) {
                    v4f_t y;
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = STEP == 1 ? o[(d + j) % VD][v] : o[j % VD][v + j / VD];
                    *reinterpret_cast<v4f_t*>(dst + VD * acc_row<L>(v, g) + d) = y * f;
                }
        }
    }
    if (lane == 0) part_jobs(a, ps, HD)[worker] = job;
}

constexpr int PF_ROWS = 32;
// Rows of the largest request up to which the streams take a whole batch; past it they take the
// requests of PF_ROWS rows at most, tiles of 256 rows the others.  Requests x tokens (four rows each) behind keys,
// streams and tiles, us:
//  * 8 kv heads of 128: 1 x 16 behind 6000 31, 31, 4 x 16 43, 64, 8 x 16 66, 103, 16 x 16 108, 178; 1 x 32 34, 33,
//    4 x 32 59, 67, 8 x 32 100, 107, behind 1000 37, 46, 16 x 32 behind 2000 75, 77; 8 x 64 behind 1000 51, 54, 16 x 64
//    73, 73;
//  * 4 of 64: 16 x 16 behind 4000 39, 58, 8 x 32 40, 39.5, 16 x 32 60, 60; 2 x 64 28, 34, 4 x 64 40, 37, 8 x 64 63, 48;
//    1 x 128 27, 33, 2 x 128 40, 38, 4 x 128 62, 49; 1 x 256 37, 37;
//  * one kv head of 128, requests x rows: 1 x 64 behind 6000 24, 28.5, 1 x 128 27, 31, 4 x 128 31, 37, 16 x 128 43, 50;
//    4 x 96 behind 4000 28, 33, 8 x 128 33, 35, 8 x 256 35, 40; of 64: 1 x 128 behind 6000 20, 22, 8 x 128 behind 4000
//    24, 27.
// The border does not look at the kv heads: between 97 and 256 rows of head_dim 128 the streams would be as fast, or up
// to a fifth faster where there are few.
static int i8_max_rows(int n_req, int hd) {
    if (hd == 64) return n_req > 6 ? 128 : 768 / n_req;
    return 96;
}

// Up to HALF_ITEMS items half the workers, one wave per SIMD, take the stream: half the pieces, and twice the work
// groups for each item's join (launch_paged_join).  Four rows per token and 8 kv heads of 128, all and half the
// workers, us:
//  * 16 rows: one request of a token behind 1000 keys 12.5, 12.6, behind 120000 70, 57, of 4 behind 4000 20, 18; 8 of
//    one behind 4000 24, 23.5, of 4 39, 30; 32 (256 items) of one behind 2000 38, 39, of 4 49, 43; 64 (512) of one
//    behind 4000 112, 107, behind 8000 202, 194, 128 (1024) behind 2000 114, 111;
//  * 32 rows: one request of 6 behind 4000 23.2, 22.8, 4 of 6 31, 28; 32 of 6 (256) behind 2000 59, 53, behind 6000
//    110, 110; 16 of 8 behind 8000 (128) 101, 83; 64 of 5 behind 3000 (512) 109, 113; 16 of 24 behind 8000 (384)
//    169, 188.
// One kv head: 32 requests of 32 rows behind 4000 40, 33, of 128 rows of head_dim 64 38.5, 39; 128 of 8 rows behind
// 2000 29, 25.
constexpr int HALF_ITEMS = 256;
static int64_t i8_items(int64_t rows, int m_shift, int n_req, int nkv) {
    return ((rows + (1 << m_shift) - 1) >> m_shift) * n_req * nkv;
}

static PaPlan i8_plan(int n_req, int max_new, int G, int nkv, int hd) {
    const int64_t rows = (int64_t)max_new * G;  // of one request, at most
    constexpr int64_t ALL = (int64_t)1 << 62;
    const bool many = rows > i8_max_rows(n_req, hd), few = !many || n_req > 1;
    PaPlan p;
    const int shift = rows > 16 && !many ? 5 : 4;
    const bool half = !many && i8_items(rows, shift, n_req, nkv) <= HALF_ITEMS;
    const int workers = !few ? 0 : half ? PF_WORKERS / 2 : PF_WORKERS;
    p.few = part_shape(shift, G, 0, many ? PF_ROWS : ALL, workers, 16, 32, 32, 0);
    const size_t few_ws = part_ws_floats(p.few.workers, p.few.M, hd);
    p.many = part_shape(PM_TILE_SHIFT, G, few ? PF_ROWS : 0, ALL, many ? PM_WORKERS : 0, 256, 128, 128, few_ws);
    return p;
}

size_t paged_attn_i8_ws_bytes(int n_req, int max_new, int G, int nkv, int hd) {
    const PaPlan p = i8_plan(n_req, max_new, G, nkv, hd);
    return 4 * (p.many.ws + part_ws_floats(p.many.workers, PM_TILE, hd));
}

template <int HD>
static void launch(const PagedAttnArgs& a, const PaPlan& p, int max_new, hipStream_t s) {
    // beside chunks there are fewer items than the batch could have: no least stretch
    const int64_t items = i8_items((int64_t)max_new * p.few.G, p.few.m_shift, a.n_req, a.c.nkv);
    const float per_item = p.many.workers || !items ? 0.0f : 4.0f / (float)items;
    const dim3 grid(p.few.workers / PF_WAVES), block(WAVE * PF_WAVES);
    if (p.few.M == 32)
        hipLaunchKernelGGL((paged_i8_few_kernel<HD, 32>), grid, block, 0, s, a, p.few, per_item);
    else
        hipLaunchKernelGGL((paged_i8_few_kernel<HD, 16>), grid, block, 0, s, a, p.few, per_item);
}

hipError_t launch_paged_attn_i8(const PagedAttnArgs& a, int max_new, hipStream_t s) {
    const PaPlan p = i8_plan(a.n_req, max_new, a.nh / a.c.nkv, a.c.nkv, a.c.hd);
    if (p.few.workers) a.c.hd == 128 ? launch<128>(a, p, max_new, s) : launch<64>(a, p, max_new, s);
    if (p.many.workers) launch_paged_many(a, p.many, s);
    return launch_paged_join(a, p, s);
}

}  // namespace hy
