// hy_paged_attn.hip -- attention of ragged batches of new tokens over a paged cache
// (hy_paged_attention): out = sum_j softmax_j(scale q . k_j) v_j over the keys a row sees.
//
// paged_few_kernel: requests of few rows (single tokens, drafts).  A stream over K and V: one
// wave works for itself on 16 NT rows (token x query head of a kv head; 32 over 16-bit caches:
// hy_paged_wide.hip) and goes over its keys
// 32 (f32: 16) at a time, straight from memory into the operands of 16 x 16 MFMAs, without LDS
// and barriers:
//  * S^T = K Q^T: lane l = 16 g + i holds key i's dims, 16 bytes at a time;
//  * the result has keys 4 g + v and row i in lane l, which is the B operand of
//    O^T = V^T P^T as it stands: V's lane holds the 4 keys 4 g .. 4 g + 3 of its dims, so for
//    16-bit types the pairs of keys are put together by byte permutes;
//  * softmax statistics: one query row per lane, joined over the four g.
// f32 accuracy from 16-bit operands: q and the probabilities are split into pieces that the
// matrix cores multiply exactly -- a f16 cache: two f16 pieces (22 bits, q scaled per row by a
// power of two, weights by 2^6); a bf16 cache: three bf16 pieces (24 bits) -- while K and V go in
// as they are.  f32 caches use the fp32 MFMAs.
// Keys that a row does not see get weight 0, but 0 times an infinity or NaN in their V would
// still be felt.  Keys that no row sees (a page's unwritten end) have their V zeroed; where
// some rows do not see a key, V is looked at, and if it is not finite the piece is computed again
// key by key (slow_rows).
// Bound by the bytes of K and V: 64 single tokens over bf16 caches of up to 8000 keys (1.24 GB)
// 225 us, 5.5 TB/s; one token over 1000 f32 keys 10 us, all of it latency (7000 cycles from launch
// to the first loads).
#include "hy_device.hpp"
#include "hy_lds.hpp"
#include "hy_paged.hpp"
#include "hy_paged_part.hpp"
#include "hy_paged_split.hpp"

namespace hy {

// over lanes i, 16 + i, 32 + i, 48 + i
__device__ __forceinline__ float group_max(float v) { return fmax_half(fmax_row(v)); }
__device__ __forceinline__ float group_sum(float v) { return fadd_half(fadd_row(v)); }

template <class E, int HD, int NT>
__global__ __launch_bounds__(WAVE * PF_WAVES, 2) void paged_few_kernel(PagedAttnArgs a, PartShape ps) {
    using P = PaType<E>;
    constexpr bool F32T = sizeof(E) == 4, F16T = std::is_same<E, _Float16>::value;
    constexpr int KB = F32T ? 16 : 32;       // keys per turn
    constexpr int KT = KB / 16;              // 16-key tiles of scores
    constexpr int NQ = F32T ? HD / 16 : HD / 32;   // 16-byte loads of a key per lane
    constexpr int VL = F32T ? HD / 64 : 1;         // loads of a value row per lane
    constexpr int VD = F32T ? 4 : HD / 16;         // dims of each
    constexpr int ND = HD / 16;              // 16-dim tiles of the output
    constexpr int PC = P::PIECES;
    constexpr int VW = VD * (int)sizeof(E) / 4;    // dwords of a V load
    __shared__ PartSums<WAVE * PF_WAVES> sums;
    const int lane = threadIdx.x % WAVE, i = lane % 16, g4 = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int64_t total = part_sums(a, ps, sums);
    const int64_t stretch = part_stretch(ps, total);
    const int worker = blockIdx.x * PF_WAVES + wave;
    int64_t x = worker * stretch;
    const int64_t x_end = min(x + stretch, total);
    const int G = ps.G, pmask = (1 << a.c.shift) - 1;
    const float qscale = a.scale * 1.4426950408889634f;

    PartJob job{};
    while (x < x_end) {
        const PartItem it = part_find(a, ps, sums, x);
        int p0, p1;
        if (!part_piece(ps, it, x, x_end, p0, p1)) continue;

        // rows of this lane's columns; rows past the last repeat it and are not stored
        const int n_live = min(it.q.n * G - it.tile * ps.M, ps.M);
        const int rho0 = it.tile * ps.M, tok0 = part_quotient(rho0, G);
        int row[NT], head[NT], end[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int rho = rho0 + min(16 * t + i, n_live - 1) - tok0 * G, tok1 = part_div(rho, G), tok = tok0 + tok1;
            row[t] = it.q.start + tok;
            head[t] = it.g * G + rho - tok1 * G;
            end[t] = a.seen ? min(a.seen[row[t]], it.q.kv) : it.q.kv - it.q.n + tok + 1;
        }
        int last, first;  // the most and the fewest keys that a row sees
        if (a.seen) {
            last = max(end[0], 0);
            first = end[0];
            if constexpr (NT == 2) {
                last = max(last, end[1]);
                first = min(first, end[1]);
            }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) {
                last = max(last, shfl_xor(last, d));
                first = min(first, shfl_xor(first, d));
            }
        } else {
            first = it.q.kv - it.q.n + tok0 + 1;
            last = max(it.q.kv - it.q.n + tok0 + part_div(rho0 - tok0 * G + n_live - 1, G) + 1, 0);
        }
        last = uniform(last);
        first = uniform(first);
        const int blocks = (last + 31) / 32;
        const int t0 = part_block(p0, it.len, blocks) * (32 / KB), t1 = part_block(p1, it.len, blocks) * (32 / KB);

        job = part_job(ps, it, p0, p1, stretch, n_live);
        const int slot_id = p0 == 0 && p1 == it.len ? -1 : 2 * worker + (p0 == 0 ? 1 : 0);  // -1: all of it is here

        // q: scaled by scale * log2(e) (scores in the base-2 domain); f16: by a power of two that
        // brings the row's largest to [2^13, 2^14), undone on the scores
        float qx[F32T ? NT : 1][F32T ? HD / 4 : 1];
        v4i_t qf[F32T ? 1 : NT][F32T ? 1 : NQ][PC];
        float unscale[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float* const qp = a.q + ((int64_t)row[t] * a.nh + head[t]) * HD;
            unscale[t] = 1.0f;
            if constexpr (F32T) {
                v4f_t q[NQ];
#pragma unroll
                for (int s = 0; s < NQ; s++) q[s] = *reinterpret_cast<const v4f_t*>(qp + 16 * s + 4 * g4);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s = 0; s < NQ; s++)
#pragma unroll
                    for (int j = 0; j < 4; j++) qx[t][4 * s + j] = q[s][j] * qscale;
            } else {
                v4f_t q[NQ][2];
                float big = 0.0f;
#pragma unroll
                for (int s = 0; s < NQ; s++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        q[s][u] = *reinterpret_cast<const v4f_t*>(qp + 32 * s + 8 * g4 + 4 * u);
                    }
                __builtin_amdgcn_sched_barrier(0);  // all of them in flight
#pragma unroll
                for (int s = 0; s < NQ; s++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        q[s][u] *= qscale;
#pragma unroll
                        for (int j = 0; j < 4; j++) big = fmaxf(big, fabsf(q[s][u][j]));
                    }
                float up = 1.0f;
                if constexpr (F16T) {
                    big = group_max(big);
                    const int e = min(max((int)((__float_as_uint(big) >> 23) & 255) - 127, -100), 127);
                    up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                    unscale[t] = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
                }
#pragma unroll
                for (int s = 0; s < NQ; s++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t w[PC];
                        P::split(q[s][j / 2][2 * (j % 2)] * up, q[s][j / 2][2 * (j % 2) + 1] * up, w);
#pragma unroll
                        for (int c = 0; c < PC; c++) qf[t][s][c][j] = (int)w[c];
                    }
            }
        }

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
        const E* const kbase = static_cast<const E*>(a.c.k) + it.g * a.c.head_stride;
        const E* const vbase = static_cast<const E*>(a.c.v) + it.g * a.c.head_stride;

        v4i_t kx[KT][NQ];
        int vx[KT][4][VL * VW];
        int vpage[KT];  // the page of this lane's value keys, -1: none
        auto page_of = [&](int key) { return __shfl(tab, (key >> a.c.shift) & 63, WAVE); };
        // loads of a turn; keys without a page read page 0
        auto load_k = [&](int t) {
            const int s = (t * KB) >> (a.c.shift + 6);
            if (s != seg) {  // wave-uniform; turns come in order
                seg = s;
                tab = tab2;
                tab2 = entries(seg + 1);
            }
#pragma unroll
            for (int u = 0; u < KT; u++) {
                const int key = t * KB + 16 * u + i;
                const E* const kp = kbase + max(page_of(key), 0) * a.c.page_stride + (key & pmask) * a.c.token_stride +
                                    16 / sizeof(E) * g4;
#pragma unroll
                for (int n = 0; n < NQ; n++) kx[u][n] = *reinterpret_cast<const v4i_t*>(kp + 64 / sizeof(E) * n);
            }
        };
        auto load_v = [&](int t) {
#pragma unroll
            for (int u = 0; u < KT; u++) {
                const int key = t * KB + 16 * u + 4 * g4;
                vpage[u] = page_of(key);
                const E* const vp =
                    vbase + max(vpage[u], 0) * a.c.page_stride + (key & pmask) * a.c.token_stride + VD * i;
#pragma unroll
                for (int v = 0; v < 4; v++)
#pragma unroll
                    for (int n = 0; n < VL; n++) {
                        const E* const src = vp + v * a.c.token_stride + 64 * n;
                        if constexpr (VW == 4) {
                            const v4i_t w = *reinterpret_cast<const v4i_t*>(src);
#pragma unroll
                            for (int j = 0; j < 4; j++) vx[u][v][4 * n + j] = w[j];
                        } else {
                            const uint2 w = *reinterpret_cast<const uint2*>(src);
                            vx[u][v][0] = (int)w.x;
                            vx[u][v][1] = (int)w.y;
                        }
                    }
            }
        };

        v4f_t o[NT][ND];
        bool odd = false;  // an infinity or NaN in V where some rows do not see a key
        float m_run[NT], l_run[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            m_run[t] = -INFINITY;
            l_run[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < ND; d++) o[t][d] = v4f_t{};
        }

        if (t0 < t1) {
            load_k(t0);
            load_v(t0);
        }
        for (int t = t0; t < t1; t++) {
            // K's registers are free after the scores, V's after its products: the next turn's
            // loads go out there and run under the rest, and under the other wave of the SIMD
            v4f_t s[NT][KT];
#pragma unroll
            for (int c = 0; c < NT; c++)
#pragma unroll
                for (int u = 0; u < KT; u++) {
                    if constexpr (F32T) {
                        // four sums (two, where registers are short) of their part of the dims: an f32
                        // score of one chain of 128 terms is off by twice as much, and each product
                        // would wait for the last
                        constexpr int CH = NT == 2 && HD == 128 ? 2 : 4;
                        v4f_t acc[CH] = {};
#pragma unroll
                        for (int n = 0; n < NQ; n++) {
                            const v4f_t k = __builtin_bit_cast(v4f_t, kx[u][n]);
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                acc[j % CH] =
                                    __builtin_amdgcn_mfma_f32_16x16x4f32(k[j], qx[c][4 * n + j], acc[j % CH], 0, 0, 0);
                        }
                        s[c][u] = acc[0] + acc[1];
                        if constexpr (CH == 4) s[c][u] += acc[2] + acc[3];
                    } else {
                        v4f_t acc = v4f_t{};
#pragma unroll
                        for (int n = 0; n < NQ; n++)
#pragma unroll
                            for (int q = PC - 1; q >= 0; q--) acc = P::mfma(kx[u][n], qf[c][n][q], acc);
                        s[c][u] = acc;
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) load_k(t + 1);
            __builtin_amdgcn_sched_barrier(0);
            bool none = false;
#pragma unroll
            for (int u = 0; u < KT; u++) none |= vpage[u] < 0;
            const bool edge = (t + 1) * KB > first || __any(none);
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < NT; c++)
#pragma unroll
                for (int u = 0; u < KT; u++) top = top_bits<4>(s[c][u], top);
            if (__any(top >= PA_MINUS_INF)) {
#pragma unroll
                for (int c = 0; c < NT; c++)
#pragma unroll
                    for (int u = 0; u < KT; u++) minus_inf_to_nan<4>(s[c][u]);
            }
#pragma unroll
            for (int c = 0; c < NT; c++) {
                if (edge) {  // wave-uniform
                    asm volatile("");
#pragma unroll
                    for (int u = 0; u < KT; u++)
#pragma unroll
                        for (int v = 0; v < 4; v++)
                            if (t * KB + 16 * u + 4 * g4 + v >= end[c] || vpage[u] < 0) s[c][u][v] = -INFINITY;
                }
                float big = -INFINITY;
#pragma unroll
                for (int u = 0; u < KT; u++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        if constexpr (F16T) s[c][u][v] *= unscale[c];
                        big = fmaxf(big, s[c][u][v]);
                    }
                if (__any(big > m_run[c] + PA_LAG)) {
                    big = group_max(big);
                    const float m = big > m_run[c] + PA_LAG ? big : m_run[c];
                    const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[c] - m);
                    m_run[c] = m;
                    l_run[c] *= alpha;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[c][d] *= alpha;
                }
                const float ref = m_run[c] == -INFINITY ? 0.0f : m_run[c];
#pragma unroll
                for (int u = 0; u < KT; u++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        s[c][u][v] = __builtin_amdgcn_exp2f(s[c][u][v] - ref);
                        l_run[c] += s[c][u][v];  // of this lane's keys; joined behind the loop
                    }
            }
            if (edge) {
#pragma unroll
                for (int u = 0; u < KT; u++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const bool gone = t * KB + 16 * u + 4 * g4 + v >= last || vpage[u] < 0;
#pragma unroll
                        for (int w = 0; w < VL * VW; w++) {
                            vx[u][v][w] = gone ? 0 : vx[u][v][w];
                            odd |= P::odd((uint32_t)vx[u][v][w]);
                        }
                    }
            }
            if constexpr (F32T) {
#pragma unroll
                for (int v = 0; v < 4; v++)
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int c = 0; c < NT; c++)
                            o[c][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vx[0][v][d]),
                                                                          s[c][0][v], o[c][d], 0, 0, 0);
            } else {
                v4i_t pf[NT][PC];
#pragma unroll
                for (int c = 0; c < NT; c++)
#pragma unroll
                    for (int u = 0; u < KT; u++)
#pragma unroll
                        for (int v = 0; v < 2; v++) {
                            uint32_t w[PC];
                            const float f = F16T ? PF_PSCALE : 1.0f;
                            P::split(s[c][u][2 * v] * f, s[c][u][2 * v + 1] * f, w);
#pragma unroll
                            for (int q = 0; q < PC; q++) pf[c][q][2 * u + v] = (int)w[q];
                        }
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    v4i_t vf;  // dims VD i + d of keys 4 g4 .. + 3 of both tiles
#pragma unroll
                    for (int u = 0; u < KT; u++)
#pragma unroll
                        for (int v = 0; v < 2; v++)
                            vf[2 * u + v] = (int)__builtin_amdgcn_perm(
                                (uint32_t)vx[u][2 * v + 1][d / 2], (uint32_t)vx[u][2 * v][d / 2],
                                d % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int c = 0; c < NT; c++)
#pragma unroll
                        for (int q = PC - 1; q >= 0; q--) o[c][d] = P::mfma(vf, pf[c][q], o[c][d]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) load_v(t + 1);
        }

#pragma unroll
        for (int c = 0; c < NT; c++) l_run[c] = group_sum(l_run[c]);
        float down = F16T ? 1.0f / PF_PSCALE : 1.0f;
        if (__any(odd)) {  // again, key by key
            down = 1.0f;
#pragma unroll
            for (int c = 0; c < NT; c++)
                slow_rows<E, HD, 4>(
                    a, trow, it.q.kv, t0 * KB, t1 * KB, end[c], a.q + ((int64_t)row[c] * a.nh + head[c]) * HD, kbase,
                    vbase,
                    [&](int n) {
                        return F32T ? 64 * (n / 16) + 4 * (4 * g4 + n % 4) + n / 4 % 4 : VD * (4 * g4 + n % 4) + n / 4;
                    },
                    [&](int n, float v) { o[c][n / 4][n % 4] = v; },
                    [&](int n) { return o[c][n / 4][n % 4]; }, m_run[c], l_run[c]);
        }
        float* const slot = a.ws + ps.ws + (size_t)max(slot_id, 0) * part_slot_floats(ps.M, HD);
#pragma unroll
        for (int c = 0; c < NT; c++) {
            if (16 * c + i >= n_live) continue;
            float* dst;
            float f = down;
            if (slot_id < 0) {
                dst = a.out + ((int64_t)row[c] * a.nh + head[c]) * HD;
                f = l_run[c] == 0.0f ? 0.0f : down / l_run[c];
            } else {
                dst = slot + (16 * c + i) * HD;
                if (g4 == 0) {
                    slot[ps.M * HD + 16 * c + i] = m_run[c];
                    slot[ps.M * (HD + 1) + 16 * c + i] = l_run[c];
                }
            }
            // dims VD (4 g4 + v) + d are in a row for d = 0 .. VD - 1
#pragma unroll
            for (int n = 0; n < VL; n++)
#pragma unroll
                for (int v = 0; v < 4; v++)
#pragma unroll
                    for (int j = 0; j < VD; j += 4) {
                        const int d = VD * n + j;
                        *reinterpret_cast<v4f_t*>(dst + 64 * n + VD * (4 * g4 + v) + j) =
                            (v4f_t){o[c][d][v], o[c][d + 1][v], o[c][d + 2][v], o[c][d + 3][v]} * f;
                    }
        }
    }
    if (lane == 0) part_jobs(a, ps, HD)[worker] = job;
}

// Joins the pieces of the items that are cut, from the jobs the workers left: work group (w, split)
// takes every splits-th set of rows of worker w's; in it, HD / 4 threads take 4 dims each of
// a row and every pl_n-th piece of it, PJ pieces at a time, and the pl_n groups of a row meet in
// LDS.  In slots by lanes neighbouring threads are neighbouring rows, eight of them (128 bytes), and
// eight threads of a row 128 bytes of the output; in slots by rows they are a row's.  Bound by the
// partial results' bytes (4 TB/s of them for tiles of 256 rows), for short ones by the latency of
// job, pieces and result: hence rows and pieces spread as far as they go.
// one of splits work groups for worker w0's item; LANES: of part_at's slots
template <int HD, int PJ, bool LANES>
__device__ __forceinline__ void join_item(const PagedAttnArgs& a, const PartShape& ps, int w0, int split, int splits,
                                          float (&meet)[6][256]) {
    const PartJob job = part_jobs(a, ps, HD)[w0];
    const int n_piece = uniform(job.n_piece), n_live = uniform(job.n_live);
    if (n_piece == 0) return;
    const size_t sf = part_slot_floats(ps.M, HD);
    const float* const first = a.ws + ps.ws + (size_t)(2 * w0 + 1) * sf;
    const float* const rest = a.ws + ps.ws + (size_t)(2 * w0) * sf;  // piece k > 0: + 2 k slots
    constexpr int TR = HD / 4, GROUPS = 256 / TR;
    int pl_n = 1;
    while (pl_n < 8 && pl_n * PJ < n_piece) pl_n *= 2;
    const int tid = threadIdx.x, rs_n = GROUPS / pl_n;
    const int d = (LANES ? tid / 8 : tid) % TR * 4, group = LANES ? tid % 8 + tid / (8 * TR) * 8 : tid / TR;
    const int pl = LANES ? group / rs_n : group % pl_n, rs = LANES ? group % rs_n : group / pl_n;
    for (int i0 = split * rs_n; i0 < n_live; i0 += rs_n * splits) {  // the same for the work group
        const int i = min(i0 + rs, n_live - 1), at = LANES ? part_at(HD, i, d) : i * HD + d;
        float m = -INFINITY, l = 0.0f;
        v4f_t o = v4f_t{};
        for (int k0 = pl; k0 < n_piece; k0 += pl_n * PJ) {
            float mk[PJ], lk[PJ];
            v4f_t ok[PJ];
#pragma unroll
            for (int j = 0; j < PJ; j++) {
                const int k = min(k0 + j * pl_n, n_piece - 1);
                const float* const s = k == 0 ? first : rest + (size_t)(2 * k) * sf;
                mk[j] = s[ps.M * HD + i];
                lk[j] = s[ps.M * (HD + 1) + i];
                ok[j] = *reinterpret_cast<const v4f_t*>(s + at);
            }
            __builtin_amdgcn_sched_barrier(0);
            float mn = m;
#pragma unroll
            for (int j = 0; j < PJ; j++) mn = fmaxf(mn, mk[j]);
            const float ref = mn == -INFINITY ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - ref);
            m = mn;
            l *= alpha;
            o *= alpha;
#pragma unroll
            for (int j = 0; j < PJ; j++) {
                const float f = __builtin_amdgcn_exp2f(mk[j] - ref);
                if (k0 + j * pl_n < n_piece) {
                    l += f * lk[j];
                    o += f * ok[j];
                }
            }
        }
        if (pl_n > 1) {
            // the thread of the row's next group: group + 1 by rows, group + rs_n by lanes, whose low
            // three bits are in tid's
            const auto other = [&](int k) {
                if (!LANES) return tid + k * TR;
                const int g = group + k * rs_n;
                return tid / 8 % TR * 8 + g % 8 + g / 8 * (8 * TR);
            };
            __syncthreads();  // the last rows' are read
            meet[4][tid] = m;
            meet[5][tid] = l;
#pragma unroll
            for (int j = 0; j < 4; j++) meet[j][tid] = o[j];
            __syncthreads();
            if (pl == 0) {
                float mn = m;
                for (int k = 1; k < pl_n; k++) mn = fmaxf(mn, meet[4][other(k)]);
                const float ref = mn == -INFINITY ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - ref);
                l *= alpha;
                o *= alpha;
                for (int k = 1; k < pl_n; k++) {
                    const int from = other(k);
                    const float f = __builtin_amdgcn_exp2f(meet[4][from] - ref);
                    l += f * meet[5][from];
#pragma unroll
                    for (int j = 0; j < 4; j++) o[j] += f * meet[j][from];
                }
            }
        }
        if (pl == 0 && i0 + rs < n_live) {
            const int rho = job.rho0 + i, tok = rho / ps.G;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t head = (int64_t)(job.start + tok) * a.nh + job.g * ps.G + rho - tok * ps.G;
            *reinterpret_cast<v4f_t*>(a.out + head * HD + d) = o * inv;
        }
    }
}

// MANY: with both in it the kernel has 78 registers, for streams alone 56
template <int HD, int PJ, bool MANY>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, PartShape few, PartShape many, int few_splits,
                                                        int many_splits) {
    __shared__ float meet[6][256];
    const int b = (int)blockIdx.x - few.workers * few_splits;
    if (!MANY || b < 0)
        join_item<HD, PJ, false>(a, few, blockIdx.x / few_splits, blockIdx.x % few_splits, few_splits, meet);
    else
        join_item<HD, PJ, true>(a, many, b / many_splits, b % many_splits, many_splits, meet);
}

constexpr int PJ_ROWS = 8;  // rows of a stream's item per work group of the join

// which launches a batch takes: workers 0: not that one
struct PaPlan {
    PartShape few, many;
};
constexpr int PF_ROWS = 32;
// Rows of the largest request up to which the streams take a whole batch; past it they take the
// requests of PF_ROWS rows at most (f16, 14 requests of up to 744 rows: 50, all up to 128 rows 62).
// They read K and V once per 32 rows (from caches, past the first), but start quickly and need no
// second launch; the tiles of 256 rows do more per key where there are rows enough.  Measured with
// both, us:
//  * head_dim 64, 16 bits: 4 requests of 1024 rows 31 by tiles, 25 by the stream; 6 requests of 2048
//    behind 1000 keys 54, 48, of 4096 78, 85.  f32: 6 of 512 53, 42, 2 of 1024 behind 6000 keys 77, 119;
//  * head_dim 128, more than two requests: f16, 16 of 128 behind 8000 keys 139, 138, of 256 203, 290;
//    bf16, of 256 227, 214, 6 of 384 behind 1000 58, 59; f32, 8 of 64 behind 1000 60, 47, 16 of 96
//    behind 8000 237, 319;
//  * one or two requests of head_dim 128 are few items, which the stream cuts into more pieces than
//    pay: 2 of 64 behind 6000, f16 42, 62.
static int pf_max_rows(int type, int n_req, int hd) {
    if (hd == 64) return type == HY_TYPE_F32 ? 512 : 2048;
    if (n_req <= 2) return PF_ROWS;
    return type == HY_TYPE_F32 ? 64 : type == HY_TYPE_F16 ? 128 : 256;
}

static PaPlan pa_plan(int type, int n_req, int max_new, int G, int hd) {
    const int64_t rows = (int64_t)max_new * G;  // of one request, at most
    constexpr int64_t ALL = (int64_t)1 << 62;
    const bool many = rows > pf_max_rows(type, n_req, hd), few = !many || n_req > 1;
    PaPlan p;
    // Beside chunks the stream's requests are mostly single tokens: 16 rows (12 requests of chunks and
    // tokens, bf16, 414 -> 406 us; 32 rows would spare drafts beside chunks a second reading of K and V,
    // which was not timed).
    // Starting an item is worth 16 keys of a full stream, 256 of a many-row tile (20 000 of its 3500
    // to 6500 cycles per 32 keys); a stretch is 32 keys at least (64: one request of
    // 1000 keys 12.6 us, 32: 10.2), 128.  Cuts within 32, 128 of an item's end move there: a small
    // piece costs its start and a partial result (2 requests of up to 172 tokens, f16, 53 -> 45 us,
    // 88 drafts of up to 15 behind 5 keys 18 -> 15; 64 for the streams: a token over 1000 keys 12 -> 14).
    p.few = part_shape(rows > 16 && !many ? 5 : 4, G, 0, many ? PF_ROWS : ALL, few ? PF_WORKERS : 0, 16, 32, 32, 0);
    const size_t few_ws = part_ws_floats(p.few.workers, p.few.M, hd);
    p.many = part_shape(PM_TILE_SHIFT, G, few ? PF_ROWS : 0, ALL, many ? PM_WORKERS : 0, 256, 128, 128, few_ws);
    return p;
}

size_t paged_attn_ws_bytes(int type, int n_req, int max_new, int G, int hd) {
    const PaPlan p = pa_plan(type, n_req, max_new, G, hd);
    return 4 * (p.many.ws + part_ws_floats(p.many.workers, PM_TILE, hd));
}

template <class E, int HD>
static void launch_few(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s) {
    if constexpr (sizeof(E) == 4) {
        if (ps.M == 32) {
            hipLaunchKernelGGL((paged_few_kernel<E, HD, 2>), dim3(PF_GROUPS), dim3(WAVE * PF_WAVES), 0, s, a, ps);
            return;
        }
    }
    hipLaunchKernelGGL((paged_few_kernel<E, HD, 1>), dim3(PF_GROUPS), dim3(WAVE * PF_WAVES), 0, s, a, ps);
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, int max_new, hipStream_t s) {
    const PaPlan p = pa_plan(a.c.type, a.n_req, max_new, a.nh / a.c.nkv, a.c.hd);
    const bool big = a.c.hd == 128;
    if (p.few.workers) {
        if (a.c.type != HY_TYPE_F32 && p.few.M == 32)
            launch_paged_wide(a, p.few, s);
        else if (a.c.type == HY_TYPE_F32)
            big ? launch_few<float, 128>(a, p.few, s) : launch_few<float, 64>(a, p.few, s);
        else if (a.c.type == HY_TYPE_F16)
            big ? launch_few<_Float16, 128>(a, p.few, s) : launch_few<_Float16, 64>(a, p.few, s);
        else
            big ? launch_few<__bf16, 128>(a, p.few, s) : launch_few<__bf16, 64>(a, p.few, s);
    }
    if (p.many.workers) launch_paged_many(a, p.many, s);
    const int splits = p.few.M / PJ_ROWS;
    const int many_splits = a.c.hd / 4;  // a tile of few pieces: one set of rows per work group
    const dim3 grid(p.few.workers * splits + p.many.workers * many_splits);
    // Items of 32 pieces and more: eight pieces at a time (1000 keys, one request: 4.0 us, by fours
    // 5.6), elsewhere four, of half the registers (32 requests of 24 rows: 11.4, by eights 12.8).
    const bool long_ = a.n_req * a.c.nkv * 32 <= p.few.workers;
    const auto join = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, p.few, p.many, splits, many_splits);
    };
    if (p.many.workers)
        big ? join(paged_join_kernel<128, 4, true>) : join(paged_join_kernel<64, 4, true>);
    else if (long_)
        big ? join(paged_join_kernel<128, 8, false>) : join(paged_join_kernel<64, 8, false>);
    else
        big ? join(paged_join_kernel<128, 4, false>) : join(paged_join_kernel<64, 4, false>);
    return hipGetLastError();
}

}  // namespace hy
