// hy_paged_wide.hip -- the paged attention of requests of 17 to 32 rows (drafts) over 16-bit caches:
// paged_few_kernel's stream (hy_paged_attn.hip) with 32 rows per wave on 32 x 32 x 16 MFMAs, which
// do 1.8 times the products of the 16 x 16 x 32 ones in the same time (2090 and 1140 TFLOP/s, two
// waves per SIMD).  A turn is 32 keys:
//  * S^T = K Q^T: lane l = 32 h + i holds key i's dims 16 c + 8 h .. + 7 in step c;
//  * the result has keys 8 u + 4 h + v and row i in lane l, the B operand of O^T = V^T P^T as it
//    stands; V's lane holds HD / 32 dims of those keys, put in pairs by byte permutes;
//  * a row's statistics: lanes i and 32 + i.
// Pieces of q and the weights, masks and V's that are not finite: as there; the weights' 2^6 is in
// the exponent, so a row's sum carries it too.
// Bound by the bytes of K and V and by what a wave does between its loads: 32 requests of 6 tokens
// over f16 caches of up to 2900 keys (255 MB) 67 us (on 16 x 16 tiles 74), 3.8 TB/s, of which
// some 10 us are the start and the end of a launch.  At head_dim 128 the f16 kernel spills 20
// registers, and the bf16 one, of three pieces, has one wave per SIMD (365 registers; not
// timed by itself).
#include "hy_device.hpp"
#include "hy_paged.hpp"
#include "hy_paged_part.hpp"
#include "hy_paged_split.hpp"

namespace hy {

template <class E, int HD>
__global__ __launch_bounds__(WAVE * PF_WAVES, PaType<E>::PIECES == 3 && HD == 128 ? 1 : 2) void paged_wide_kernel(
    PagedAttnArgs a, PartShape ps) {
    using P = PaType<E>;
    constexpr bool F16T = std::is_same<E, _Float16>::value;
    constexpr int KB = 32, M = 32;
    constexpr int NQ = HD / 16;        // 16-byte loads of a key per lane
    constexpr int ND = HD / 32;        // dims of a value row per lane, 32-dim tiles of the output
    constexpr int PC = P::PIECES;
    constexpr int WUP = F16T ? 6 : 0;  // of the weights
    typedef typename std::conditional<ND == 4, uint2, uint32_t>::type vrow_t;
    __shared__ PartSums<WAVE * PF_WAVES> sums;
    const int lane = threadIdx.x % WAVE, i = lane % 32, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int64_t total = part_sums(a, ps, sums);
    const int64_t stretch = part_stretch(ps, total);
    const int worker = blockIdx.x * PF_WAVES + wave;
    int64_t x = worker * stretch;
    const int64_t x_end = min(x + stretch, total);
    const int G = ps.G, pmask = (1 << a.c.shift) - 1;
    const uint32_t ts = (uint32_t)a.c.token_stride;
    const uint32_t v_off = (4 * h * ts + ND * i) * sizeof(E);

    PartJob job{};
    while (x < x_end) {
        const PartItem it = part_find(a, ps, sums, x);
        int p0, p1;
        if (!part_piece(ps, it, x, x_end, p0, p1)) continue;

        // this lane's row; rows past the last repeat it and are not stored
        const int n_live = min(it.q.n * G - it.tile * M, M);
        const int rho0 = it.tile * M, tok0 = part_quotient(rho0, G);
        const int rho = rho0 + min(i, n_live - 1) - tok0 * G, tok1 = part_div(rho, G), tok = tok0 + tok1;
        const int row = it.q.start + tok, head = it.g * G + rho - tok1 * G;
        const int end = a.seen ? min(a.seen[row], it.q.kv) : it.q.kv - it.q.n + tok + 1;
        int last = end, first = end;  // the most and the fewest keys that a row sees
        if (a.seen) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                last = max(last, shfl_xor(last, d));
                first = min(first, shfl_xor(first, d));
            }
        } else {  // the last row's, the first row's
            last = __builtin_amdgcn_readlane(end, 31);
        }
        last = max(uniform(last), 0);
        first = uniform(first);
        const int blocks = (last + 31) / 32;
        const int t0 = part_block(p0, it.len, blocks), t1 = part_block(p1, it.len, blocks);

        job = part_job(ps, it, p0, p1, stretch, n_live);
        const int slot_id = p0 == 0 && p1 == it.len ? -1 : 2 * worker + (p0 == 0 ? 1 : 0);  // -1: all of it is here

        const float* const qp = a.q + ((int64_t)row * a.nh + head) * HD;
        v4i_t qf[NQ][PC];
        float unscale = 1.0f;
        {
            const float qscale = a.scale * 1.4426950408889634f;
            v4f_t q[NQ][2];
            float big = 0.0f;
#pragma unroll
            for (int s = 0; s < NQ; s++)
#pragma unroll
                for (int u = 0; u < 2; u++) q[s][u] = *reinterpret_cast<const v4f_t*>(qp + 16 * s + 8 * h + 4 * u);
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
                big = fmax_half(big);
                const int e = min(max((int)((__float_as_uint(big) >> 23) & 255) - 127, -100), 127);
                up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                unscale = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
            }
#pragma unroll
            for (int s = 0; s < NQ; s++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w[PC];
                    P::split(q[s][j / 2][2 * (j % 2)] * up, q[s][j / 2][2 * (j % 2) + 1] * up, w);
#pragma unroll
                    for (int c = 0; c < PC; c++) qf[s][c][j] = (int)w[c];
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

        v4i_t kx[NQ];
        vrow_t vx[4][4];  // keys 8 u + 4 h + v
        int vpage[4];     // the page of keys 8 u .. + 7 (a page has 8 at least), -1: none
        // loads of a turn; keys without a page read page 0
        auto load_k = [&](int t) {
            const int s = (t * KB) >> (a.c.shift + 6);
            if (s != seg) {  // wave-uniform; turns come in order
                seg = s;
                tab = tab2;
                tab2 = entries(seg + 1);
            }
            const int key = t * KB + i, page = __shfl(tab, (key >> a.c.shift) & 63, WAVE);
            const E* const kp = kbase + max(page, 0) * a.c.page_stride + (key & pmask) * a.c.token_stride + 8 * h;
#pragma unroll
            for (int n = 0; n < NQ; n++) kx[n] = *reinterpret_cast<const v4i_t*>(kp + 16 * n);
        };
        auto load_v = [&](int t) {  // after load_k(t)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int key = t * KB + 8 * u;
                vpage[u] = __builtin_amdgcn_readlane(tab, (key >> a.c.shift) & 63);
                const char* const vp = reinterpret_cast<const char*>(vbase + max(vpage[u], 0) * a.c.page_stride +
                                                                     (key & pmask) * a.c.token_stride);
#pragma unroll
                for (int v = 0; v < 4; v++)
                    vx[u][v] = *reinterpret_cast<const vrow_t*>(vp + (v_off + v * ts * (uint32_t)sizeof(E)));
            }
        };

        v16f_t o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = v16f_t{};
        bool odd = false;  // an infinity or NaN in V where some rows do not see a key
        float m_run = -INFINITY, l_run = 0.0f;
        if (t0 < t1) {
            load_k(t0);
            load_v(t0);
        }
        for (int t = t0; t < t1; t++) {
            // K's registers are free after the scores, V's after its products: the next turn's
            // loads go out there and run under the rest, and under the other wave of the SIMD
            v16f_t s = v16f_t{};
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int q = PC - 1; q >= 0; q--) s = P::mfma(kx[n], qf[n][q], s);
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) load_k(t + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (__any(top_bits<16>(s) >= PA_MINUS_INF)) minus_inf_to_nan<16>(s);
            const bool edge = (t + 1) * KB > first || (vpage[0] | vpage[1] | vpage[2] | vpage[3]) < 0;
            if (edge) {  // wave-uniform
                asm volatile("");
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int key = t * KB + 8 * u + 4 * h + v;
                        if (key >= end || vpage[u] < 0) s[4 * u + v] = -INFINITY;
                        const bool gone = key >= last || vpage[u] < 0;
                        if constexpr (ND == 4) {
                            vx[u][v].x = gone ? 0 : vx[u][v].x;
                            vx[u][v].y = gone ? 0 : vx[u][v].y;
                            odd |= P::odd(vx[u][v].x) || P::odd(vx[u][v].y);
                        } else {
                            vx[u][v] = gone ? 0 : vx[u][v];
                            odd |= P::odd(vx[u][v]);
                        }
                    }
            }
            float big = s[0];
#pragma unroll
            for (int v = 1; v < 16; v++) big = fmaxf(big, s[v]);
            if constexpr (F16T) big *= unscale;
            if (__any(big > m_run + PA_LAG)) {
                big = fmax_half(big);
                const float m = big > m_run + PA_LAG ? big : m_run;
                const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m);
                m_run = m;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= alpha;
            }
            const float up = (m_run == -INFINITY ? 0.0f : m_run) - (float)WUP;
#pragma unroll
            for (int v = 0; v < 16; v++) {
                s[v] = __builtin_amdgcn_exp2f(F16T ? fmaf(s[v], unscale, -up) : s[v] - up);
                l_run += s[v];  // of this lane's keys; joined behind the loop
            }
            v4i_t pf[2][PC];
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w[PC];
                    P::split(s[8 * c + 2 * j], s[8 * c + 2 * j + 1], w);
#pragma unroll
                    for (int q = 0; q < PC; q++) pf[c][q][j] = (int)w[q];
                }
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    v4i_t vf;  // dim ND i + d of the lane's 8 keys of step c
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const vrow_t &v0 = vx[2 * c + j / 2][2 * (j % 2)], &v1 = vx[2 * c + j / 2][2 * (j % 2) + 1];
                        uint32_t w0, w1;
                        if constexpr (ND == 4) {
                            w0 = d / 2 ? v0.y : v0.x;
                            w1 = d / 2 ? v1.y : v1.x;
                        } else {
                            w0 = v0;
                            w1 = v1;
                        }
                        vf[j] = (int)__builtin_amdgcn_perm(w1, w0, d % 2 ? 0x07060302u : 0x05040100u);
                    }
#pragma unroll
                    for (int q = PC - 1; q >= 0; q--) o[d] = P::mfma(vf, pf[c][q], o[d]);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) load_v(t + 1);
        }

        l_run = fadd_half(l_run);
        float down = 1.0f;
        // the n-th of a lane's dims: tile n / 16, its row 8 u + 4 h + v
        const auto dim = [&](int n) { return ND * (8 * (n % 16 / 4) + 4 * h + n % 4) + n / 16; };
        if (__any(odd)) {  // again, key by key
            slow_rows<E, HD, 2>(
                a, trow, it.q.kv, t0 * KB, t1 * KB, end, qp, kbase, vbase, dim,
                [&](int n, float v) { o[n / 16][n % 16] = v; }, [&](int n) { return o[n / 16][n % 16]; }, m_run, l_run);
            down = (float)(1 << WUP);  // as the other pieces of its item
            l_run *= down;
        }
        if (i < n_live) {
            float* dst;
            float f = down;
            if (slot_id < 0) {
                dst = a.out + ((int64_t)row * a.nh + head) * HD;
                f = l_run == 0.0f ? 0.0f : down / l_run;
            } else {
                float* const slot = a.ws + ps.ws + (size_t)slot_id * part_slot_floats(M, HD);
                dst = slot + i * HD;
                if (h == 0) {
                    slot[M * HD + i] = m_run;
                    slot[M * (HD + 1) + i] = l_run;
                }
            }
            constexpr int STEP = 4 / ND;
#pragma unroll
            for (int v = 0; v < 16; v += STEP) {
                v4f_t y;
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = o[j % ND][v + j / ND] * f;
                *reinterpret_cast<v4f_t*>(dst + dim(v)) = y;
            }
        }
    }
    if (lane == 0) part_jobs(a, ps, HD)[worker] = job;
}

template <class E>
static void launch(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s) {
    if (a.c.hd == 128)
        hipLaunchKernelGGL((paged_wide_kernel<E, 128>), dim3(PF_GROUPS), dim3(WAVE * PF_WAVES), 0, s, a, ps);
    else
        hipLaunchKernelGGL((paged_wide_kernel<E, 64>), dim3(PF_GROUPS), dim3(WAVE * PF_WAVES), 0, s, a, ps);
}

void launch_paged_wide(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s) {
    if (a.c.type == HY_TYPE_F16)
        launch<_Float16>(a, ps, s);
    else
        launch<__bf16>(a, ps, s);
}

}  // namespace hy
