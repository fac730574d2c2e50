// hy_paged_many.hip -- the paged attention of requests with many rows (chunks of a prompt): a
// work group of eight waves per tile of 256 rows (token x query head of a kv head, 32 per
// wave) and stretch of keys (hy_paged_part.hpp), both products on the f16 matrix cores with f32
// accuracy.
//
// Splits.  q and the weights go in as two f16 pieces, hi + lo (11 + 11 bits, each rounded to
// nearest: 2^-24 of the value), an f32 cache's K and V too, 16-bit caches as one (exact).  A
// product is hi hi + hi lo + lo hi; the missing lo lo is below 2^-24 of it.  f16 has few
// exponents, so every vector is scaled by a power of two that brings its largest element to
// the top of its range: q per row, and for f32 and bf16 caches K and V per key (elements down to
// 2^-27 of their vector's largest keep all bits of a piece, none is off by more than 2^-38 of it).  K's
// factor is undone on the scores.  V's, 2^e_j, joins the weights: with R the running
// maximum of s_j + e_j the accumulators sum w_j v_j 2^-e_j, w_j = 2^(s_j + e_j - R),
// and w_j 2^-e_j = 2^(s_j - R), which leaves out = O / l in any reference R.  e_j lies in
// PM_ELO .. PM_EHI: then a w_j that l is formed from stays above 2^-126 wherever 2^(s_j - R) counts
// in l (2^-30 of its largest term: -30 + PM_ELO - PM_EHI + PM_WUP > -126), within a piece
// and where pieces meet.  A row of zeros takes PM_ELO, which raises no R above the others'; smaller
// values share it; a piece with larger ones is computed again key by key.  s_j + e_j is rounded at its
// own size: 300 keys, f32, values of size 1 are 2e-7 off 64 bits, of 1e-10 1e-6.
//
// Blocks of 32 keys: every thread loads its share of a block of K and V one block ahead,
// splits it and stores the pieces to LDS, K as it is and V transposed, both in MFMA operand
// order.  Scores are computed transposed, S^T = K Q^T, so a query's statistics stay in its
// lane pair and its weights are the operand of O^T += V^T W^T as they lie.
//
// Bound by instruction issue and the power it draws: a SIMD's two waves have, per block and head_dim
// 128 of a bf16 cache, 64 products (32 cycles each, 2050) and 2700 cycles of vector operations
// (half of them the softmax), and take 4700, about their sum (running the waves half a block apart
// changed nothing; what keeps the two kinds of work apart is not known), and the clock falls to
// 1.6 GHz under it.  2048 rows of 32 heads behind 8192 keys, f32: 0.93 ms (the first passes of
// a run 1.07), 330 TFLOP/s of attention and three times that of f16 products (a large f16 matrix
// product reaches 1110, the instruction alone 2090); head_dim 64, five prompts of up to 1500 tokens,
// f16: 61 us, of which 20 000 cycles (10 us) per piece go to its start and end.  The f32 kernel
// of head_dim 128 spills 37 vector registers, the others none.
//
// Keys that no row sees are stored as zeros and masked; where V holds an infinity or NaN, which 0
// times a weight would not keep out, or 2^35 and more under scaling, the piece is computed again
// key by key (slow_rows).
//
// Caches of 8-bit integers (E = int8_t): codes are exact in f16 and take one piece; K's scale of a block joins the
// scores, V's, 2^(e + f) with e whole and 0 <= f < 1, the exponent: a weight is 2^(s + f + (e - R)), R a maximum of
// s + e, and e - R comes first, so that nothing that counts is rounded at the size of e (2^-19 where that is 50).
// Scales lie in the lanes of a wave, 64 blocks of the cache at a time, and are read from there.  2048 rows of 32
// heads behind 8192 keys: 581 us, 530 TFLOP/s of attention, 1060 of f16 products, matrix pipe busy in 47 % of the
// cycles, vector instructions issued in 48 %; five prompts of up to 1500 tokens, head_dim 64: 69 us, waves waiting (at
// barriers, and for a piece's start) for 36 % of their time.
#include "hy_device.hpp"
#include "hy_int8.hpp"
#include "hy_lds.hpp"
#include "hy_paged.hpp"
#include "hy_paged_part.hpp"
#include "hy_paged_split.hpp"

namespace hy {

constexpr int PM_WAVES = 8, PM_THREADS = WAVE * PM_WAVES, PM_M = PM_TILE;
static_assert(PM_M == 32 * PM_WAVES && PM_WORKERS % 8 == 0, "32 rows per wave, whole XCDs");
constexpr int PM_UP = 14;   // q's and K's largest elements go to [2^14, 2^15)
constexpr int PM_VUP = 13;  // V's to [2^13, 2^14)
constexpr int PM_ELO = -60, PM_EHI = 34;  // exponents that V's rows are scaled by
// The running maximum R that weights are relative to is left behind while a block does not pass
// it by more than PM_LAG: weights are up to 2^PM_LAG, and the sums are rescaled once or twice
// per row instead of at every new maximum.  Weights carry a factor 2^PM_WUP.
constexpr float PM_LAG = 8.0f;
constexpr int PM_WUP = 6;

__device__ __forceinline__ v16f_t mfma_f16(v4i_t a, v4i_t b, v16f_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h16_t, a), __builtin_bit_cast(v8h16_t, b), c, 0,
                                                  0, 0);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126..127
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
// exponent of the power of two at or below a magnitude (as f32 bits), not below lo
__device__ __forceinline__ int exponent(uint32_t magnitude, int lo) {
    return min(max((int)(magnitude >> 23) - 127, lo), 127);
}

template <class E, int HD>
struct PmLds {
    static constexpr int KP = sizeof(E) == 4 ? 2 : 1;  // pieces of K and V
    // K: per piece HD / 8 chunks (8 dims) of 32 keys x 16 bytes; 32 bytes between chunks put the
    // chunks that a wave stores at once on different banks
    static constexpr int CHUNK_K = 32 * 16 + 32, PIECE_K = HD / 8 * CHUNK_K, BUF_K = KP * PIECE_K;
    // V: per piece 4 chunks (2 c + h: keys 16 c + 4 h .. + 3 and 16 c + 8 + 4 h .. + 3) of HD dims
    // x 16 bytes, even dims before odd ones
    static constexpr int CHUNK_V = HD * 16, PIECE_V = 4 * CHUNK_V, BUF_V = KP * PIECE_V;
    static constexpr int OFF_V = 2 * BUF_K, BYTES = OFF_V + 2 * BUF_V;
};

template <class E, int HD>
__global__ __launch_bounds__(PM_THREADS, 2) void paged_many_kernel(PagedAttnArgs a, PartShape ps) {
    using L = PmLds<E, HD>;
    constexpr bool I8 = std::is_same<E, int8_t>::value, SCALED = !std::is_same<E, _Float16>::value;
    constexpr int KP = L::KP;
    constexpr int NC = HD / 16, ND = HD / 32;
    constexpr int KL = HD / 8;  // threads per key of K
    constexpr int RING = KP == 2 ? 2 : 3;  // operands read ahead of the products (registers allowing)
    __shared__ __attribute__((aligned(1024))) uint8_t lds[L::BYTES];
    __shared__ __attribute__((aligned(16))) float k_fac[2][I8 ? 1 : 32], v_exp[2][I8 ? 1 : 32], v_inv[2][I8 ? 1 : 32];
    __shared__ v4f_t i8_fac[2][I8 ? 8 : 1];  // of four keys: K's scale, V's e, reciprocal and f
    __shared__ int odd_s;  // V of this piece that the scaled products do not take
    __shared__ int last_s[PM_WAVES];
    __shared__ PartSums<PM_THREADS> sums;
    const int tid = threadIdx.x, lane = tid % WAVE, lr = lane % 32, h = lane / 32;
    const int wv = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int64_t total = part_sums(a, ps, sums);
    const int64_t stretch = part_stretch(ps, total);
    // neighbouring stretches, which share kv heads, on one XCD (work groups go round the XCDs)
    const int per_xcd = ps.workers / 8, worker = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
    int64_t x = worker * stretch;
    const int64_t x_end = min(x + stretch, total);
    const int G = ps.G, pmask = (1 << a.c.shift) - 1;

    PartJob job{};
    while (x < x_end) {
        const PartItem it = part_find(a, ps, sums, x);
        int p0, p1;
        if (!part_piece(ps, it, x, x_end, p0, p1)) continue;
        const int kv = it.q.kv;
        const int n_live = min(it.q.n * G - it.tile * PM_M, PM_M);
        // this lane's row (the last one again past the end) and the keys it sees
        const int tok0 = part_quotient(it.tile * PM_M, G);
        const int my = 32 * wv + lr, rho = it.tile * PM_M + min(my, n_live - 1) - tok0 * G, tok1 = part_div(rho, G);
        const int tok = tok0 + tok1, row = it.q.start + tok, head = it.g * G + rho - tok1 * G;
        const int end = a.seen ? min(a.seen[row], kv) : kv - it.q.n + tok + 1;
        int last = end, first = end;  // the most and the fewest keys that a row of the wave sees
        if (a.seen) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                last = max(last, shfl_xor(last, d));
                first = min(first, shfl_xor(first, d));
            }
        } else {  // the last row's (in all rows order), the first row's
            last = __builtin_amdgcn_readlane(end, 31);
        }
        last = 32 * wv < n_live ? max(uniform(last), 0) : 0;
        first = uniform(first);
        if (lane == 0) last_s[wv] = last;
        if (tid == 0) odd_s = 0;
        __syncthreads();
        int tile_last = 0;
#pragma unroll
        for (int w = 0; w < PM_WAVES; w++) tile_last = max(tile_last, last_s[w]);
        tile_last = __builtin_amdgcn_readfirstlane(tile_last);
        const int blocks = (tile_last + 31) / 32;
        const int kb0 = part_block(p0, it.len, blocks), kb1 = part_block(p1, it.len, blocks);
        const int my_kb1 = min((last + 31) / 32, kb1);
        job = part_job(ps, it, p0, p1, stretch, n_live);
        const int slot_id = p0 == 0 && p1 == it.len ? -1 : 2 * worker + (p0 == 0 ? 1 : 0);  // -1: all of it is here

        // ---- loads and stores of blocks
        // Block table: where the pages of 64 entries start, in the lanes, and of the next 64: a
        // block's page is a lane read away (an entry fetched per block was waited for with all
        // loads before it: 2 us a block).  Addresses are a scalar base and a 32-bit lane offset.
        const int* const trow = a.table + (int64_t)it.r * a.max_pages;
        const int n_tab = (kv + pmask) >> a.c.shift;
        bool bad = false;  // an entry that names no page; its keys are read from page 0 and masked
        auto page_ok = [&](int key) {
            const int p = key >> a.c.shift;
            if (p >= n_tab) return false;
            const int e = trow[p];
            return e >= 0 && e < a.c.n_pages;
        };
        auto entry = [&](int seg) { return trow[min(seg * 64 + lane, max(n_tab - 1, 0))]; };
        auto page_at = [&](int seg, int e) {
            const bool there = seg * 64 + lane < n_tab, ok = e >= 0 && e < a.c.n_pages;
            bad |= (bool)__any(there && !ok);
            return there && ok ? e * a.c.page_stride : 0;
        };
        int seg = (kb0 * 32) >> (a.c.shift + 6);
        const int e1 = entry(seg), e2 = entry(seg + 1);
        __builtin_amdgcn_sched_barrier(0);
        // q's dims 16 c + 8 h .. + 7: on their way before the pages are known
        const float* const qp = a.q + ((int64_t)row * a.nh + head) * HD + 8 * h;
        v4f_t q[NC][2];
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int u = 0; u < 2; u++) q[c][u] = *reinterpret_cast<const v4f_t*>(qp + 16 * c + 4 * u);
        __builtin_amdgcn_sched_barrier(0);
        int64_t tab = page_at(seg, e1), tab2 = page_at(seg + 1, e2);
        auto lane64 = [](int64_t v, int l) {
            return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) |
                             (uint32_t)__builtin_amdgcn_readlane((int)v, l));
        };
        // scales of an 8-bit cache: those of 64 blocks of positions in the lanes, the next 64's, and the pages of
        // the 64 behind them (a load per block of keys cost 10 % of a prompt)
        auto scale_page = [&](int sseg) {
            return trow[min((sseg * 64 + lane) >> (a.c.shift - a.bshift), max(n_tab - 1, 0))];
        };
        auto scale_from = [&](const float* scales, int sseg, int e) {
            const int64_t p = e >= 0 && e < a.c.n_pages ? e : 0;
            const int per_page = 1 << (a.c.shift - a.bshift);
            return scales[(p * a.c.nkv + it.g) * per_page + ((sseg * 64 + lane) & (per_page - 1))];
        };
        int sseg = 0, sp = 0;
        float ks = 0.0f, ks2 = 0.0f, vs2 = 0.0f;
        // V's as the two parts of their logarithms and their reciprocals (to 2^-23 of the keys' weights in the sum);
        // below the range the lowest e and values of 0, an infinity as NaN
        float v_e = 0.0f, v_f = 0.0f, v_rcp = 0.0f;
        auto of_v = [&](float v) {
            v = v < pow2(PM_ELO) ? pow2(PM_ELO) : fmaf(v, 0.0f, v);
            const int e = min(exponent(__float_as_uint(v), PM_ELO), 126);  // 2^-e is normal
            const float m = v * pow2(-e);
            v_e = (float)e;
            v_f = __builtin_amdgcn_logf(m);
            v_rcp = __builtin_amdgcn_rcpf(m) * pow2(-e);
        };
        if constexpr (I8) {
            sseg = (kb0 * 32) >> (a.bshift + 6);
            const int pg = scale_page(sseg), pg2 = scale_page(sseg + 1);
            sp = scale_page(sseg + 2);
            ks = scale_from(a.ks, sseg, pg);
            of_v(scale_from(a.vs, sseg, pg));
            ks2 = scale_from(a.ks, sseg + 1, pg2), vs2 = scale_from(a.vs, sseg + 1, pg2);
        }
        auto lane_f = [](float v, int l) {
            return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l));
        };
        auto cell_of = [&](int key) {  // wave-uniform; keys up to 64 pages past those of load_v
            const int p = (key >> a.c.shift) - seg * 64;
            const int64_t page = p < 64 ? lane64(tab, p) : lane64(tab2, p - 64);
            return page + ((key & ~31) & pmask) * a.c.token_stride;
        };
        const E* const kg = static_cast<const E*>(a.c.k) + it.g * a.c.head_stride;
        const E* const vg = static_cast<const E*>(a.c.v) + it.g * a.c.head_stride;
        constexpr int KPW = WAVE / KL;  // keys of K per wave
        // head_dim 64: every vector is loaded twice (loads under a condition could not be counted, and
        // every wait would wait for all of them), and stored once
        const bool k_mine = HD == 128 || tid < 32 * KL, v_mine = HD == 128 || lane < HD / 2;
        const int k_key = tid / KL % 32, k_ch = tid % KL;
        const uint32_t in_page = min(pmask, 31), ts = (uint32_t)a.c.token_stride;
        const uint32_t k_off = ((k_key & in_page) * ts + 8 * k_ch) * sizeof(E);
        const uint32_t v_off = (((4 * wv) & in_page) * ts + 2 * (lane % (HD / 2))) * sizeof(E);
        uint8_t* const k_dst = lds + k_ch * L::CHUNK_K + k_key * 16;
        uint8_t* const v_dst = lds + L::OFF_V + (2 * (wv / 4) + wv % 2) * L::CHUNK_V + lane * 16 + 8 * (wv / 2 % 2);
        typedef typename std::conditional<I8, uint2, v4i_t>::type krow_t;
        krow_t kx[KP];
        float k_scale = 0.0f, v_ex = 0.0f, v_fr = 0.0f, v_in = 0.0f;
        typedef typename std::conditional<KP == 2, uint2, typename std::conditional<I8, uint16_t, uint32_t>::type>::type vrow_t;
        vrow_t vx[4];
        uint32_t v_big = 0;  // the largest magnitude of V's: whether one was infinite, no number, or past PM_EHI
        auto load_k = [&](int kb) {
            const char* const p = reinterpret_cast<const char*>(kg + cell_of(kb * 32 + (wv * KPW) % 32));
#pragma unroll
            for (int u = 0; u < KP; u++) kx[u] = *reinterpret_cast<const krow_t*>(p + k_off + 16 * u);
            if constexpr (I8) {  // up to 64 blocks of positions past those of load_v
                const int b = ((kb * 32 + (wv * KPW) % 32) >> a.bshift) - sseg * 64;
                k_scale = lane_f(b < 64 ? ks : ks2, b & 63);
            }
        };
        auto load_v = [&](int kb) {
            const char* const p = reinterpret_cast<const char*>(vg + cell_of(kb * 32 + 4 * wv));
#pragma unroll
            for (int j = 0; j < 4; j++) vx[j] = *reinterpret_cast<const vrow_t*>(p + (v_off + j * ts * sizeof(E)));
            if constexpr (I8) {
                const int b = ((kb * 32 + 4 * wv) >> a.bshift) - sseg * 64;
                v_ex = lane_f(v_e, b);
                v_fr = lane_f(v_f, b);
                v_in = lane_f(v_rcp, b);
            }
            const int s = ((kb + 1) * 32) >> (a.c.shift + 6);  // the next call's
            if (s != seg) {
                seg = s;
                tab = tab2;
                tab2 = page_at(seg + 1, entry(seg + 1));
            }
            if constexpr (I8) {
                const int t = ((kb + 1) * 32) >> (a.bshift + 6);
                if (t != sseg) {
                    sseg = t;
                    ks = ks2;
                    of_v(vs2);
                    ks2 = scale_from(a.ks, sseg + 1, sp), vs2 = scale_from(a.vs, sseg + 1, sp);
                    sp = scale_page(sseg + 2);
                }
            }
        };
        // block kb, r = kb % 2
        auto put_k = [&](int r) {
            uint8_t* const d = k_dst + r * L::BUF_K;
            // a key with an infinity makes NaN of every score (a row's q with one does by its pieces):
            // through its factor, or its element x becomes 0 x + x
            if constexpr (I8) {
                uint32_t w0, w1, w2, w3;
                i8_to_f16(kx[0].x, w0, w1);
                i8_to_f16(kx[0].y, w2, w3);
                if (k_mine) {
                    *reinterpret_cast<v4i_t*>(d) = v4i_t{(int)w0, (int)w1, (int)w2, (int)w3};
                    if (k_ch == 0 && k_key % 4 == 0) i8_fac[r][k_key / 4][0] = fmaf(k_scale, 0.0f, k_scale);
                }
            } else if constexpr (!SCALED) {
                const v8h16_t x = __builtin_bit_cast(v8h16_t, kx[0]);
                const v8h16_t y = __builtin_elementwise_fma(x, (v8h16_t)((_Float16)0), x);
                if (k_mine) *reinterpret_cast<v8h16_t*>(d) = y;
            } else {
                float f[8];
                uint32_t big = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    uint32_t w;
                    if constexpr (KP == 2)
                        w = (uint32_t)kx[j / 4][j % 4];
                    else
                        w = j % 2 ? (uint32_t)kx[0][j / 2] & 0xffff0000u : (uint32_t)kx[0][j / 2] << 16;
                    f[j] = __uint_as_float(w);
                    big = max(big, w & 0x7fffffffu);
                }
                big = dpp_umax<0xB1>(big);   // the key's KL neighbouring lanes
                big = dpp_umax<0x4E>(big);
                big = dpp_umax<0x141>(big);
                if constexpr (KL == 16) big = dpp_umax<0x140>(big);
                const int e = exponent(big, -100);
                const float up = pow2(PM_UP - e);
                v4i_t hi, lo;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w0, w1;
                    if constexpr (KP == 2) {
                        split_f16(f[2 * j] * up, f[2 * j + 1] * up, w0, w1);
                        lo[j] = (int)w1;
                    } else {
                        w0 = pk_f16(f[2 * j] * up, f[2 * j + 1] * up);
                    }
                    hi[j] = (int)w0;
                }
                if (k_mine) {
                    *reinterpret_cast<v4i_t*>(d) = hi;
                    if constexpr (KP == 2) *reinterpret_cast<v4i_t*>(d + L::PIECE_K) = lo;
                    if (k_ch == 0) k_fac[r][k_key] = big < 0x7f800000u ? pow2(e - PM_UP) : __builtin_nanf("");
                }
            }
        };
        auto put_v = [&](int kb, int r) {
            uint8_t* const d = v_dst + r * L::BUF_V;
            const int key0 = kb * 32 + 4 * wv;
            if constexpr (I8) {
                const bool tiny = v_ex + v_fr == (float)PM_ELO;  // the same for the wave: values of 0
                if (v_mine) {
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const uint2 w = make_uint2(i8_pair(vx[0], vx[1], n), i8_pair(vx[2], vx[3], n));
                        *reinterpret_cast<uint2*>(d + n * (HD / 2) * 16) = make_uint2(tiny ? 0 : w.x, tiny ? 0 : w.y);
                    }
                }
                if (lane == 0) {
                    i8_fac[r][wv][1] = v_ex;
                    i8_fac[r][wv][2] = v_in;
                    i8_fac[r][wv][3] = v_fr;
                }
                return;
            }
            if (bad || key0 + 4 > kv) {  // wave-uniform: keys that are not there are zeros
                const bool ok = page_ok(key0);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (!ok || key0 + j >= kv) vx[j] = vrow_t{};
            }
            float f[4][2];
            uint32_t big[4];
            if constexpr (SCALED && !I8) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w0, w1;
                    if constexpr (KP == 2) {
                        w0 = vx[j].x;
                        w1 = vx[j].y;
                    } else {
                        w0 = vx[j] << 16;
                        w1 = vx[j] & 0xffff0000u;
                    }
                    big[j] = v_mine ? max(w0 & 0x7fffffffu, w1 & 0x7fffffffu) : 0;
                    f[j][0] = __uint_as_float(w0);
                    f[j][1] = __uint_as_float(w1);
                }
            }
            if constexpr (SCALED && !I8) {
                // row j's largest: lanes of equal l % 4 share one row from the second step on
                uint32_t b0 = lane & 1 ? big[1] : big[0], g0 = lane & 1 ? big[0] : big[1];
                uint32_t b1 = lane & 1 ? big[3] : big[2], g1 = lane & 1 ? big[2] : big[3];
                b0 = max(b0, dpp_u<0xB1>(g0));
                b1 = max(b1, dpp_u<0xB1>(g1));
                uint32_t b = lane & 2 ? b1 : b0;
                const uint32_t g = lane & 2 ? b0 : b1;
                b = max(b, dpp_u<0x4E>(g));   // lane l: row l % 4 of its quad
                b = dpp_umax<0x124>(b);       // rotations by 4 and 8 in 16 lanes
                b = dpp_umax<0x128>(b);
                const auto umax = [](uint32_t p, uint32_t q) { return max(p, q); };
                b = with_half(with_row(b, umax), umax);
                v_big = max(v_big, b);
                const int e = min(exponent(b, PM_ELO), PM_EHI);
                if (lane < 4) {
                    v_exp[r][4 * wv + lane] = (float)e;
                    v_inv[r][4 * wv + lane] = pow2(-e);
                }
                const uint32_t up = __float_as_uint(pow2(PM_VUP - e));
                const float u0 = __uint_as_float(dpp_u<0x00>(up)), u1 = __uint_as_float(dpp_u<0x55>(up));
                const float u2 = __uint_as_float(dpp_u<0xAA>(up)), u3 = __uint_as_float(dpp_u<0xFF>(up));
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    uint2 hi, lo;
                    if constexpr (KP == 2) {
                        split_f16(f[0][n] * u0, f[1][n] * u1, hi.x, lo.x);
                        split_f16(f[2][n] * u2, f[3][n] * u3, hi.y, lo.y);
                    } else {
                        hi.x = pk_f16(f[0][n] * u0, f[1][n] * u1);
                        hi.y = pk_f16(f[2][n] * u2, f[3][n] * u3);
                    }
                    if (v_mine) {
                        *reinterpret_cast<uint2*>(d + n * (HD / 2) * 16) = hi;
                        if constexpr (KP == 2) *reinterpret_cast<uint2*>(d + n * (HD / 2) * 16 + L::PIECE_V) = lo;
                    }
                }
            } else if constexpr (!I8) {
                typedef unsigned short v2u16_t __attribute__((ext_vector_type(2)));
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v_big = __builtin_bit_cast(
                        uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u16_t, v_big),
                                                            __builtin_bit_cast(v2u16_t, vx[j] & 0x7fff7fffu)));
                if (v_mine) {
#pragma unroll
                    for (int n = 0; n < 2; n++)
                        *reinterpret_cast<uint2*>(d + n * (HD / 2) * 16) =
                            make_uint2(__builtin_amdgcn_perm(vx[1], vx[0], n ? 0x07060302u : 0x05040100u),
                                       __builtin_amdgcn_perm(vx[3], vx[2], n ? 0x07060302u : 0x05040100u));
                }
            }
        };

        v16f_t o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = v16f_t{};
        float m_run = -INFINITY, l_run = 0.0f;
        if (kb0 < kb1) {
            load_k(kb0);
            load_v(kb0);
        }

        // ---- q: its pieces, times scale * log2(e) (scores in the base-2 domain) and the row's power
        // of two
        v4i_t qf[NC][2];
        float unscale;
        {
            const float qscale = a.scale * 1.4426950408889634f;
            uint32_t big = 0;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    q[c][u] *= qscale;
#pragma unroll
                    for (int j = 0; j < 4; j++) big = max(big, __float_as_uint(q[c][u][j]) & 0x7fffffffu);
                }
            big = with_half(big, [](uint32_t p, uint32_t q) { return max(p, q); });
            const int e = exponent(big, -100);
            const float up = pow2(PM_UP - e);
            unscale = pow2(e - PM_UP);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w0, w1;
                    split_f16(q[c][j / 2][2 * (j % 2)] * up, q[c][j / 2][2 * (j % 2) + 1] * up, w0, w1);
                    qf[c][0][j] = (int)w0;
                    qf[c][1][j] = (int)w1;
                }
        }

        v4i_t pf[2][2];  // the weights' pieces, keys 16 c .. in step c
        // scores of block kb and its weights' pieces
        auto scores = [&](int kb, int r) {
            const uint8_t* const kb_ = lds + r * L::BUF_K + h * L::CHUNK_K + lr * 16;
            v4i_t kf[RING][KP];
            auto read = [&](int c) {
#pragma unroll
                for (int q = 0; q < KP; q++)
                    kf[c % RING][q] = *reinterpret_cast<const v4i_t*>(kb_ + q * L::PIECE_K + 2 * c * L::CHUNK_K);
            };
            v16f_t s = v16f_t{};
#pragma unroll
            for (int c = 0; c < RING - 1; c++) read(c);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                if (c + RING - 1 < NC) read(c + RING - 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (KP == 2) s = mfma_f16(kf[c % RING][1], qf[c][0], s);
                s = mfma_f16(kf[c % RING][0], qf[c][1], s);
                s = mfma_f16(kf[c % RING][0], qf[c][0], s);
                __builtin_amdgcn_sched_barrier(0);
            }
            v4f_t inv[4];
            float i8_k[4], i8_v[4], i8_f[4];  // of an 8-bit cache: K's factor, V's e and f
#pragma unroll
            for (int u = 0; u < 4; u++) {
                v4f_t fac, ex;
                if constexpr (I8) {
                    const v4f_t f = i8_fac[r][2 * u + h];
                    i8_k[u] = f[0] * unscale;
                    i8_v[u] = f[1];
                    i8_f[u] = f[3];
                    inv[u][0] = f[2];
                    continue;
                } else if constexpr (SCALED) {
                    fac = *reinterpret_cast<const v4f_t*>(&k_fac[r][8 * u + 4 * h]);
                    ex = *reinterpret_cast<const v4f_t*>(&v_exp[r][8 * u + 4 * h]);
                    inv[u] = *reinterpret_cast<const v4f_t*>(&v_inv[r][8 * u + 4 * h]);
                }
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    float t = s[4 * u + v];
                    if constexpr (SCALED) t = fmaf(t, fac[v] * unscale, ex[v]);
                    s[4 * u + v] = t;
                }
            }
            if (bad || kb * 32 + 32 > first) {  // wave-uniform
                asm volatile("");               // a branch, not 80 operations more in every block
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int key = kb * 32 + 8 * u + 4 * h;
                    const bool ok = !bad || page_ok(key);
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        if (!ok || key + v >= end) s[4 * u + v] = -INFINITY;
                    if constexpr (I8) {
                        // four keys of one block: what its scales are where this row sees none of them does not
                        // matter, and a NaN is the row's where it sees one; -inf times a scale of 0 would be NaN
                        const bool sees = ok && key < end;
                        i8_k[u] = !sees || i8_k[u] < 0x1p-126f ? 0x1p-126f : i8_k[u];
                        i8_f[u] = sees ? i8_f[u] : 0.0f;
                        inv[u][0] = sees ? inv[u][0] : 0.0f;
                    }
                }
            }
            float big;
            if constexpr (I8) {  // scales are not negative: a group's largest score has its largest s + e
                big = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float m = fmaxf(fmaxf(s[4 * u], s[4 * u + 1]), fmaxf(s[4 * u + 2], s[4 * u + 3]));
                    big = fmaxf(big, fmaf(m, i8_k[u], i8_v[u]));
                }
            } else {
                big = s[0];
#pragma unroll
                for (int v = 1; v < 16; v++) big = fmaxf(big, s[v]);
            }
            if constexpr (!SCALED) big *= unscale;
            if (__any(big > m_run + PM_LAG)) {
                big = fmax_half(big);
                const float m = big > m_run + PM_LAG ? big : m_run;
                const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m);
                m_run = m;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= alpha;  // all blocks before kb are in it
            }
            const float ref = m_run == -INFINITY ? 0.0f : m_run;
            const float up = ref - (float)PM_WUP;
            if constexpr (I8) {
#pragma unroll
                for (int u = 0; u < 4; u++) i8_v[u] = i8_f[u] + (i8_v[u] - up);
            }
#pragma unroll
            for (int v = 0; v < 16; v++) {  // l_run: of this lane's keys; joined behind the loop
                if constexpr (I8) {
                    s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], i8_k[v / 4], i8_v[v / 4]));
                    l_run = fmaf(s[v], inv[v / 4][0], l_run);
                } else if constexpr (SCALED) {
                    s[v] = __builtin_amdgcn_exp2f(s[v] - up);
                    l_run = fmaf(s[v], inv[v / 4][v % 4], l_run);
                } else {
                    s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], unscale, -up));
                    l_run += s[v];
                }
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t w0, w1;
                    split_f16(s[8 * c + 2 * j], s[8 * c + 2 * j + 1], w0, w1);
                    pf[c][0][j] = (int)w0;
                    pf[c][1][j] = (int)w1;
                }
        };
        auto values = [&](int r) {
            const uint8_t* const vb = lds + L::OFF_V + r * L::BUF_V + h * L::CHUNK_V + lr * 16;
            v4i_t vf[RING][KP];
            auto read = [&](int i) {  // slots 32 (i % ND) .. of step i / ND
#pragma unroll
                for (int q = 0; q < KP; q++)
                    vf[i % RING][q] = *reinterpret_cast<const v4i_t*>(vb + q * L::PIECE_V + 2 * (i / ND) * L::CHUNK_V +
                                                                   512 * (i % ND));
            };
#pragma unroll
            for (int i = 0; i < RING - 1; i++) read(i);
#pragma unroll
            for (int i = 0; i < 2 * ND; i++) {
                if (i + RING - 1 < 2 * ND) read(i + RING - 1);
                __builtin_amdgcn_sched_barrier(0);
                v16f_t& t = o[i % ND];
                if constexpr (KP == 2) t = mfma_f16(vf[i % RING][1], pf[i / ND][0], t);
                t = mfma_f16(vf[i % RING][0], pf[i / ND][1], t);
                t = mfma_f16(vf[i % RING][0], pf[i / ND][0], t);
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        if (kb0 < kb1) {
            put_k(kb0 & 1);
            load_k(kb0 + 1);
        }
        for (int kb = kb0; kb < kb1; kb++) {
            const int r = kb & 1;
            put_v(kb, r);
            load_v(kb + 1);
            __syncthreads();  // block kb is in LDS, block kb - 1 read out
            if (kb < my_kb1) scores(kb, r);
            if (kb + 1 < kb1) put_k(r ^ 1);
            load_k(kb + 2);
            if (kb < my_kb1) values(r);
        }
        l_run = fadd_half(l_run);

        // l carries the weights' factor too, scaled values have one of their own
        float down = SCALED && !I8 ? pow2(-PM_VUP) : 1.0f;
        if constexpr (I8) {  // codes are finite, whatever they are
        } else if constexpr (SCALED)
            v_big = v_big >= (uint32_t)(127 + PM_EHI + 1) << 23;
        else
            v_big = (v_big & 0xffffu) >= 0x7c00u || v_big >= 0x7c000000u;
        if constexpr (!I8) {
            if (__any(v_big != 0)) odd_s = 1;
            __syncthreads();
            if (odd_s) {  // again, key by key
                slow_rows<E, HD, 2>(
                    a, trow, kv, kb0 * 32, my_kb1 * 32, end, a.q + ((int64_t)row * a.nh + head) * HD, kg, vg,
                    [&](int i) { return 2 * (32 * (i / 16 % (ND / 2)) + 8 * (i % 16 / 4) + 4 * h + i % 4) + i / (8 * ND); },
                    [&](int i, float v) { o[i / 16][i % 16] = v; }, [&](int i) { return o[i / 16][i % 16]; }, m_run, l_run);
                // as the other pieces of its item; in the reference, the sums of large values have no room for it
                down = 1.0f;
                m_run += (float)PM_WUP;
            }
        }
        if (my < n_live) {
            float* dst;
            float f = down;
            if (slot_id < 0) {
                dst = a.out + ((int64_t)row * a.nh + head) * HD;
                f = l_run == 0.0f ? 0.0f : down / l_run;
            } else {
                float* const slot = a.ws + ps.ws + (size_t)slot_id * part_slot_floats(PM_M, HD);
                dst = slot + 32 * wv * HD + 4 * lane;  // part_at
                if (h == 0) {
                    slot[PM_M * HD + my] = m_run;
                    slot[PM_M * (HD + 1) + my] = l_run;
                }
            }
#pragma unroll
            for (int d = 0; d < ND / 2; d++)
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    float* const p = dst + (slot_id < 0 ? 2 * (32 * d + 8 * u + 4 * h) : 512 * (4 * d + u));
                    const int next = slot_id < 0 ? 4 : 256;
#pragma unroll
                    for (int v = 0; v < 2; v++)
                        *reinterpret_cast<v4f_t*>(p + v * next) =
                            (v4f_t){o[d][4 * u + 2 * v], o[d + ND / 2][4 * u + 2 * v], o[d][4 * u + 2 * v + 1],
                                    o[d + ND / 2][4 * u + 2 * v + 1]} *
                            f;
                }
        }
        __syncthreads();  // last_s and the buffers are free
    }
    if (tid == 0) part_jobs(a, ps, HD)[worker] = job;
}

template <class E>
static void launch(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s) {
    if (a.c.hd == 128)
        hipLaunchKernelGGL((paged_many_kernel<E, 128>), dim3(ps.workers), dim3(PM_THREADS), 0, s, a, ps);
    else
        hipLaunchKernelGGL((paged_many_kernel<E, 64>), dim3(ps.workers), dim3(PM_THREADS), 0, s, a, ps);
}

void launch_paged_many(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s) {
    if (a.c.type == HY_TYPE_F32)
        launch<float>(a, ps, s);
    else if (a.c.type == HY_TYPE_F16)
        launch<_Float16>(a, ps, s);
    else if (a.c.type == HY_TYPE_I8)
        launch<int8_t>(a, ps, s);
    else
        launch<__bf16>(a, ps, s);
}

}  // namespace hy
