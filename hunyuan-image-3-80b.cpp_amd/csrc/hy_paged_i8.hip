// hy_paged_i8.hip -- the write into a paged cache of 8-bit integers (hy_rope_qknorm_paged_i8): rotary
// embedding and QK-norm, queries to [rows][nh][hd], keys and values to codes with a scale per block of
// positions and head.
//
// A scale belongs to all rows that a call brings into its block, so the unit of work is a run (rows
// whose slots follow one another inside a block) times a kv head, a work group each, which the
// run's first row names.  HD / 4 lanes share a row, 4 dims each; a work group holds 16 rows, or 32
// where blocks are longer (1 to 4 per lane); longer runs are gone through twice (largest magnitude, then codes).
// A key is rotated and normed in 64 bits and rounded to f32 once: a value next to the border
// between two codes would otherwise fall by the order of the sum, and a step is 2^-7 of the largest.
//
// 32 heads and 8 kv heads of 128: 4096 rows 41 us, 4.4 TB/s, bound by memory and, beside it, the 64-bit
// rotation and norm of keys (a fifth of the rows' values); 5 rows 6 us, a chain of dependent reads (slots,
// table entries and rows, the block's scale and codes, two barriers).
#include "hy_device.hpp"
#include "hy_int8.hpp"
#include "hy_paged_rotary.hpp"

namespace hy {

typedef double v4d_t __attribute__((ext_vector_type(4)));

// sine and cosine of `turn` turns, to 2^-50: whole quarters off, then the series of the angle |t| <= pi / 4
// (remainders (pi / 4)^17 / 17! = 4.6e-17, (pi / 4)^18 / 18! = 2.0e-18)
__device__ __forceinline__ void sincos_turn(double turn, double& sn, double& cs) {
    const double n = rint(4.0 * turn), t = fma(-0.25, n, turn) * 6.283185307179586476925, z = t * t;
    double s = 1.0 / 1307674368000.0;  // 15!, with alternating signs
    s = fma(-s, z, 1.0 / 6227020800.0);
    s = fma(-s, z, 1.0 / 39916800.0);
    s = fma(-s, z, 1.0 / 362880.0);
    s = fma(-s, z, 1.0 / 5040.0);
    s = fma(-s, z, 1.0 / 120.0);
    s = fma(-s, z, 1.0 / 6.0);
    s = t * fma(-s, z, 1.0);
    double c = 1.0 / 20922789888000.0;  // 16!
    c = fma(-c, z, 1.0 / 87178291200.0);
    c = fma(-c, z, 1.0 / 479001600.0);
    c = fma(-c, z, 1.0 / 3628800.0);
    c = fma(-c, z, 1.0 / 40320.0);
    c = fma(-c, z, 1.0 / 720.0);
    c = fma(-c, z, 1.0 / 24.0);
    c = fma(-c, z, 0.5);
    c = fma(-c, z, 1.0);
    const int q = (int)n;
    const double a = q & 1 ? c : s, b = q & 1 ? s : c;
    sn = q & 2 ? -a : a;
    cs = (q + 1) & 2 ? -b : b;
}

template <int CTRL>
__device__ __forceinline__ double add_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// over the lanes of a head
template <int HD>
__device__ __forceinline__ double head_sum(double v) {
    v = add_dpp<0x128>(v);
    v = add_dpp<0x124>(v);
    v = add_dpp<0x122>(v);
    v = add_dpp<0x121>(v);
    if constexpr (HD == 128) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
        const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
        v = __builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]) + __builtin_bit_cast(double, (uint64_t)h[1] << 32 | l[1]);
    }
    return v;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}

constexpr int PQ_STEPS = 4;  // of query heads
constexpr int PW_THREADS = 256;
// Rows whose runs a work group goes through: one, or past PW_ALONE rows PW_ROWS, so that a prompt does not
// launch a work group for each of its rows (4096 rows in blocks of 16: by 8 rows 59 us, 16 41, 32 44).
constexpr int PW_ROWS = 16, PW_ALONE = 512;

struct AppendI8 {
    PagedAppendArgs a;
    float* ks;
    float* vs;
    int bshift;
    int rows;        // of a work group that writes the cache
    int64_t blocks;  // work groups
    double q_share;  // of them that take queries (and half a one, so that rounding loses none)
};

__device__ __forceinline__ bool row_ok(const PagedAppendArgs& a, int slot, int pos) {
    return slot >= 0 && (slot >> a.c.shift) < a.c.n_pages && !(a.rotate == 2 && (pos < 0 || pos >= a.n_pos));
}

// queries: as paged_append_kernel, a row per wave
template <int HD>
__device__ __forceinline__ void append_queries(const PagedAppendArgs& a, int64_t b) {
    constexpr int LPU = HD / 4, UNITS = PQ_STEPS * WAVE / LPU;
    const int units = a.nh + 2 * a.c.nkv, groups = (a.nh + UNITS - 1) / UNITS;
    const int t = (int)(b / groups) * 4 + (int)threadIdx.x / WAVE, u0 = (int)(b % groups) * UNITS;
    if (t >= a.n_rows) return;
    const int l = threadIdx.x % WAVE, d = 4 * (l % LPU);
    const float* const row = a.qkv + (int64_t)t * units * HD + d;
    v4f_t x[PQ_STEPS];
#pragma unroll
    for (int s = 0; s < PQ_STEPS; s++)
        x[s] = *reinterpret_cast<const v4f_t*>(row + (int64_t)min(u0 + (s * WAVE + l) / LPU, a.nh - 1) * HD);
    const int slot = a.slots[t], pos = a.positions[t];
    const auto clear = [&](float* to) {
#pragma unroll
        for (int s = 0; s < PQ_STEPS; s++) {
            const int u = u0 + (s * WAVE + l) / LPU;
            if (u < a.nh) *reinterpret_cast<v4f_t*>(to + ((int64_t)t * a.nh + u) * HD + d) = v4f_t{};
        }
    };
    if (a.merged && t >= a.row_end[0]) clear(a.merged);
    if (!row_ok(a, slot, pos)) {
        if (a.merged) clear(a.q);
        return;
    }
    float cs[2] = {1.0f, 1.0f}, sn[2] = {0.0f, 0.0f};
    if (a.rotate == 1) {
#pragma unroll
        for (int p = 0; p < 2; p++) rope_angle(pos, a.freq[d / 2 + p], sn[p], cs[p]);
    } else if (a.rotate == 2) {
        const v4f_t c = *reinterpret_cast<const v4f_t*>(a.cos_t + (int64_t)pos * HD + d);
        const v4f_t s = *reinterpret_cast<const v4f_t*>(a.sin_t + (int64_t)pos * HD + d);
        cs[0] = c[0], cs[1] = c[2], sn[0] = s[0], sn[1] = s[2];
    }
    const v4f_t one = {1.0f, 1.0f, 1.0f, 1.0f};
    const v4f_t wq = a.q_norm ? *reinterpret_cast<const v4f_t*>(a.q_norm + d) : one;
#pragma unroll
    for (int s = 0; s < PQ_STEPS; s++) {
        const int u = u0 + (s * WAVE + l) / LPU;
        v4f_t y;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            y[2 * p] = fmaf(x[s][2 * p], cs[p], -(x[s][2 * p + 1] * sn[p]));
            y[2 * p + 1] = fmaf(x[s][2 * p], sn[p], x[s][2 * p + 1] * cs[p]);
        }
        const float rms = head_rms<HD>(y, a.eps);
        if (u < a.nh) *reinterpret_cast<v4f_t*>(a.q + ((int64_t)t * a.nh + u) * HD + d) = y * rms * wq;
    }
}

// a key's 4 values of a lane, rotated and normed, as they are quantized
template <int HD>
__device__ __forceinline__ v4f_t norm_key(const PagedAppendArgs& a, v4f_t x, const double (&sn)[2],
                                          const double (&cs)[2], v4f_t w) {
    v4d_t y;
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const double x0 = x[2 * p], x1 = x[2 * p + 1];
        y[2 * p] = fma(x0, cs[p], -(x1 * sn[p]));
        y[2 * p + 1] = fma(x0, sn[p], x1 * cs[p]);
    }
    const double ss = head_sum<HD>((y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]));
    // an estimate (2^-24) and two steps of Newton's
    const double ms = fma(ss, 1.0 / HD, (double)a.eps);
    double e = __builtin_amdgcn_rsq(ms);
    if (ms > 0.0 && ms < (double)INFINITY) {
        e = fma(0.5 * e, fma(-ms * e, e, 1.0), e);
        e = fma(0.5 * e, fma(-ms * e, e, 1.0), e);
    }
    v4f_t z;
#pragma unroll
    for (int j = 0; j < 4; j++) z[j] = (float)(y[j] * e * (double)w[j]);
    return z;
}

// The run of n rows at least that begins with row t, for kv head u.  pos_l: in lane at + i the position of row
// t + i, for the n rows; more: the run may go on behind them.
template <int HD, int STEPS>
__device__ __forceinline__ void append_run(const AppendI8& g, int t, int n, bool more, int pos_l, int at, int u,
                                          uint32_t (&part)[2][PW_THREADS / WAVE]) {
    constexpr int LPU = HD / 4, RPS = PW_THREADS / LPU, HELD = STEPS * RPS;
    const PagedAppendArgs& a = g.a;
    const int tid = threadIdx.x, l = tid % WAVE, d = 4 * (tid % LPU), bmask = (1 << g.bshift) - 1;
    const int units = a.nh + 2 * a.c.nkv;
    const int slot = a.slots[t], off = slot & bmask;
    const int n_lanes = n;
    while (more) {
        const int i = n + l, r = min(t + i, a.n_rows - 1), s = a.slots[r];
        const bool in = t + i < a.n_rows && i <= bmask - off && s == slot + i && row_ok(a, s, a.positions[r]);
        const unsigned long long out = __ballot(!in);
        n += out ? __builtin_ctzll(out) : WAVE;
        more = !out;
    }
    n = __builtin_amdgcn_readfirstlane(n);
    const int page = slot >> a.c.shift, in_page = slot & ((1 << a.c.shift) - 1);
    const int64_t block = (int64_t)page * a.c.page_stride + (int64_t)u * a.c.head_stride +
                          (int64_t)(in_page - off) * a.c.token_stride;
    const int64_t sc = (((int64_t)page * a.c.nkv + u) << (a.c.shift - g.bshift)) + (in_page >> g.bshift);
    // of K, of V
    int8_t* const pool[2] = {static_cast<int8_t*>(a.c.k) + block, static_cast<int8_t*>(a.c.v) + block};
    float* const scale[2] = {g.ks + sc, g.vs + sc};
    const float* const src = a.qkv + (int64_t)t * units * HD + (int64_t)(a.nh + u) * HD + d;
    const v4f_t one = {1.0f, 1.0f, 1.0f, 1.0f};
    const v4f_t w = a.k_norm ? *reinterpret_cast<const v4f_t*>(a.k_norm + d) : one;
    // what the block holds besides, 16 codes per lane: the first rows of it on their way
    constexpr int LPC = HD / 16, CPS = PW_THREADS / LPC;
    const int c = 16 * (tid % LPC), c_row = tid / LPC;
    const auto cell = [&](int x, int i) {
        return reinterpret_cast<v4i_t*>(pool[x] + (int64_t)i * a.c.token_stride + c);
    };
    float old[2] = {0.0f, 0.0f};
    v4i_t held[2] = {};
    if (off) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            old[x] = scale[x][0];
            held[x] = *cell(x, min(c_row, bmask));
        }
    }

    v4f_t y[2][STEPS];
    const auto rows = [&](int i0) {
        int pos[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int i = min(i0 + s * RPS + tid / LPU, n - 1);
            pos[s] = n == n_lanes ? __shfl(pos_l, at + i, WAVE) : a.positions[t + i];
#pragma unroll
            for (int x = 0; x < 2; x++)
                y[x][s] = *reinterpret_cast<const v4f_t*>(src + (int64_t)i * units * HD + x * a.c.nkv * HD);
        }
        v4f_t ct[STEPS], st[STEPS];
        if (a.rotate == 2) {
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                ct[s] = *reinterpret_cast<const v4f_t*>(a.cos_t + (int64_t)pos[s] * HD + d);
                st[s] = *reinterpret_cast<const v4f_t*>(a.sin_t + (int64_t)pos[s] * HD + d);
            }
        }
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            if (i0 + s * RPS >= n) break;  // the same for the work group
            double cs[2] = {1.0, 1.0}, sn[2] = {0.0, 0.0};
            if (a.rotate == 1) {
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const double turn = (double)pos[s] * a.freq[d / 2 + p];
                    sincos_turn(turn - rint(turn), sn[p], cs[p]);
                }
            } else if (a.rotate == 2) {
                cs[0] = ct[s][0], cs[1] = ct[s][2], sn[0] = st[s][0], sn[1] = st[s][2];
            }
            y[0][s] = norm_key<HD>(a, y[0][s], sn, cs, w);
        }
    };
    uint32_t big[2] = {0, 0};
    for (int i0 = 0; i0 < n; i0 += HELD) {
        rows(i0);
#pragma unroll
        for (int s = 0; s < STEPS; s++)
            if (i0 + s * RPS < n) {  // rows past the last are the last again
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int j = 0; j < 4; j++) big[x] = max(big[x], __float_as_uint(y[x][s][j]) & 0x7fffffffu);
            }
    }
    const auto umax = [](uint32_t p, uint32_t q) { return max(p, q); };
#pragma unroll
    for (int x = 0; x < 2; x++) {
        big[x] = dpp_umax<0x128>(big[x]);  // rotations by 8 .. 1 in 16 lanes
        big[x] = dpp_umax<0x124>(big[x]);
        big[x] = dpp_umax<0x122>(big[x]);
        big[x] = dpp_umax<0x121>(big[x]);
        big[x] = with_half(with_row(big[x], umax), umax);
    }
    __syncthreads();  // the last run's are read
    if (l < 2) part[l][tid / WAVE] = l ? big[1] : big[0];
    __syncthreads();
    QuantScale q[2];
    bool grows[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
#pragma unroll
        for (int k = 0; k < PW_THREADS / WAVE; k++) big[x] = max(big[x], part[x][k]);
        q[x] = quant_scale(big[x]);
        grows[x] = !(old[x] >= q[x].d || old[x] != old[x]);  // q.d of NaN too
        if (!grows[x])
            q[x] = old[x] >= 0x1p-126f && old[x] < INFINITY ? QuantScale{old[x], 1.0f / old[x]} : QuantScale{old[x], 0.0f};
    }
    for (int i0 = 0; i0 < n; i0 += HELD) {
        if (n > HELD) rows(i0);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int i = i0 + s * RPS + tid / LPU;
            if (i < n) {
#pragma unroll
                for (int x = 0; x < 2; x++)
                    *reinterpret_cast<uint32_t*>(pool[x] + (int64_t)(off + i) * a.c.token_stride + d) =
                        quant4(y[x][s][0], y[x][s][1], y[x][s][2], y[x][s][3], q[x].inv);
            }
        }
    }
    // gone where it begins anew, at the new scale where that grew.  The old scale has been read by all waves:
    // two barriers lie behind
#pragma unroll
    for (int x = 0; x < 2; x++) {
        if (off && !grows[x]) continue;
        if (tid == 0) scale[x][0] = q[x].d;
        const float ratio = q[x].d > 0.0f ? old[x] / q[x].d : 0.0f;
        for (int i = c_row; i <= bmask; i += CPS) {
            if (i >= off && i < off + n) continue;
            v4i_t v = i == c_row ? held[x] : off ? *cell(x, i) : v4i_t{};
            if (off) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float f[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) f[k] = (float)(v[j] << (24 - 8 * k) >> 24);
                    v[j] = (int)quant4(f[0], f[1], f[2], f[3], ratio);
                }
            }
            *cell(x, i) = v;
        }
    }
}

template <int HD, int STEPS>
__global__ __launch_bounds__(PW_THREADS, STEPS > 2 ? 3 : 4) void paged_append_i8_kernel(AppendI8 g) {
    __shared__ uint32_t part[2][PW_THREADS / WAVE];
    const PagedAppendArgs& a = g.a;
    // the two kinds of work groups in turns: the queries stream, the cache's wait for one another's loads
    const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (b >= g.blocks) return;
    const int64_t bq = (int64_t)((double)b * g.q_share), bq1 = (int64_t)((double)(b + 1) * g.q_share);
    if (bq1 > bq) {
        append_queries<HD>(a, bq);
        return;
    }
    const int u = (int)((b - bq) % a.c.nkv);
    const int64_t t0 = (b - bq) / a.c.nkv * g.rows;
    if (t0 >= a.n_rows) return;
    // which of the work group's rows are the first of their runs, and how far these go: 64 rows in the lanes
    const int l = threadIdx.x % WAVE, bmask = (1 << g.bshift) - 1;
    const int t = (int)min(t0 + l, (int64_t)a.n_rows - 1);
    const int slot = a.slots[t], pos = a.positions[t], before = t0 ? (int)t0 - 1 : 0;
    const int slot0 = a.slots[before], pos0 = a.positions[before];
    const bool ok = t0 + l < a.n_rows && row_ok(a, slot, pos);
    int prev = __shfl_up(ok ? slot : -2, 1, WAVE);
    if (l == 0) prev = t0 && row_ok(a, slot0, pos0) ? slot0 : -2;
    const bool on = ok && prev == slot - 1 && (slot & bmask) != 0;
    const unsigned long long goes_on = __ballot(on);
    for (unsigned long long todo = __ballot(ok && !on && l < g.rows); todo; todo &= todo - 1) {
        const int f = __builtin_ctzll(todo);
        const unsigned long long stops = f == WAVE - 1 ? 0 : ~goes_on >> (f + 1);
        const int n = stops ? 1 + __builtin_ctzll(stops) : WAVE - f;
        append_run<HD, STEPS>(g, __builtin_amdgcn_readfirstlane((int)t0 + f), n, !stops, pos, f, u, part);
    }
}

hipError_t launch_paged_append_i8(const PagedAppendArgs& a, const PagedViewI8& v, hipStream_t s) {
    const int per = PQ_STEPS * WAVE * 4 / a.c.hd, rows = a.n_rows <= PW_ALONE ? 1 : PW_ROWS;
    const int64_t q_blocks = (int64_t)((a.n_rows + 3) / 4) * ((a.nh + per - 1) / per);
    const int64_t n = q_blocks + (int64_t)((a.n_rows + rows - 1) / rows) * a.c.nkv;
    const int64_t gx = n < 1 << 22 ? n : 1 << 22;  // a launch has fewer than 2^32 threads along x
    const AppendI8 g{a, v.ks, v.vs, v.bshift, rows, n, ((double)q_blocks + 0.5) / (double)n};
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));
    const bool longer = v.bshift > 4;
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(PW_THREADS), 0, s, g); };
    if (a.c.hd == 128)
        longer ? launch(paged_append_i8_kernel<128, 4>) : launch(paged_append_i8_kernel<128, 2>);
    else
        longer ? launch(paged_append_i8_kernel<64, 2>) : launch(paged_append_i8_kernel<64, 1>);
    return hipGetLastError();
}

}  // namespace hy
