// hy_paged_i8.hip -- the write into a paged cache of 8-bit integers (hy_rope_qknorm_paged_i8): rotary
// embedding and QK-norm, queries to [rows][nh][hd], keys and values to codes with a scale per block of
// positions and head.
//
// A scale belongs to all rows that a call brings into its block, so the unit of work is a run (rows
// whose slots follow one another inside a block) times a head of K or of V, a wave each: the wave of
// a run's first row does all of it, those of the others find that they are not the first and
// end.  HD / 4 lanes share a row, 4 dims each; 16 rows are held at a time, and runs that are longer are
// gone through twice (largest magnitude, then codes).
// A key is rotated and normed in 64 bits and rounded to f32 once: a value next to the border
// between two codes would otherwise fall by the order of the sum, and a step is 2^-7 of the largest.
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

constexpr int PQ_STEPS = 4;  // of query heads

struct AppendI8 {
    PagedAppendArgs a;
    float* ks;
    float* vs;
    int bshift;
    int q_blocks;  // work groups of the queries; those behind write the cache
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

// row t of head u of K, (u < nkv) or of head u - nkv of V: this lane's 4 values, as they are quantized
template <int HD>
__device__ __forceinline__ v4f_t cache_row(const PagedAppendArgs& a, v4f_t x, int pos, int d, v4f_t w) {
    double cs[2] = {1.0, 1.0}, sn[2] = {0.0, 0.0};
    if (a.rotate == 1) {
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const double turn = (double)pos * a.freq[d / 2 + p];
            sincos_turn(turn - rint(turn), sn[p], cs[p]);
        }
    } else if (a.rotate == 2) {
        const v4f_t c = *reinterpret_cast<const v4f_t*>(a.cos_t + (int64_t)pos * HD + d);
        const v4f_t s = *reinterpret_cast<const v4f_t*>(a.sin_t + (int64_t)pos * HD + d);
        cs[0] = c[0], cs[1] = c[2], sn[0] = s[0], sn[1] = s[2];
    }
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

template <int HD>
__device__ __forceinline__ void append_run(const AppendI8& g, int t, int u) {
    constexpr int LPU = HD / 4, RPS = WAVE / LPU, STEPS = 16 / RPS;  // 16 rows at a time
    const PagedAppendArgs& a = g.a;
    const int l = threadIdx.x % WAVE, d = 4 * (l % LPU), bmask = (1 << g.bshift) - 1;
    const int units = a.nh + 2 * a.c.nkv;
    // is t the first row of its run?
    const int slot = a.slots[t], pos0 = a.positions[t];
    if (!row_ok(a, slot, pos0)) return;
    const int off = slot & bmask;
    if (t > 0 && off > 0 && a.slots[t - 1] == slot - 1 && row_ok(a, slot - 1, a.positions[t - 1])) return;
    int n = 0;  // rows of the run
    for (;;) {
        const int i = n + l, r = min(t + i, a.n_rows - 1);
        const int s = a.slots[r];
        const bool in = t + i < a.n_rows && i <= bmask - off && s == slot + i && row_ok(a, s, a.positions[r]);
        const unsigned long long out = __ballot(!in);
        n += out ? __builtin_ctzll(out) : WAVE;
        if (out) break;
    }
    n = __builtin_amdgcn_readfirstlane(n);
    const bool key = u < a.c.nkv;
    const int head = key ? u : u - a.c.nkv, page = slot >> a.c.shift, in_page = slot & ((1 << a.c.shift) - 1);
    int8_t* const pool = static_cast<int8_t*>(key ? a.c.k : a.c.v) + (int64_t)page * a.c.page_stride +
                         (int64_t)head * a.c.head_stride + (int64_t)(in_page - off) * a.c.token_stride;
    float* const scale = (key ? g.ks : g.vs) + ((((int64_t)page * a.c.nkv + head) << (a.c.shift - g.bshift)) +
                                                (in_page >> g.bshift));
    const float* const src = a.qkv + (int64_t)t * units * HD + (int64_t)(a.nh + u) * HD + d;
    const v4f_t one = {1.0f, 1.0f, 1.0f, 1.0f};
    const v4f_t w = key && a.k_norm ? *reinterpret_cast<const v4f_t*>(a.k_norm + d) : one;
    const float old = off ? scale[0] : 0.0f;
    v4f_t y[STEPS];
    uint32_t big = 0;
    const auto rows = [&](int i0) {
        int pos[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int i = min(i0 + s * RPS + l / LPU, n - 1);
            y[s] = *reinterpret_cast<const v4f_t*>(src + (int64_t)i * units * HD);
            pos[s] = a.positions[t + i];
        }
        if (key) {
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                if (i0 + s * RPS >= n) break;  // the same for the wave
                y[s] = cache_row<HD>(a, y[s], pos[s], d, w);
            }
        }
    };
    for (int i0 = 0; i0 < n; i0 += 16) {
        rows(i0);
#pragma unroll
        for (int s = 0; s < STEPS; s++)
            if (i0 + s * RPS < n) {  // rows past the last are the last again
#pragma unroll
                for (int j = 0; j < 4; j++) big = max(big, __float_as_uint(y[s][j]) & 0x7fffffffu);
            }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) big = max(big, (uint32_t)shfl_xor((int)big, m));
    QuantScale q = quant_scale(big);
    const bool grows = !(old >= q.d || old != old);  // q.d of NaN too
    if (!grows) q = old >= 0x1p-126f && old < INFINITY ? QuantScale{old, 1.0f / old} : QuantScale{old, 0.0f};
    for (int i0 = 0; i0 < n; i0 += 16) {
        if (n > 16) rows(i0);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int i = i0 + s * RPS + l / LPU;
            if (i < n)
                *reinterpret_cast<uint32_t*>(pool + (int64_t)(off + i) * a.c.token_stride + d) =
                    quant4(y[s][0], y[s][1], y[s][2], y[s][3], q.inv);
        }
    }
    if (l == 0 && (grows || off == 0)) scale[0] = q.d;
    // what the block holds besides: gone where it begins anew, at the new scale where that grew
    if (off && !grows) return;
    const float ratio = q.d > 0.0f ? old / q.d : 0.0f;
    constexpr int LPC = HD / 16, CPS = WAVE / LPC;  // 16 codes per lane
    const int c = 16 * (l % LPC);
    for (int i = l / LPC; i <= bmask; i += CPS) {
        if (i >= off && i < off + n) continue;
        v4i_t* const cell = reinterpret_cast<v4i_t*>(pool + (int64_t)i * a.c.token_stride + c);
        v4i_t v = {};
        if (off) {
            v = *cell;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float f[4];
#pragma unroll
                for (int k = 0; k < 4; k++) f[k] = (float)(v[j] << (24 - 8 * k) >> 24);
                v[j] = (int)quant4(f[0], f[1], f[2], f[3], ratio);
            }
        }
        *cell = v;
    }
}

template <int HD>
__global__ __launch_bounds__(256) void paged_append_i8_kernel(AppendI8 g) {
    const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (b < g.q_blocks) {
        append_queries<HD>(g.a, b);
        return;
    }
    const int64_t wave = (b - g.q_blocks) * 4 + threadIdx.x / WAVE;
    const int units = 2 * g.a.c.nkv;
    const int64_t t = wave / units;
    if (t >= g.a.n_rows) return;
    append_run<HD>(g, __builtin_amdgcn_readfirstlane((int)t), __builtin_amdgcn_readfirstlane((int)(wave % units)));
}

hipError_t launch_paged_append_i8(const PagedAppendArgs& a, const PagedViewI8& v, hipStream_t s) {
    const int per = PQ_STEPS * WAVE * 4 / a.c.hd;
    const int64_t q_blocks = (int64_t)((a.n_rows + 3) / 4) * ((a.nh + per - 1) / per);
    const int64_t n = q_blocks + ((int64_t)a.n_rows * 2 * a.c.nkv + 3) / 4;
    const int64_t gx = n < 1 << 22 ? n : 1 << 22;  // a launch has fewer than 2^32 threads along x
    const AppendI8 g{a, v.ks, v.vs, v.bshift, (int)q_blocks};
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));
    if (a.c.hd == 128)
        hipLaunchKernelGGL(paged_append_i8_kernel<128>, grid, dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL(paged_append_i8_kernel<64>, grid, dim3(256), 0, s, g);
    return hipGetLastError();
}

}  // namespace hy
