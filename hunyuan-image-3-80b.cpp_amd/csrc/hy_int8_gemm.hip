// hy_int8_gemm.hip -- products of tokens and weights in 8-bit integers (hy_gemm_i8, hy_linear_i8) and
// the quantization of rows that they are fed by (hy_quantize_rows_i8).
#include <cmath>

#include "hy_device.hpp"
#include "hy_int8.hpp"
#include "hy_lds.hpp"
#include "hy_mfma.hpp"
#include "hy_split.hpp"

namespace hy {

// ---------------------------------------------------------------- quantization of rows
// A work group per row: largest magnitude (as bits, so that an infinity or NaN is among the largest),
// then codes.  Rows up to QR_KEEP values stay in registers between the two, longer ones are read again.
// Bound by memory: 4096 rows of 4096 20 us, 4.2 TB/s; few rows by latency, 4 us.
constexpr int QR_THREADS = 256, QR_VEC = 4, QR_KEEP = QR_THREADS * QR_VEC * 4;

__global__ __launch_bounds__(QR_THREADS) void quantize_rows_kernel(const float* __restrict__ x, int rows, int cols,
                                                                  int8_t* __restrict__ codes,
                                                                  float* __restrict__ scales) {
    __shared__ uint32_t part[QR_THREADS / WAVE];
    const int tid = threadIdx.x;
    const int64_t r = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (r >= rows) return;
    const float* const row = x + r * cols;
    v4f_t v[QR_VEC];
    uint32_t big = 0;
    const auto load = [&](int c0) {
#pragma unroll
        for (int j = 0; j < QR_VEC; j++) {
            const int c = c0 + 4 * (tid + QR_THREADS * j);
            v[j] = c < cols ? *reinterpret_cast<const v4f_t*>(row + c) : v4f_t{};
        }
    };
    for (int c0 = 0; c0 < cols; c0 += QR_KEEP) {
        load(c0);
#pragma unroll
        for (int j = 0; j < QR_VEC; j++)
#pragma unroll
            for (int k = 0; k < 4; k++) big = max(big, __float_as_uint(v[j][k]) & 0x7fffffffu);
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) big = max(big, (uint32_t)shfl_xor((int)big, m));
    if (tid % WAVE == 0) part[tid / WAVE] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < QR_THREADS / WAVE; w++) big = max(big, part[w]);
    const QuantScale q = quant_scale(big);
    if (tid == 0) scales[r] = q.d;
    int8_t* const out = codes + r * cols;
    for (int c0 = 0; c0 < cols; c0 += QR_KEEP) {
        if (cols > QR_KEEP) load(c0);
#pragma unroll
        for (int j = 0; j < QR_VEC; j++) {
            const int c = c0 + 4 * (tid + QR_THREADS * j);
            if (c < cols)
                *reinterpret_cast<uint32_t*>(out + c) = quant4(v[j][0], v[j][1], v[j][2], v[j][3], q.inv);
        }
    }
}

hipError_t launch_quantize_rows(const float* x, int rows, int cols, int8_t* codes, float* scales, hipStream_t s) {
    const unsigned gx = rows < 1 << 22 ? rows : 1 << 22;  // fewer than 2^32 threads along x
    hipLaunchKernelGGL(quantize_rows_kernel, dim3(gx, (rows + gx - 1) / gx), dim3(QR_THREADS), 0, s, x, rows, cols,
                       codes, scales);
    return hipGetLastError();
}

// ---------------------------------------------------------------- products of few tokens
// A stream over the weights: a work group of GS_WAVES waves takes 16 channels of 16 tokens, each wave a part of
// the reduction, straight from memory into the operands of v_mfma_i32_16x16x64_i8 (lane l: 16 bytes of row
// l % 16 at k offset 16 (l / 16), of A and of B alike; result v is A's row 4 (l / 16) + v, B's row l % 16),
// GS_DEPTH steps of 64 ahead.  The waves' sums meet in LDS: whole numbers, so in any order.
// FUSED: the tokens are f32, up to GF_TOKENS of them, and every work group quantizes them for itself while its
// first weights are on their way, which spares a launch (one token, 4096 x 6144: 10.0 us, in two launches 9.9 + 2.6).
// Bound by a chain: GS_DEPTH of a wave's 16 steps of weights (4096 wide) are asked for before the tokens are read twice,
// with two barriers, the others only behind that; 25 MB of weights would take 5 us at a copy's rate.
constexpr int GS_WAVES = 4, GS_THREADS = WAVE * GS_WAVES, GS_DEPTH = 8;
constexpr int GF_TOKENS = 4, GF_WIDTH = 8192;

template <bool FUSED>
__global__ __launch_bounds__(GS_THREADS) void gemm_i8_stream_kernel(GemmI8Args a, int tiles_n) {
    __shared__ int sum[256];
    __shared__ __attribute__((aligned(16))) int8_t codes[FUSED ? GF_TOKENS : 1][FUSED ? GF_WIDTH : 16];
    __shared__ uint32_t part[FUSED ? GF_TOKENS : 1][GS_WAVES];
    const int tid = threadIdx.x, lane = tid % WAVE, r = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int n0 = (int)(b % tiles_n) * 16;
    const int64_t t64 = b / tiles_n * 16;
    if (t64 >= a.T) return;
    const int t0 = (int)t64;
    const int steps = (a.K + 63) / 64, s0 = steps * wave / GS_WAVES, s1 = steps * (wave + 1) / GS_WAVES;
    const int8_t* const wp = a.w + (int64_t)min(n0 + r, a.N - 1) * a.K;
    const int8_t* const xp = FUSED ? codes[min(r, a.T - 1)] : a.x + (int64_t)min(t0 + r, a.T - 1) * a.K;
    v4i_t wf[GS_DEPTH], xf[GS_DEPTH];
    // steps past the last are read again and not used
    const auto at = [&](int s) { return min(64 * min(s, s1 - 1) + 16 * g, a.K - 16); };
    const auto load = [&](int s, int d) {
        wf[d] = *reinterpret_cast<const v4i_t*>(wp + at(s));
        if constexpr (!FUSED) xf[d] = *reinterpret_cast<const v4i_t*>(xp + at(s));
    };
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < GS_DEPTH; d++) load(s0 + d, d);
    }
    sum[tid] = 0;
    float xs[GF_TOKENS];
    if constexpr (FUSED) {
        __builtin_amdgcn_sched_barrier(0);
        uint32_t big[GF_TOKENS];
#pragma unroll
        for (int t = 0; t < GF_TOKENS; t++) {
            big[t] = 0;
            if (t >= a.T) continue;  // the same for the work group
            for (int c = 4 * tid; c < a.K; c += 4 * GS_THREADS) {
                const v4f_t v = *reinterpret_cast<const v4f_t*>(a.xf + (int64_t)t * a.K + c);
#pragma unroll
                for (int j = 0; j < 4; j++) big[t] = max(big[t], __float_as_uint(v[j]) & 0x7fffffffu);
            }
#pragma unroll
            for (int m = 32; m; m >>= 1) big[t] = max(big[t], (uint32_t)shfl_xor((int)big[t], m));
            if (lane == 0) part[t][wave] = big[t];
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < GF_TOKENS; t++) {
            if (t >= a.T) continue;
#pragma unroll
            for (int w = 0; w < GS_WAVES; w++) big[t] = max(big[t], part[t][w]);
            const QuantScale q = quant_scale(big[t]);
            xs[t] = q.d;
            for (int c = 4 * tid; c < a.K; c += 4 * GS_THREADS) {
                const v4f_t v = *reinterpret_cast<const v4f_t*>(a.xf + (int64_t)t * a.K + c);
                *reinterpret_cast<uint32_t*>(&codes[t][c]) = quant4(v[0], v[1], v[2], v[3], q.inv);
            }
        }
    }
    __syncthreads();
    v4i_t acc = {};
    for (int s = s0; s < s1; s += GS_DEPTH) {
#pragma unroll
        for (int d = 0; d < GS_DEPTH; d++) {
            if (s + d < s1) {  // the same for the wave
                if constexpr (FUSED) xf[d] = *reinterpret_cast<const v4i_t*>(xp + at(s + d));
                // behind the reduction's end the weights count as 0
                if (64 * (s + d) + 64 > a.K) wf[d] = 64 * (s + d) + 16 * g >= a.K ? v4i_t{} : wf[d];
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[d], wf[d], acc, 0, 0, 0);
            }
            load(s + GS_DEPTH + d, d);
        }
    }
#pragma unroll
    for (int v = 0; v < 4; v++) atomicAdd(&sum[(4 * g + v) * 16 + r], acc[v]);
    __syncthreads();
    const int row = tid / 16, t = t0 + row, n = n0 + tid % 16;
    if (t >= a.T || n >= a.N) return;
    float scale;
    if constexpr (FUSED) {
        scale = xs[0];
#pragma unroll
        for (int i = 1; i < GF_TOKENS; i++) scale = row == i ? xs[i] : scale;
    } else {
        scale = a.xs[t];
    }
    const int64_t o = (int64_t)t * a.N + n;
    float y = (float)sum[tid] * scale * a.ws[n];
    if (a.resid) y += a.resid[o];
    a.out[o] = y;
}

// ---------------------------------------------------------------- products of many tokens
// Tiles of BT tokens x BN channels, WT x WN waves, results of v_mfma_i32_32x32x32_i8 (lane l holds 16 bytes of
// row l % 32 at k offset 16 (l / 32); result v is A's row 8 (v / 4) + 4 (l / 32) + v % 4, B's row l % 32; A is
// the tokens, so that a store's lanes are neighbouring channels).  Stages of KB bytes of the reduction are
// copied from memory into a ring in LDS, all but the one that is multiplied on their way; one barrier
// per stage; operands are read from LDS one step of 32 ahead of their products.
// Piece c (16 bytes) of a stage's row lies in place c ^ swap(row), so that 16 rows' reads of one piece touch
// every bank once.  The copies' places are fixed, so they fetch the pieces swapped.
// Rows of 128 bytes: with 64 the copies are half as fast (a request of the L2 is 64 bytes of a line of
// 128).
// Bounds.  Tiles of 256 x 256 (4096 tokens x 4096 x 6144: 103 us, 2.0 PO/s; 8192^3 reaches 2.17, a library
// product 2.09): the matrix pipe and the power it draws, the copies from the L2 and, at 6144 channels, one
// and a half rounds of 256 work groups.  Small tiles (300 tokens x 4096 x 4096: 16.5 us, 0.6 PO/s): 32 stages that wait
// for one another, 0.5 us each, in 320 work groups on 256 CUs; their copies, 168 MB, come at 10 TB/s where the L2
// gives three times that.  One row of tiles (16 tokens x 4096 x 133120: 112 us): the weights at 4.9 TB/s.
template <int BT_, int BN_, int WT_, int WN_, int RING_, int KB_>
struct GtShape {
    static constexpr int BT = BT_, BN = BN_, WT = WT_, WN = WN_, RING = RING_, KB = KB_;
    static constexpr int PIECES = KB / 16, ROWS = 64 / PIECES, Q = KB / 32;  // of a row, of a copy, products deep
    static constexpr int WAVES = WT * WN, THREADS = WAVE * WAVES;
    static constexpr int MT = BT / WT / 32, NT = BN / WN / 32;  // 32 x 32 results of a wave
    static constexpr int A = BT * KB, STAGE = A + BN * KB, LDS = RING * STAGE;
    // copies of 1 KB per wave and stage, of tokens and of both; copy i of wave w is the stage's KB i WAVES + w
    static constexpr int COPIES_A = A / 1024 / WAVES, COPIES = STAGE / 1024 / WAVES;
    static_assert(COPIES * WAVES * 1024 == STAGE && MT * 32 * WT == BT && NT * 32 * WN == BN, "whole copies and results");
    static_assert(COPIES_A * WAVES * 1024 == A && ROWS * WAVES % (256 / KB * PIECES) == 0, "one swap per lane");
    __device__ static __forceinline__ int swap(int row) { return row / (256 / KB) % PIECES; }
};

__device__ const int8_t i8_zeros[16] = {};

template <class S, bool ONCE>
__device__ __forceinline__ void gemm_i8_tile(const GemmI8Args& a, int t0, int n0, uint8_t* lds) {
    const int tid = threadIdx.x, lane = tid % WAVE, lr = lane % 32, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int K = a.K, stages = (K + S::KB - 1) / S::KB;

    uint32_t off[S::COPIES];
    const int piece = (lane % S::PIECES) ^ S::swap(lane / S::PIECES + S::ROWS * wave);
    const __amdgpu_buffer_rsrc_t xr = buf_rsrc(a.x + (int64_t)t0 * K), wr = buf_rsrc(a.w + (int64_t)n0 * K);
#pragma unroll
    for (int i = 0; i < S::COPIES; i++) {
        const int row = S::ROWS * (i * S::WAVES + wave) + lane / S::PIECES;
        const int clamped = row < S::BT ? min(row, a.T - 1 - t0) : min(row - S::BT, a.N - 1 - n0);
        off[i] = (uint32_t)clamped * K + 16 * piece;
    }
    const auto copy = [&](int s) {
        uint8_t* const dst = lds + (s % S::RING) * S::STAGE + 1024 * wave;
        if (S::KB * s + S::KB <= K) {
#pragma unroll
            for (int i = 0; i < S::COPIES; i++) {
                if (i < S::COPIES_A)
                    b2l(xr, dst + 1024 * S::WAVES * i, off[i], S::KB * s);
                else
                    b2l<16, ONCE ? HY_CPOL_NT : 0>(wr, dst + 1024 * S::WAVES * i, off[i], S::KB * s);
            }
        } else {  // the reduction ends inside the stage: zeros behind it
#pragma unroll
            for (int i = 0; i < S::COPIES; i++) {
                const int8_t* const base = i < S::COPIES_A ? a.x + (int64_t)t0 * K : a.w + (int64_t)n0 * K;
                g2l16(S::KB * s + 16 * piece < K ? base + off[i] + S::KB * s : i8_zeros, dst + 1024 * S::WAVES * i);
            }
        }
    };
    v16i_t acc[S::MT][S::NT];
#pragma unroll
    for (int i = 0; i < S::MT; i++)
#pragma unroll
        for (int j = 0; j < S::NT; j++) acc[i][j] = v16i_t{};
    // this lane's rows of the wave's tokens and channels
    const int wt = wave % S::WT, wn = wave / S::WT;
    const uint32_t a_row = lds_off(lds) + (uint32_t)(32 * S::MT * wt + lr) * S::KB;
    const uint32_t b_row = lds_off(lds) + S::A + (uint32_t)(32 * S::NT * wn + lr) * S::KB;
    uint32_t place[S::Q];
#pragma unroll
    for (int q = 0; q < S::Q; q++) place[q] = 16 * ((2 * q + h) ^ S::swap(lr));

    int n[S::NT];  // this lane's channels, and the token of its result v of row i of results
#pragma unroll
    for (int j = 0; j < S::NT; j++) n[j] = n0 + 32 * (S::NT * wn + j) + lr;
    const auto token = [&](int i, int v) { return t0 + 32 * (S::MT * wt + i) + 8 * (v / 4) + 4 * h + v % 4; };
    // What is added: read ahead of the copies where there are registers for it, else four results at a time
    // (300 tokens x 4096 x 4096 23.4 us, so 18.4)
    constexpr bool EARLY = S::MT * S::NT <= 2;
    float resid[EARLY ? S::MT : 1][S::NT][EARLY ? 16 : 4];
    const auto read_resid = [&](int i, int v0, int v1) {
#pragma unroll
        for (int v = v0; v < v1; v++)
#pragma unroll
            for (int j = 0; j < S::NT; j++)
                resid[EARLY ? i : 0][j][EARLY ? v : v - v0] =
                    a.resid[(int64_t)min(token(i, v), a.T - 1) * a.N + min(n[j], a.N - 1)];
    };
    if constexpr (EARLY) {
        if (a.resid) {
#pragma unroll
            for (int i = 0; i < S::MT; i++) read_resid(i, 0, 16);
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    v4i_t af[2][S::MT], bf[2][S::NT];
    const auto read = [&](int s, int q) {
        const uint32_t at = (uint32_t)(s % S::RING) * S::STAGE + place[q];
        static_for<S::MT>([&](auto i) { af[q % 2][i] = lds_b128_at<32 * S::KB * i>(a_row + at); });
        static_for<S::NT>([&](auto j) { bf[q % 2][j] = lds_b128_at<32 * S::KB * j>(b_row + at); });
    };
    const auto multiply = [&](int q) {
#pragma unroll
        for (int i = 0; i < S::MT; i++) lds_pin(af[q][i]);
#pragma unroll
        for (int j = 0; j < S::NT; j++) lds_pin(bf[q][j]);
        __builtin_amdgcn_s_setprio(1);  // a wave with its operands goes first: 8192 tokens 302 -> 290 us
#pragma unroll
        for (int j = 0; j < S::NT; j++)
#pragma unroll
            for (int i = 0; i < S::MT; i++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[q][i], bf[q][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int s = 0; s < S::RING; s++)
        if (s < stages) copy(s);
    wait_copies<S::COPIES, S::RING - 1>(stages - 1);
    __syncthreads();
    read(0, 0);
    for (int s = 0; s < stages; s++) {
#pragma unroll
        for (int q = 0; q + 1 < S::Q; q++) {
            read(s, q + 1);
            lds_wait_upto<S::MT + S::NT>();
            multiply(q % 2);
        }
        if (s + 1 < stages) {
            // the next stage's copies have arrived, later ones' are on their way; this wave has read its part of
            // the stage out (the wait is for LDS reads too)
            wait_copies<S::COPIES, S::RING - 2>(stages - 2 - s);
            __syncthreads();  // and so have the others
            if (s + S::RING < stages) copy(s + S::RING);
            read(s + 1, 0);
            lds_wait_upto<S::MT + S::NT>();
        } else {
            lds_wait_upto<0>();
        }
        multiply((S::Q - 1) % 2);
    }
    float wscale[S::NT];
#pragma unroll
    for (int j = 0; j < S::NT; j++) wscale[j] = a.ws[min(n[j], a.N - 1)];
#pragma unroll
    for (int i = 0; i < S::MT; i++)
#pragma unroll
        for (int v0 = 0; v0 < 16; v0 += 4) {
            float xs[4];
#pragma unroll
            for (int v = v0; v < v0 + 4; v++) xs[v - v0] = a.xs[min(token(i, v), a.T - 1)];
            if constexpr (!EARLY)
                if (a.resid) read_resid(i, v0, v0 + 4);
#pragma unroll
            for (int v = v0; v < v0 + 4; v++)
#pragma unroll
                for (int j = 0; j < S::NT; j++) {
                    float y = (float)acc[i][j][v] * xs[v - v0] * wscale[j];
                    if (a.resid) y += EARLY ? resid[i][j][v] : resid[0][j][v - v0];
                    if (token(i, v) < a.T && n[j] < a.N) a.out[(int64_t)token(i, v) * a.N + n[j]] = y;
                }
            __builtin_amdgcn_sched_barrier(0);
        }
}

constexpr int GT_XCDS = 8, GT_CUS = 32;  // of an XCD

// HALF: the shape of half a tile of channels, which what is left over of the last round falls into, or S itself.
// ONCE: the weights are read once and past the caches (tiles_once)
template <class S, class HALF, bool ONCE>
__global__ __launch_bounds__(S::THREADS, S::WAVES / 4 * (S::LDS > 81920 ? 1 : 2)) void gemm_i8_tile_kernel(
    GemmI8Args a, int tiles_n, int tiles) {
    constexpr bool SPLIT = HALF::BN < S::BN;
    static_assert(HALF::THREADS == S::THREADS && HALF::LDS <= S::LDS, "the same work group");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::LDS];
    // tiles in bands of 8 of channels, tokens outer; neighbouring ones on one XCD (work groups go round the
    // XCDs), where those that run at once share rows and columns of tiles
    const int xcd = blockIdx.x % GT_XCDS, lo = (int)((int64_t)tiles * xcd / GT_XCDS);
    const int mine = (int)((int64_t)tiles * (xcd + 1) / GT_XCDS) - lo, left = mine % GT_CUS;
    const int whole = SPLIT && left <= GT_CUS / 2 ? mine - left : mine;
    int i = blockIdx.x / GT_XCDS, half = -1;
    if (i >= whole) {
        half = (i - whole) % 2;
        i = whole + (i - whole) / 2;
    }
    if (i >= mine) return;
    const int o = lo + i, tiles_t = tiles / tiles_n, band = o / (8 * tiles_t), width = min(8, tiles_n - 8 * band);
    const int in_band = o - band * 8 * tiles_t;
    const int n0 = (8 * band + in_band % width) * S::BN, t0 = in_band / width * S::BT;
    if (!SPLIT || half < 0) {
        gemm_i8_tile<S, ONCE>(a, t0, n0, lds);
    } else if (n0 + half * HALF::BN < a.N) {
        gemm_i8_tile<HALF, ONCE>(a, t0, n0 + half * HALF::BN, lds);
    }
}

template <bool FUSED>
static void stream(const GemmI8Args& a, hipStream_t s) {
    const int tiles_n = (a.N + 15) / 16;
    const int64_t n = (int64_t)tiles_n * ((a.T + 15) / 16), gx = n < 1 << 22 ? n : 1 << 22;
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));  // fewer than 2^32 threads along x
    hipLaunchKernelGGL(gemm_i8_stream_kernel<FUSED>, grid, dim3(GS_THREADS), 0, s, a, tiles_n);
}

template <class S, class HALF = S, bool ONCE = false>
static void tiles(const GemmI8Args& a, hipStream_t s) {
    const int tiles_n = (a.N + S::BN - 1) / S::BN, tiles = tiles_n * ((a.T + S::BT - 1) / S::BT);
    const int per_xcd = (tiles + GT_XCDS - 1) / GT_XCDS + (HALF::BN < S::BN ? GT_CUS / 2 : 0);
    hipLaunchKernelGGL((gemm_i8_tile_kernel<S, HALF, ONCE>), dim3((unsigned)(GT_XCDS * per_xcd)), dim3(S::THREADS), 0, s, a,
                       tiles_n, tiles);
}
// one row of tiles over weights that the Infinity Cache does not hold: past the caches (16 tokens x 133120 channels
// 120 us, so 112; 20 x 6144, which it holds, 12.1 and 12.7)
template <class S>
static void tiles_once(const GemmI8Args& a, hipStream_t s) {
    if (a.T <= S::BT && (size_t)a.N * a.K > INFINITY_CACHE)
        tiles<S, S, true>(a, s);
    else
        tiles<S>(a, s);
}
typedef GtShape<256, 256, 4, 4, 2, 128> GtBig;
typedef GtShape<256, 128, 4, 4, 2, 128> GtBigHalf;
typedef GtShape<128, 128, 2, 4, 2, 128> GtMid;
typedef GtShape<64, 128, 2, 4, 3, 128> GtWide;
typedef GtShape<64, 64, 2, 2, 4, 128> GtSmall;
typedef GtShape<32, 64, 1, 2, 4, 128> GtTiny;

// Which kernel, by what each takes at hidden 4096 (all in proportion to it), us:
//  * the stream, for up to 4 tokens and 128 MB of weights.  1 and 4 tokens x 6144 channels 9.3, 9.8, by tiles of
//    32 x 64 10.9, 11.3; x 32000 30.5, 34.7 and 31.8, 32.4 (and a launch more where tokens are f32); x 133120
//    117, 133 and 97, 102;
//  * tiles of 32 x 64 for up to 32: 32 x 6144 12.6, by 64 x 64 14.5, 20 11.9 and 13.8, x 133120 128 and 129;
//  * tiles of 64 x 64: 17.5 for up to 512, which all run at once, then 6 and 38 ns per tile (rings of 5 stages, of
//    which one work group fits a CU where there are more than 256: 18.9; of 64 x 32: 17.9);
//  * tiles of 64 x 128, where all run at once: 18.5, or 12 and 38 ns per tile;
//  * tiles of 128 x 128: 28, or 8 and 93 ns per tile;
//  * tiles of 256 x 256: 70 per round of 256, 45 for a last round of up to 128, which takes half tiles.
// 64 x 64, 64 x 128, 128 and 256 wide tiles measured: 300 tokens x 4096 channels 17.4, 18.8, 27, 33; 512 x 6144
// 34, 27, 35, 44; 700 x 4096 31, 26, 29, -; 1024 x 4096 38, 31, 35, -; 1024 x 6144 58, 47, 42, 49; 2048 x 6144
// 103, 84, 75, 70; 4096 x 6144 226, -, 144, 127 (without half tiles 144); 64 x 133120 140, 135, 175, -; 256 x
// 133120 312, 266, 243, 233.
static double tiles_of(const GemmI8Args& a, int bt, int bn) {
    return (double)((a.T + bt - 1) / bt) * ((a.N + bn - 1) / bn);
}
static bool by_stream(const GemmI8Args& a) {
    return a.T <= GF_TOKENS && a.K <= GF_WIDTH && (size_t)a.N * a.K <= (size_t)1 << 27;
}

bool gemm_i8_takes_f32(const GemmI8Args& a) { return by_stream(a); }

hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s) {
    if (by_stream(a)) {
        a.xf ? stream<true>(a, s) : stream<false>(a, s);
        return hipGetLastError();
    }
    const double n64 = tiles_of(a, 64, 64), nwide = tiles_of(a, 64, 128);
    const double n128 = tiles_of(a, 128, 128), n256 = tiles_of(a, 256, 256);
    const double small = n64 <= 512.0 ? 17.5 : 6.0 + 0.038 * n64, mid = fmax(28.0, 8.0 + 0.093 * n128);
    const double wide = nwide <= 512.0 ? fmax(18.5, 12.0 + 0.038 * nwide) : HUGE_VAL;
    const double rounds = floor(n256 / 256.0), left = n256 - 256.0 * rounds;
    const double big = 70.0 * rounds + (left == 0.0 ? 0.0 : left <= 128.0 ? 45.0 : 70.0);
    if (a.T <= 32)
        tiles_once<GtTiny>(a, s);
    else if (small <= wide && small <= mid && small <= big)
        tiles_once<GtSmall>(a, s);
    else if (wide <= mid && wide <= big)
        tiles<GtWide>(a, s);
    else if (mid <= big)
        tiles<GtMid>(a, s);
    else
        tiles<GtBig, GtBigHalf>(a, s);
    return hipGetLastError();
}

}  // namespace hy
