// hy_int8_gemm.hip -- products of tokens and weights in 8-bit integers (hy_gemm_i8, hy_linear_i8) and
// the quantization of rows that they are fed by (hy_quantize_rows_i8).
#include "hy_device.hpp"
#include "hy_int8.hpp"
#include "hy_lds.hpp"
#include "hy_mfma.hpp"

namespace hy {

// ---------------------------------------------------------------- quantization of rows
// A work group per row: largest magnitude (as bits, so that an infinity or NaN is among the largest),
// then codes.  Rows up to QR_KEEP values stay in registers between the two, longer ones are read again.
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
// A stream over the weights: a work group of GS_WAVES waves takes 16 NT channels of 16 TT tokens, each
// wave a part of the reduction, straight from memory into the operands of v_mfma_i32_16x16x64_i8 (lane l:
// 16 bytes of row l % 16 at k offset 16 (l / 16), of A and of B alike; result v is A's row 4 (l / 16) + v, B's
// row l % 16), GS_D steps of 64 ahead.  The waves' sums meet in LDS: whole numbers, so in any order.
constexpr int GS_WAVES = 4;

template <int NT, int TT, int D>
__global__ __launch_bounds__(WAVE * GS_WAVES) void gemm_i8_stream_kernel(GemmI8Args a, int tiles_n) {
    constexpr int BN = 16 * NT, BT = 16 * TT;
    __shared__ int sum[BT * BN];
    const int tid = threadIdx.x, lane = tid % WAVE, r = lane % 16, g = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int n0 = (int)(b % tiles_n) * BN;
    const int64_t t64 = b / tiles_n * BT;
    if (t64 >= a.T) return;
    const int t0 = (int)t64;
    const int steps = (a.K + 63) / 64, s0 = steps * wave / GS_WAVES, s1 = steps * (wave + 1) / GS_WAVES;
    const int8_t* wp[NT];
    const int8_t* xp[TT];
#pragma unroll
    for (int i = 0; i < NT; i++) wp[i] = a.w + (int64_t)min(n0 + 16 * i + r, a.N - 1) * a.K;
#pragma unroll
    for (int j = 0; j < TT; j++) xp[j] = a.x + (int64_t)min(t0 + 16 * j + r, a.T - 1) * a.K;
    v4i_t wf[D][NT], xf[D][TT];
    // steps past the last are read again and not used; behind the reduction's end the weights count as 0
    const auto load = [&](int s, int d) {
        const int k = 64 * min(s, s1 - 1) + 16 * g, at = min(k, a.K - 16);
#pragma unroll
        for (int i = 0; i < NT; i++) wf[d][i] = *reinterpret_cast<const v4i_t*>(wp[i] + at);
#pragma unroll
        for (int j = 0; j < TT; j++) xf[d][j] = *reinterpret_cast<const v4i_t*>(xp[j] + at);
    };
    v4i_t acc[TT][NT] = {};
    if (s0 < s1) {
#pragma unroll
        for (int d = 0; d < D; d++) load(s0 + d, d);
    }
    for (int i = tid; i < BT * BN; i += WAVE * GS_WAVES) sum[i] = 0;
    __syncthreads();
    for (int s = s0; s < s1; s += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            if (s + d < s1) {  // the same for the wave
                if (64 * (s + d) + 64 > a.K) {
                    const bool gone = 64 * (s + d) + 16 * g >= a.K;
#pragma unroll
                    for (int i = 0; i < NT; i++) wf[d][i] = gone ? v4i_t{} : wf[d][i];
                }
#pragma unroll
                for (int j = 0; j < TT; j++)
#pragma unroll
                    for (int i = 0; i < NT; i++)
                        acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[d][j], wf[d][i], acc[j][i], 0, 0, 0);
            }
            load(s + D + d, d);
        }
    }
#pragma unroll
    for (int j = 0; j < TT; j++)
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int v = 0; v < 4; v++) atomicAdd(&sum[(16 * j + 4 * g + v) * BN + 16 * i + r], acc[j][i][v]);
    __syncthreads();
    for (int i = tid; i < BT * BN; i += WAVE * GS_WAVES) {
        const int t = t0 + i / BN, n = n0 + i % BN;
        if (t >= a.T || n >= a.N) continue;
        const int64_t at = (int64_t)t * a.N + n;
        float y = (float)sum[i] * a.xs[t] * a.ws[n];
        if (a.resid) y += a.resid[at];
        a.out[at] = y;
    }
}

// ---------------------------------------------------------------- products of many tokens
// Tiles of 128 tokens x 256 channels: a work group of four waves, each 64 tokens x 128 channels (2 x 4
// results of v_mfma_i32_32x32x32_i8: lane l holds 16 bytes of row l % 32 at k offset 16 (l / 32); result v
// is A's row 8 (v / 4) + 4 (l / 32) + v % 4, B's row l % 32; A is the tokens, so that a store's lanes are
// neighbouring channels).  Stages of 64 bytes of the reduction are copied from memory into a ring of three
// in LDS, two of them on their way while one is multiplied; one barrier per stage.
// A row of a stage is four pieces of 16 bytes; piece c lies in place c ^ (row / 4 % 4), so that
// 16 rows' reads of one piece touch every bank once.  The copies' places are fixed, so they fetch
// the pieces swapped.
constexpr int GT_BT = 128, GT_BN = 256, GT_KB = 64, GT_RING = 3, GT_WAVES = 4;
constexpr int GT_A = GT_BT * GT_KB, GT_STAGE = GT_A + GT_BN * GT_KB;
constexpr int GT_COPIES = GT_STAGE / 1024 / GT_WAVES;  // of 1 KB per wave and stage
static_assert(GT_BT == 128 && GT_BN == 256 && GT_COPIES == 6, "8 copies of tokens, 16 of weights");

__device__ const int8_t i8_zeros[16] = {};

__global__ __launch_bounds__(WAVE * GT_WAVES, 2) void gemm_i8_tile_kernel(GemmI8Args a, int tiles_n, int tiles) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[GT_RING * GT_STAGE];
    const int tid = threadIdx.x, lane = tid % WAVE, lr = lane % 32, h = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    // tiles in bands of 8 x 256 channels, tokens outer; neighbouring ones on one XCD (work groups go round
    // the XCDs): 64 that run there at once share 8 x 8 rows and columns of tiles
    const int per = (tiles + 7) / 8, o = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= per || o >= tiles) return;
    const int tiles_t = tiles / tiles_n, band = o / (8 * tiles_t), width = min(8, tiles_n - 8 * band);
    const int in_band = o - band * 8 * tiles_t;
    const int n0 = (8 * band + in_band % width) * GT_BN, t0 = in_band / width * GT_BT;
    const int K = a.K, stages = (K + GT_KB - 1) / GT_KB;

    // copy i of this wave: 16 rows x 64 bytes from row 16 (6 wave + i) of the stage on (tokens, then weights)
    uint32_t off[GT_COPIES];
    const int piece = (lane % 4) ^ (lane / 16);
    const __amdgpu_buffer_rsrc_t xr = buf_rsrc(a.x + (int64_t)t0 * K), wr = buf_rsrc(a.w + (int64_t)n0 * K);
#pragma unroll
    for (int i = 0; i < GT_COPIES; i++) {
        const int row = 16 * (GT_COPIES * wave + i) + lane / 4;
        const int clamped = row < GT_BT ? min(row, a.T - 1 - t0) : min(row - GT_BT, a.N - 1 - n0);
        off[i] = (uint32_t)clamped * K + 16 * piece;
    }
    const auto copy = [&](int s) {
        uint8_t* const dst = lds + (s % GT_RING) * GT_STAGE + GT_COPIES * 1024 * wave;
        if (64 * s + 64 <= K) {
#pragma unroll
            for (int i = 0; i < GT_COPIES; i++)
                b2l(GT_COPIES * wave + i < GT_A / 1024 ? xr : wr, dst + 1024 * i, off[i], 64 * s);
        } else {  // the reduction ends inside the stage: zeros behind it
#pragma unroll
            for (int i = 0; i < GT_COPIES; i++) {
                const int8_t* const base =
                    GT_COPIES * wave + i < GT_A / 1024 ? a.x + (int64_t)t0 * K : a.w + (int64_t)n0 * K;
                g2l16(64 * s + 16 * piece < K ? base + off[i] + 64 * s : i8_zeros, dst + 1024 * i);
            }
        }
    };
    v16i_t acc[2][4];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = v16i_t{};
    // this lane's rows of the wave's tokens and channels; rows 32 apart are 2 KB apart
    const int wt = wave % 2, wn = wave / 2;
    const uint32_t a_row = lds_off(lds) + (uint32_t)(64 * wt + lr) * GT_KB;
    const uint32_t b_row = lds_off(lds) + GT_A + (uint32_t)(128 * wn + lr) * GT_KB;
    const uint32_t p0 = 16 * ((0 + h) ^ (lr / 4 % 4)), p1 = 16 * ((2 + h) ^ (lr / 4 % 4));

    copy(0);
    if (stages > 1) copy(1);
    for (int s = 0; s < stages; s++) {
        wait_copies<GT_COPIES, 1>(stages - 1 - s);  // this stage's are there, the next one's may be on their way
        __syncthreads();                            // the others' too; all have read stage s - 1 out
        if (s + 2 < stages) copy(s + 2);
        const uint32_t slot = (uint32_t)(s % GT_RING) * GT_STAGE;
        v4i_t af[2][2], bf[2][4];
        const auto read = [&](int q, uint32_t p) {
            const uint32_t ab = a_row + slot + p, bb = b_row + slot + p;
            af[q][0] = lds_b128_at<0>(ab);
            bf[q][0] = lds_b128_at<0>(bb);
            bf[q][1] = lds_b128_at<2048>(bb);
            af[q][1] = lds_b128_at<2048>(ab);
            bf[q][2] = lds_b128_at<4096>(bb);
            bf[q][3] = lds_b128_at<6144>(bb);
        };
        const auto pin = [&](int q) {
            lds_pin(af[q][0]), lds_pin(af[q][1]);
            lds_pin(bf[q][0]), lds_pin(bf[q][1]), lds_pin(bf[q][2]), lds_pin(bf[q][3]);
        };
        const auto multiply = [&](int q) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[q][i], bf[q][j], acc[i][j], 0, 0, 0);
        };
        read(0, p0);
        read(1, p1);
        lds_wait_upto<6>();
        pin(0);
        multiply(0);
        lds_wait_upto<0>();
        pin(1);
        multiply(1);
    }
    float wscale[4];
    int n[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        n[j] = n0 + 128 * wn + 32 * j + lr;
        wscale[j] = a.ws[min(n[j], a.N - 1)];
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int v = 0; v < 16; v++) {
            const int t = t0 + 64 * wt + 32 * i + 8 * (v / 4) + 4 * h + v % 4;
            if (t >= a.T) continue;
            const float xs = a.xs[t];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (n[j] >= a.N) continue;
                const int64_t at = (int64_t)t * a.N + n[j];
                float y = (float)acc[i][j][v] * xs * wscale[j];
                if (a.resid) y += a.resid[at];
                a.out[at] = y;
            }
        }
}

size_t gemm_i8_ws_bytes(int, int, int) { return 16; }

template <int NT, int TT, int D>
static void stream(const GemmI8Args& a, hipStream_t s) {
    const int tiles_n = (a.N + 16 * NT - 1) / (16 * NT);
    const int64_t n = (int64_t)tiles_n * ((a.T + 16 * TT - 1) / (16 * TT)), gx = n < 1 << 22 ? n : 1 << 22;
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));  // fewer than 2^32 threads along x
    hipLaunchKernelGGL((gemm_i8_stream_kernel<NT, TT, D>), grid, dim3(WAVE * GS_WAVES), 0, s, a, tiles_n);
}

hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s) {
    const int64_t tiles = (int64_t)((a.N + GT_BN - 1) / GT_BN) * ((a.T + GT_BT - 1) / GT_BT);
    if (a.T > 64 && tiles >= 200) {
        const int64_t per = (tiles + 7) / 8;
        hipLaunchKernelGGL(gemm_i8_tile_kernel, dim3((unsigned)(8 * per)), dim3(WAVE * GT_WAVES), 0, s, a,
                           (a.N + GT_BN - 1) / GT_BN, (int)tiles);
    } else if (a.T > 32) {
        stream<4, 4, 2>(a, s);
    } else if (a.T > 16) {
        a.N >= 32768 ? stream<4, 2, 4>(a, s) : stream<1, 2, 6>(a, s);
    } else {
        a.N >= 32768 ? stream<4, 1, 4>(a, s) : stream<1, 1, 8>(a, s);
    }
    return hipGetLastError();
}

}  // namespace hy
