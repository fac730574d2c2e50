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

// ---------------------------------------------------------------- products
// The simple form: a wave per 32 tokens x 32 channels, operands straight from memory.  Lane l of
// v_mfma_i32_32x32x32_i8 holds 16 bytes of row l % 32 of A and of B at k offset 16 (l / 32); result
// v is A's row 8 (v / 4) + 4 (l / 32) + v % 4, B's row l % 32.  A is the weights, so a lane has
// four neighbouring channels of one token.
__global__ __launch_bounds__(256) void gemm_i8_simple_kernel(GemmI8Args a) {
    const int lane = threadIdx.x % WAVE, lr = lane % 32, h = lane / 32;
    const int tiles_n = (a.N + 31) / 32;
    const int64_t tile = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + threadIdx.x / WAVE;
    if (tile >= (int64_t)tiles_n * ((a.T + 31) / 32)) return;
    const int n0 = (int)(tile % tiles_n) * 32, t0 = (int)(tile / tiles_n) * 32;
    const int8_t* const w = a.w + (int64_t)min(n0 + lr, a.N - 1) * a.K;
    const int8_t* const x = a.x + (int64_t)min(t0 + lr, a.T - 1) * a.K;
    v16i_t acc = {};
    for (int k0 = 0; k0 < a.K; k0 += 32) {
        const int k = k0 + 16 * h;
        v4i_t wf = {}, xf = {};
        if (k < a.K) {
            wf = *reinterpret_cast<const v4i_t*>(w + k);
            xf = *reinterpret_cast<const v4i_t*>(x + k);
        }
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf, xf, acc, 0, 0, 0);
    }
    const int t = t0 + lr;
    if (t >= a.T) return;
    const float xs = a.xs[t];
#pragma unroll
    for (int v = 0; v < 16; v++) {
        const int n = n0 + 8 * (v / 4) + 4 * h + v % 4;
        if (n >= a.N) continue;
        const int64_t at = (int64_t)t * a.N + n;
        float y = (float)acc[v] * xs * a.ws[n];
        if (a.resid) y += a.resid[at];
        a.out[at] = y;
    }
}

size_t gemm_i8_ws_bytes(int, int, int) { return 16; }

hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s) {
    const int64_t n = ((int64_t)((a.N + 31) / 32) * ((a.T + 31) / 32) + 3) / 4, gx = n < 1 << 22 ? n : 1 << 22;
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));  // fewer than 2^32 threads along x
    hipLaunchKernelGGL(gemm_i8_simple_kernel, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace hy
