// hy_int8.hpp -- serving in 8 bits: arguments of the kernels, launchers, the quantizer.
#pragma once
#include "../../include/hy_int8.h"
#include "hy_paged.hpp"

namespace hy {

// hy_paged_cache_i8 with its strides filled in
struct PagedViewI8 {
    PagedView c;
    float* ks;
    float* vs;
    int bshift;  // block = 1 << bshift
};

// codes of a group whose largest magnitude has the given bits: d, and 1 / d (0: all codes 0)
struct QuantScale {
    float d, inv;
};
__device__ __forceinline__ QuantScale quant_scale(uint32_t big) {
    if (big >= 0x7f800000u) return {__builtin_nanf(""), 0.0f};
    const float d = __uint_as_float(big) / 127.0f;
    if (d < 0x1p-126f) return {0.0f, 0.0f};
    return {d, 1.0f / d};
}
// the codes of four values, packed: x * inv rounded to f32; adding 1.5 x 2^23 rounds that to the
// nearest whole number, ties to even, whose low byte is the code.  inv 0: codes 0, whatever x
__device__ __forceinline__ uint32_t quant4(float x0, float x1, float x2, float x3, float inv) {
    constexpr float M = 12582912.0f;
    const uint32_t a = __float_as_uint(x0 * inv + M), b = __float_as_uint(x1 * inv + M);
    const uint32_t c = __float_as_uint(x2 * inv + M), d = __float_as_uint(x3 * inv + M);
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return inv == 0.0f ? 0u : lo | hi;
}

hipError_t launch_quantize_rows(const float* x, int rows, int cols, int8_t* codes, float* scales, hipStream_t s);

struct GemmI8Args {
    const int8_t* x;      // [T][K]
    const float* xs;      // [T]
    const int8_t* w;      // [N][K]
    const float* ws;      // [N]
    const float* resid;   // [T][N] or null
    float* out;           // [T][N]
    int T, K, N;
    const float* xf;      // the tokens in f32, of calls that gemm_i8_takes_f32; x and xs are not read then
};
bool gemm_i8_takes_f32(const GemmI8Args& a);
hipError_t launch_gemm_i8(const GemmI8Args& a, hipStream_t s);

hipError_t launch_paged_append_i8(const PagedAppendArgs& a, const PagedViewI8& v, hipStream_t s);

// host checks and calls that the C entries share (hy_int8_capi.hip)
int paged_cache_i8_check(const hy_paged_cache_i8* cache, uint32_t n_heads, PagedViewI8* out);
int paged_ws_i8_check(const hy_paged_batch* b, uint32_t n_heads, const PagedViewI8& v, const void* ws, size_t ws_bytes);
int paged_attention_i8(const float* q, uint32_t n_heads, const PagedViewI8& v, const hy_paged_batch* b, float scale,
                       float* out, void* ws, size_t ws_bytes, hipStream_t s);

hipError_t launch_paged_attn_i8(const PagedAttnArgs& a, int max_new, hipStream_t s);
size_t paged_attn_i8_ws_bytes(int n_req, int max_new, int G, int nkv, int hd);

}  // namespace hy
