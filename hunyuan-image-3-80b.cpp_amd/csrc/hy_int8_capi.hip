// hy_int8_capi.hip -- the C ABI of serving in 8 bits (include/hy_int8.h): argument checks and launches.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "hy_int8.hpp"

namespace hy {
int set_last_error(int code, const std::string& msg);  // hy_capi.hip
}

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return hy::set_last_error(code, buf);
}

#define HIP_TRY(expr)                                                                                    \
    do {                                                                                                 \
        hipError_t e_ = (expr);                                                                          \
        if (e_ != hipSuccess) return fail(HY_ERR_HIP, "%s: %s (%s:%d)", #expr, hipGetErrorString(e_),   \
                                          __FILE__, __LINE__);                                           \
    } while (0)

#define HY_TRY(expr)                \
    do {                            \
        int r_ = (expr);            \
        if (r_ != HY_OK) return r_; \
    } while (0)

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int width_check(const char* name, uint32_t n) {
    if (n == 0 || n % 16 || n >= 1u << 17)
        return fail(HY_ERR_INVALID, "%s=%u must be a positive multiple of 16 below 2^17", name, n);
    return HY_OK;
}

int gemm_sizes_check(uint32_t T, uint32_t hidden, uint32_t n_out) {
    HY_TRY(width_check("hidden", hidden));
    if (T == 0 || T > 1u << 20) return fail(HY_ERR_INVALID, "T=%u must be in 1..2^20", T);
    if (n_out == 0 || n_out > 1u << 22) return fail(HY_ERR_INVALID, "n_out=%u must be in 1..2^22", n_out);
    return HY_OK;
}

int ws_check(const void* ws, size_t ws_bytes, size_t need) {
    if (!ws || ws_bytes < need || !aligned(ws, 16))
        return fail(HY_ERR_INVALID, "workspace of %zu bytes at %p: %zu bytes aligned to 16 needed", ws_bytes, ws, need);
    return HY_OK;
}

size_t al16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

namespace hy {

int paged_cache_i8_check(const hy_paged_cache_i8* cache, uint32_t n_heads, PagedViewI8* out) {
    if (!cache) return fail(HY_ERR_INVALID, "null cache");
    HY_TRY(paged_cache_check(&cache->pool, n_heads, &out->c, HY_TYPE_I8));
    if (!cache->k_scale_dev || !cache->v_scale_dev) return fail(HY_ERR_INVALID, "null scales");
    if (!aligned(cache->k_scale_dev, 4) || !aligned(cache->v_scale_dev, 4))
        return fail(HY_ERR_INVALID, "scales must be aligned to 4 bytes");
    const uint32_t b = cache->block;
    if (b < 8 || b > cache->pool.page_size || (b & (b - 1)))
        return fail(HY_ERR_UNSUPPORTED, "block=%u: the kernels take powers of two, 8..page_size=%u", b,
                    cache->pool.page_size);
    out->ks = cache->k_scale_dev;
    out->vs = cache->v_scale_dev;
    out->bshift = __builtin_ctz(b);
    return HY_OK;
}

static size_t paged_batch_i8_ws(const hy_paged_batch* b, uint32_t n_heads, const PagedViewI8& v) {
    return paged_attn_i8_ws_bytes((int)b->n_req, (int)(b->max_new < b->n_rows ? b->max_new : b->n_rows),
                                  (int)n_heads / v.c.nkv, v.c.nkv, v.c.hd);
}

int paged_ws_i8_check(const hy_paged_batch* b, uint32_t n_heads, const PagedViewI8& v, const void* ws,
                      size_t ws_bytes) {
    return ws_check(ws, ws_bytes, paged_batch_i8_ws(b, n_heads, v));
}

int paged_attention_i8(const float* q, uint32_t n_heads, const PagedViewI8& v, const hy_paged_batch* b, float scale,
                       float* out, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!q || !out) return fail(HY_ERR_INVALID, "null q/out");
    if (!std::isfinite(scale)) return fail(HY_ERR_INVALID, "scale is not finite");
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(HY_ERR_INVALID, "q and out must be aligned to 16 bytes");
    HY_TRY(paged_ws_i8_check(b, n_heads, v, ws, ws_bytes));
    const PagedAttnArgs a{q, out, v.c, (int)n_heads, (int)b->n_req, (int)b->n_rows, (int)b->max_pages, b->q_start_dev,
                          b->kv_len_dev, b->table_dev, b->seen_dev, scale, static_cast<float*>(ws), v.ks, v.vs,
                          v.bshift};
    HIP_TRY(launch_paged_attn_i8(a, (int)(b->max_new < b->n_rows ? b->max_new : b->n_rows), s));
    return HY_OK;
}

}  // namespace hy

extern "C" {

int hy_quantize_rows_i8(const float* x, uint32_t rows, uint32_t cols, int8_t* codes, float* scales, void* stream) {
    HY_TRY(width_check("cols", cols));
    if (rows == 0 || rows > 1u << 24) return fail(HY_ERR_INVALID, "rows=%u must be in 1..2^24", rows);
    if (!x || !codes || !scales) return fail(HY_ERR_INVALID, "null pointer");
    if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(scales, 4))
        return fail(HY_ERR_INVALID, "x and codes must be aligned to 16 bytes, scales to 4");
    HIP_TRY(hy::launch_quantize_rows(x, (int)rows, (int)cols, codes, scales, static_cast<hipStream_t>(stream)));
    return HY_OK;
}

size_t hy_gemm_i8_ws(uint32_t T, uint32_t hidden, uint32_t n_out) {
    if (gemm_sizes_check(T, hidden, n_out) != HY_OK) return 0;
    return 16;  // the present kernels need none
}

int hy_gemm_i8(const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, const float* resid,
               uint32_t T, uint32_t hidden, uint32_t n_out, float* out, void* ws, size_t ws_bytes, void* stream) {
    HY_TRY(gemm_sizes_check(T, hidden, n_out));
    if (!x || !x_scale || !w || !w_scale || !out) return fail(HY_ERR_INVALID, "null pointer");
    if (!aligned(x, 16) || !aligned(w, 16)) return fail(HY_ERR_INVALID, "x and w must be aligned to 16 bytes");
    if (!aligned(x_scale, 4) || !aligned(w_scale, 4) || !aligned(out, 4) || !aligned(resid, 4))
        return fail(HY_ERR_INVALID, "f32 arrays must be aligned to 4 bytes");
    HY_TRY(ws_check(ws, ws_bytes, hy_gemm_i8_ws(T, hidden, n_out)));
    const hy::GemmI8Args a{x, x_scale, w, w_scale, resid, out, (int)T, (int)hidden, (int)n_out, nullptr};
    HIP_TRY(hy::launch_gemm_i8(a, static_cast<hipStream_t>(stream)));
    return HY_OK;
}

// codes, scales, and the product's own
size_t hy_linear_i8_ws(uint32_t T, uint32_t hidden, uint32_t n_out) {
    if (gemm_sizes_check(T, hidden, n_out) != HY_OK) return 0;
    return (size_t)T * hidden + al16((size_t)T * 4) + hy_gemm_i8_ws(T, hidden, n_out);
}

int hy_linear_i8(const float* x, const int8_t* w, const float* w_scale, const float* resid, uint32_t T,
                 uint32_t hidden, uint32_t n_out, float* out, void* ws, size_t ws_bytes, void* stream) {
    HY_TRY(gemm_sizes_check(T, hidden, n_out));
    if (!x || !w || !w_scale || !out) return fail(HY_ERR_INVALID, "null pointer");
    if (!aligned(x, 16) || !aligned(w, 16)) return fail(HY_ERR_INVALID, "x and w must be aligned to 16 bytes");
    if (!aligned(w_scale, 4) || !aligned(out, 4) || !aligned(resid, 4))
        return fail(HY_ERR_INVALID, "f32 arrays must be aligned to 4 bytes");
    HY_TRY(ws_check(ws, ws_bytes, hy_linear_i8_ws(T, hidden, n_out)));
    int8_t* const codes = static_cast<int8_t*>(ws);
    float* const scales = reinterpret_cast<float*>(codes + (size_t)T * hidden);
    hipStream_t s = static_cast<hipStream_t>(stream);
    hy::GemmI8Args a{codes, scales, w, w_scale, resid, out, (int)T, (int)hidden, (int)n_out, nullptr};
    if (hy::gemm_i8_takes_f32(a))
        a.xf = x;
    else
        HIP_TRY(hy::launch_quantize_rows(x, (int)T, (int)hidden, codes, scales, s));
    HIP_TRY(hy::launch_gemm_i8(a, s));
    return HY_OK;
}

int hy_rope_qknorm_paged_i8(const float* qkv, uint32_t n_rows, uint32_t n_heads, const hy_paged_cache_i8* cache,
                            const int32_t* positions, const int32_t* slots, float theta, const float* cos_t,
                            const float* sin_t, uint32_t n_pos, const float* q_norm, const float* k_norm, float eps,
                            float* q, void* stream) {
    hy::PagedViewI8 v;
    HY_TRY(hy::paged_cache_i8_check(cache, n_heads, &v));
    return hy::paged_append(qkv, n_rows, n_heads, v.c, positions, slots, theta, cos_t, sin_t, n_pos, q_norm, k_norm,
                            eps, q, static_cast<hipStream_t>(stream), nullptr, nullptr, &v);
}

size_t hy_paged_attention_i8_ws(uint32_t n_heads, const hy_paged_cache_i8* cache, const hy_paged_batch* batch) {
    hy::PagedViewI8 v;
    if (hy::paged_cache_i8_check(cache, n_heads, &v) != HY_OK || hy::paged_batch_check(batch, v.c, false) != HY_OK)
        return 0;
    return hy::paged_batch_i8_ws(batch, n_heads, v);
}

int hy_paged_attention_i8(const float* q, uint32_t n_heads, const hy_paged_cache_i8* cache,
                          const hy_paged_batch* batch, float scale, float* out, void* ws, size_t ws_bytes,
                          void* stream) {
    hy::PagedViewI8 v;
    HY_TRY(hy::paged_cache_i8_check(cache, n_heads, &v));
    HY_TRY(hy::paged_batch_check(batch, v.c, false));
    return hy::paged_attention_i8(q, n_heads, v, batch, scale, out, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
