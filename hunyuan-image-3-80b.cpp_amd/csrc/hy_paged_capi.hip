// hy_paged_capi.hip -- the C ABI of paged serving (include/hy_paged.h), the calls without a
// context: argument checks and launches.  hy_attn_forward_paged and hy_model_forward_paged
// are in hy_attn_capi.hip, with their contexts.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "hy_paged.hpp"

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

int page_shift(uint32_t page_size) {
    if (page_size < 8 || page_size > 4096 || (page_size & (page_size - 1))) return -1;
    return __builtin_ctz(page_size);
}

// sizes that the plan and the batches share
int sizes_check(uint32_t n_req, uint32_t n_rows, uint32_t page_size, uint32_t max_pages, uint32_t n_pages) {
    if (n_req == 0 || n_req > (uint32_t)hy::PG_MAX_REQ)
        return fail(HY_ERR_INVALID, "n_req=%u must be in 1..%d", n_req, hy::PG_MAX_REQ);
    if (n_rows == 0 || n_rows > 1u << 20) return fail(HY_ERR_INVALID, "n_rows=%u must be in 1..2^20", n_rows);
    if (page_shift(page_size) < 0)
        return fail(HY_ERR_UNSUPPORTED, "page_size=%u: the kernels take powers of two, 8..4096", page_size);
    if (n_pages == 0 || (uint64_t)n_pages * page_size >= 1ull << 31)
        return fail(HY_ERR_INVALID, "n_pages=%u of %u positions: 1 page at least, fewer than 2^31 positions", n_pages,
                    page_size);
    if (max_pages == 0 || (uint64_t)max_pages * page_size > 1ull << 30)
        return fail(HY_ERR_INVALID, "max_pages=%u of %u positions: 1 page at least, 2^30 positions at most", max_pages,
                    page_size);
    return HY_OK;
}

int verify_check(uint32_t n_req, uint32_t n_rows, uint32_t vocab) {
    if (n_req == 0 || n_req > (uint32_t)hy::PG_MAX_REQ || n_rows == 0 || n_rows > 1u << 20 || vocab == 0 ||
        vocab > 1u << 22)
        return fail(HY_ERR_INVALID, "n_req=%u n_rows=%u vocab=%u out of range", n_req, n_rows, vocab);
    if ((uint64_t)n_rows * vocab > 1ull << 36)  // 256 GiB of logits, the most that one launch covers
        return fail(HY_ERR_UNSUPPORTED, "n_rows=%u of vocab=%u: 2^36 logits at most", n_rows, vocab);
    return HY_OK;
}

}  // namespace

namespace hy {

int paged_cache_check(const hy_paged_cache* c, uint32_t n_heads, PagedView* out) {
    if (!c) return fail(HY_ERR_INVALID, "null cache");
    if (!c->k_dev || !c->v_dev) return fail(HY_ERR_INVALID, "null cache pointer");
    if (c->type != HY_TYPE_F32 && c->type != HY_TYPE_F16 && c->type != HY_TYPE_BF16)
        return fail(HY_ERR_UNSUPPORTED, "cache type %d: F32, F16 or BF16 expected", c->type);
    const int shift = page_shift(c->page_size);
    if (shift < 0)
        return fail(HY_ERR_UNSUPPORTED, "page_size=%u: the kernels take powers of two, 8..4096", c->page_size);
    if (c->n_pages == 0 || (uint64_t)c->n_pages * c->page_size >= 1ull << 31)
        return fail(HY_ERR_INVALID, "n_pages=%u of %u positions: 1 page at least, fewer than 2^31 positions",
                    c->n_pages, c->page_size);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(HY_ERR_UNSUPPORTED, "head_dim=%u: the kernels take 64 or 128", c->head_dim);
    if (c->n_kv_heads == 0 || n_heads == 0 || n_heads % c->n_kv_heads || n_heads > 1024)
        return fail(HY_ERR_INVALID, "n_heads=%u n_kv_heads=%u: a multiple, 1024 at most", n_heads, c->n_kv_heads);
    uint64_t ps = c->page_stride, hs = c->head_stride, ts = c->token_stride;
    if (!ps && !hs && !ts) {
        ts = c->head_dim;
        hs = ts * c->page_size;
        ps = hs * c->n_kv_heads;
    }
    const uint64_t unit = c->type == HY_TYPE_F32 ? 4 : 8;  // 16 bytes
    if (ts < c->head_dim || hs < c->head_dim || ps < c->head_dim)
        return fail(HY_ERR_INVALID, "cache strides %llu / %llu / %llu below head_dim", (unsigned long long)ps,
                    (unsigned long long)hs, (unsigned long long)ts);
    if (ps % unit || hs % unit || ts % unit || !aligned(c->k_dev, 16) || !aligned(c->v_dev, 16))
        return fail(HY_ERR_INVALID, "cache pointers and strides must be multiples of 16 bytes");
    if (ps >> 40 || hs >> 40) return fail(HY_ERR_INVALID, "cache stride of 2^40 or more elements");
    if (ts > 1u << 24)
        return fail(HY_ERR_UNSUPPORTED, "token_stride=%llu: 2^24 elements at most", (unsigned long long)ts);
    *out = {c->k_dev, c->v_dev, (int64_t)ps, (int64_t)hs, (int64_t)ts, c->type, (int)c->n_pages, shift,
            (int)c->n_kv_heads, (int)c->head_dim};
    return HY_OK;
}

int paged_batch_check(const hy_paged_batch* b, const PagedView& c, bool writes) {
    if (!b) return fail(HY_ERR_INVALID, "null batch");
    HY_TRY(sizes_check(b->n_req, b->n_rows, 1u << c.shift, b->max_pages, (uint32_t)c.n_pages));
    if (!b->q_start_dev || !b->kv_len_dev || !b->table_dev) return fail(HY_ERR_INVALID, "null batch array");
    if (writes && (!b->positions_dev || !b->slots_dev)) return fail(HY_ERR_INVALID, "null positions or slots");
    return HY_OK;
}

int paged_rotary_check(float theta, const float* cos_t, const float* sin_t, uint32_t n_pos, float eps) {
    if ((cos_t == nullptr) != (sin_t == nullptr)) return fail(HY_ERR_INVALID, "give both rotary tables or neither");
    if (cos_t && (n_pos == 0 || n_pos > 1u << 30)) return fail(HY_ERR_INVALID, "n_pos=%u must be in 1..2^30", n_pos);
    if (!cos_t && !(theta == 0.0f || (theta > 0.0f && std::isfinite(theta))))
        return fail(HY_ERR_INVALID, "theta=%g must be positive, or 0 for no rotation", theta);
    if (!(eps >= 0.0f)) return fail(HY_ERR_INVALID, "eps=%g must not be negative", eps);
    if (cos_t && (!aligned(cos_t, 16) || !aligned(sin_t, 16)))
        return fail(HY_ERR_INVALID, "rotary tables must be aligned to 16 bytes");
    return HY_OK;
}

int paged_append(const float* qkv, uint32_t n_rows, uint32_t n_heads, const PagedView& c, const int32_t* positions,
                 const int32_t* slots, float theta, const float* cos_t, const float* sin_t, uint32_t n_pos,
                 const float* q_norm, const float* k_norm, float eps, float* q, hipStream_t s,
                 float* merged, const int32_t* row_end) {
    if (!qkv || !positions || !slots || !q) return fail(HY_ERR_INVALID, "null pointer");
    if (n_rows == 0 || n_rows > 1u << 20) return fail(HY_ERR_INVALID, "n_rows=%u must be in 1..2^20", n_rows);
    HY_TRY(paged_rotary_check(theta, cos_t, sin_t, n_pos, eps));
    if (!aligned(qkv, 16) || !aligned(q, 16) || (q_norm && !aligned(q_norm, 16)) || (k_norm && !aligned(k_norm, 16)))
        return fail(HY_ERR_INVALID, "f32 arrays must be aligned to 16 bytes");
    PagedAppendArgs a{qkv,   (int)n_rows, (int)n_heads, c,      positions, slots, cos_t, sin_t,
                      (int)n_pos, cos_t ? 2 : theta > 0.0f ? 1 : 0, q_norm, k_norm, eps, q, merged, row_end, {}};
    if (a.rotate == 1) {  // theta^(-2 (8 p + r) / hd) as a product: 16 powers, not 64 (0.6 us of the call)
        double low[8];
        for (int r = 0; r < 8; r++) low[r] = std::pow((double)theta, -2.0 * r / c.hd) / 6.283185307179586476925;
        for (int p = 0; p < c.hd / 16; p++) {
            const double high = std::pow((double)theta, -16.0 * p / c.hd);
            for (int r = 0; r < 8; r++) a.freq[8 * p + r] = high * low[r];
        }
    }
    HIP_TRY(launch_paged_append(a, s));
    return HY_OK;
}

size_t paged_batch_ws(const hy_paged_batch* b, uint32_t n_heads, const PagedView& c) {
    return paged_attn_ws_bytes(c.type, (int)b->n_req, (int)(b->max_new < b->n_rows ? b->max_new : b->n_rows),
                               (int)n_heads / c.nkv, c.hd);
}

int paged_ws_check(const hy_paged_batch* b, uint32_t n_heads, const PagedView& c, const void* ws, size_t ws_bytes) {
    const size_t need = paged_batch_ws(b, n_heads, c);
    if (!ws || ws_bytes < need || !aligned(ws, 16))
        return fail(HY_ERR_INVALID, "workspace of %zu bytes at %p: %zu bytes aligned to 16 needed", ws_bytes, ws, need);
    return HY_OK;
}

int paged_attention(const float* q, uint32_t n_heads, const PagedView& c, const hy_paged_batch* b, float scale,
                    float* out, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!q || !out) return fail(HY_ERR_INVALID, "null q/out");
    if (!std::isfinite(scale)) return fail(HY_ERR_INVALID, "scale is not finite");
    if (!aligned(q, 16) || !aligned(out, 16)) return fail(HY_ERR_INVALID, "q and out must be aligned to 16 bytes");
    HY_TRY(paged_ws_check(b, n_heads, c, ws, ws_bytes));
    const PagedAttnArgs a{q, out, c, (int)n_heads, (int)b->n_req, (int)b->n_rows, (int)b->max_pages, b->q_start_dev,
                          b->kv_len_dev, b->table_dev, b->seen_dev, scale, static_cast<float*>(ws)};
    HIP_TRY(launch_paged_attn(a, (int)(b->max_new < b->n_rows ? b->max_new : b->n_rows), s));
    return HY_OK;
}

}  // namespace hy

extern "C" {

int hy_paged_plan(const int32_t* cached, const int32_t* add, uint32_t n_req, uint32_t n_rows, uint32_t page_size,
                  uint32_t max_pages, uint32_t n_pages, int32_t* table, const int32_t* held, int32_t* held_out,
                  int32_t* free_list, const int32_t* n_free, int32_t* n_free_out, int32_t* q_start, int32_t* kv_len,
                  int32_t* positions, int32_t* slots, int32_t* status, void* stream) {
    HY_TRY(sizes_check(n_req, n_rows, page_size, max_pages, n_pages));
    const void* all[] = {cached, add, table, held, held_out, free_list, n_free, n_free_out, q_start, kv_len, positions,
                         slots, status};
    for (const void* p : all)
        if (!p) return fail(HY_ERR_INVALID, "null pointer");
    const hy::PagedPlanArgs a{cached, add, (int)n_req, (int)n_rows, page_shift(page_size), (int)max_pages, (int)n_pages,
                              table, held, held_out, free_list, n_free, n_free_out, q_start, kv_len, positions, slots,
                              status};
    HIP_TRY(hy::launch_paged_plan(a, static_cast<hipStream_t>(stream)));
    return HY_OK;
}

int hy_rope_qknorm_paged(const float* qkv, uint32_t n_rows, uint32_t n_heads, const hy_paged_cache* cache,
                         const int32_t* positions, const int32_t* slots, float theta, const float* cos_t,
                         const float* sin_t, uint32_t n_pos, const float* q_norm, const float* k_norm, float eps,
                         float* q, void* stream) {
    hy::PagedView c;
    HY_TRY(hy::paged_cache_check(cache, n_heads, &c));
    return hy::paged_append(qkv, n_rows, n_heads, c, positions, slots, theta, cos_t, sin_t, n_pos, q_norm, k_norm, eps,
                            q, static_cast<hipStream_t>(stream));
}

size_t hy_paged_attention_ws(uint32_t n_heads, const hy_paged_cache* cache, const hy_paged_batch* batch) {
    hy::PagedView c;
    if (hy::paged_cache_check(cache, n_heads, &c) != HY_OK || hy::paged_batch_check(batch, c, false) != HY_OK) return 0;
    return hy::paged_batch_ws(batch, n_heads, c);
}

int hy_paged_attention(const float* q, uint32_t n_heads, const hy_paged_cache* cache, const hy_paged_batch* batch,
                       float scale, float* out, void* ws, size_t ws_bytes, void* stream) {
    hy::PagedView c;
    HY_TRY(hy::paged_cache_check(cache, n_heads, &c));
    HY_TRY(hy::paged_batch_check(batch, c, false));
    return hy::paged_attention(q, n_heads, c, batch, scale, out, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t hy_verify_drafts_ws(uint32_t n_req, uint32_t n_rows, uint32_t vocab) {
    if (verify_check(n_req, n_rows, vocab) != HY_OK) return 0;
    return hy::verify_ws_bytes((int)n_req, (int)n_rows, (int)vocab);
}

int hy_verify_drafts(const float* logits, const float* draft_probs, const int32_t* ids, const int32_t* q_start,
                     uint32_t n_req, uint32_t n_rows, uint32_t max_new, uint32_t vocab, const float* temperature,
                     const float* u_accept, const float* u_sample, int32_t* accepted, int32_t* tokens, void* ws,
                     size_t ws_bytes, void* stream) {
    if (!logits || !ids || !q_start || !u_accept || !u_sample || !accepted || !tokens)
        return fail(HY_ERR_INVALID, "null pointer");
    if (max_new == 0 || max_new > 1u << 20) return fail(HY_ERR_INVALID, "max_new=%u must be in 1..2^20", max_new);
    HY_TRY(verify_check(n_req, n_rows, vocab));
    const size_t need = hy::verify_ws_bytes((int)n_req, (int)n_rows, (int)vocab);
    if (!ws || ws_bytes < need || !aligned(ws, 16))
        return fail(HY_ERR_INVALID, "workspace of %zu bytes at %p: %zu bytes aligned to 16 needed", ws_bytes, ws, need);
    const hy::VerifyArgs a{logits, draft_probs, ids, q_start, (int)n_req, (int)n_rows, (int)max_new, (int)vocab,
                           temperature, u_accept, u_sample, accepted, tokens, ws};
    HIP_TRY(hy::launch_verify_drafts(a, static_cast<hipStream_t>(stream)));
    return HY_OK;
}

}  // extern "C"
