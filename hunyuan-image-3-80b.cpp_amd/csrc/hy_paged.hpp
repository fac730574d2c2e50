// hy_paged.hpp -- paged serving: arguments of the kernels, launchers, and what the C ABI of
// the calls shares.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hy_paged.h"

namespace hy {

constexpr int PG_MAX_REQ = 4096;

// hy_paged_cache with its strides filled in
struct PagedView {
    void* k;
    void* v;
    int64_t page_stride, head_stride, token_stride;  // elements
    int type, n_pages, shift, nkv, hd;               // page_size = 1 << shift
};

struct PagedViewI8;  // hy_int8.hpp

struct PagedPlanArgs {
    const int* cached;
    const int* add;
    int n_req, n_rows, shift, max_pages, n_pages;
    int* table;
    const int* held;
    int* held_out;
    int* free_;
    const int* n_free;
    int* n_free_out;
    int* q_start;
    int* kv_len;
    int* positions;
    int* slots;
    int* status;
};
hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t s);

constexpr int PG_MAX_HD = 128;
struct PagedAppendArgs {
    const float* qkv;
    int n_rows, nh;
    PagedView c;
    const int* positions;
    const int* slots;
    const float* cos_t;  // tables [n_pos][hd], or null
    const float* sin_t;
    int n_pos;
    int rotate;          // 0: no rotation; 1: by freq; 2: by the tables
    const float* q_norm;
    const float* k_norm;
    float eps;
    float* q;
    float* merged;       // of a layer: the attention's output [rows][nh][hd]; null: rows without a slot are
    const int* row_end;  // left alone; and the first row that belongs to nobody
    double freq[PG_MAX_HD / 2];  // turns per position of pair i: theta^(-2i / hd) / (2 pi)
};
hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s);

struct PagedAttnArgs {
    const float* q;
    float* out;
    PagedView c;
    int nh;
    int n_req, n_rows, max_pages;
    const int* q_start;
    const int* kv_len;
    const int* table;
    const int* seen;  // or null: causal
    float scale;
    float* ws;
    const float* ks;  // of an 8-bit cache: the scales, of blocks of 1 << bshift positions
    const float* vs;
    int bshift;
};
hipError_t launch_paged_attn(const PagedAttnArgs& a, int max_new, hipStream_t s);
size_t paged_attn_ws_bytes(int type, int n_req, int max_new, int G, int hd);

struct VerifyArgs {
    const float* logits;
    const float* draft;  // or null
    const int* ids;
    const int* q_start;
    int n_req, n_rows, max_new, vocab;
    const float* temp;   // or null
    const float* u_accept;
    const float* u_sample;
    int* accepted;
    int* tokens;
    void* ws;
};
hipError_t launch_verify_drafts(const VerifyArgs& a, hipStream_t s);
size_t verify_ws_bytes(int n_req, int n_rows, int vocab);

// host checks shared by the calls (hy_paged_capi.hip): HY_OK, or a status with the last error set
// only: the one type that is taken; 0: those of hy_paged.h
int paged_cache_check(const hy_paged_cache* cache, uint32_t n_heads, PagedView* out, int only = 0);
int paged_batch_check(const hy_paged_batch* b, const PagedView& c, bool writes);
int paged_rotary_check(float theta, const float* cos_t, const float* sin_t, uint32_t n_pos, float eps);
int paged_append(const float* qkv, uint32_t n_rows, uint32_t n_heads, const PagedView& c, const int32_t* positions,
                 const int32_t* slots, float theta, const float* cos_t, const float* sin_t, uint32_t n_pos,
                 const float* q_norm, const float* k_norm, float eps, float* q, hipStream_t s,
                 float* merged = nullptr, const int32_t* row_end = nullptr, const PagedViewI8* i8 = nullptr);
size_t paged_batch_ws(const hy_paged_batch* b, uint32_t n_heads, const PagedView& c);
int paged_ws_check(const hy_paged_batch* b, uint32_t n_heads, const PagedView& c, const void* ws, size_t ws_bytes);
int paged_attention(const float* q, uint32_t n_heads, const PagedView& c, const hy_paged_batch* b, float scale,
                    float* out, void* ws, size_t ws_bytes, hipStream_t s);

}  // namespace hy
