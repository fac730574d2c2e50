/*
 * hy_int8.h -- C ABI of serving in 8 bits on the MI355X (gfx950): products of tokens and
 * weights in 8-bit integers with a scale per token and per output channel, a paged key /
 * value cache of 8-bit integers with a scale per block of tokens and head, and attention of
 * ragged batches over it.
 *
 * Conventions as hy_paged.h: device pointers, `stream` = hipStream_t as void* (NULL: default
 * stream), HY_OK or a negative hy_status with hy_last_error() set, arguments checked before
 * anything is launched; calls only queue work on their stream, allocate nothing, and can be
 * captured into a graph; calls that overlap in time need workspaces of their own.
 * Calls without a context run on the calling thread's current device.
 *
 * A group of values (a token, a weight row, a block of tokens of one head) is held as whole
 * numbers -127..127 and one scale:
 *   d = a / 127, a the group's largest magnitude; i = 1 / d; code = x * i, each rounded to
 *   f32, the last one to the nearest whole number then, ties to even;
 *   d = 0 and codes 0 where d would be below 2^-126; d = NaN and codes 0 where a value is
 *   infinite or NaN.
 * The value held is code * d.  No counterpart in the reference, which computes in f32 but for
 * the experts' GGUF blocks (a scale per 32 values along the reduction: hy_moe.h).
 */
#ifndef HY_INT8_H
#define HY_INT8_H

#include <stddef.h>
#include <stdint.h>

#include "hy_attn.h"
#include "hy_moe.h"
#include "hy_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* cache type of the pools below (ggml.h numbering); the calls of hy_paged.h refuse it */
enum { HY_TYPE_I8 = 24 };

/* ---- products ---------------------------------------------------------------- */

/* codes [rows][cols] and scales [rows] of the rows of x [rows][cols], as above: weights, once,
 * or tokens.  cols a multiple of 16 below 2^17, rows 1..2^24; x and codes aligned to 16 bytes. */
int hy_quantize_rows_i8(const float* x_dev, uint32_t rows, uint32_t cols, int8_t* codes_dev, float* scales_dev,
                        void* stream);

/* out[t][n] = (sum_k x[t][k] w[n][k]) * x_scale[t] * w_scale[n] (+ resid[t][n] when resid_dev is
 * not NULL), in that order; the sum is exact (32-bit integers, any codes -128..127).  x
 * [T][hidden] and w [n_out][hidden] codes, out and resid f32 [T][n_out]; out may be resid_dev
 * itself.  hidden a multiple of 16 below 2^17, T 1..2^20, n_out 1..2^22; x and w aligned to 16
 * bytes, all other arrays to 4.  ws_dev: hy_gemm_i8_ws bytes (0 for bad arguments, 16 at
 * least), aligned to 16 bytes, contents indifferent. */
size_t hy_gemm_i8_ws(uint32_t T, uint32_t hidden, uint32_t n_out);
int hy_gemm_i8(const int8_t* x_dev, const float* x_scale_dev, const int8_t* w_dev, const float* w_scale_dev,
               const float* resid_dev, uint32_t T, uint32_t hidden, uint32_t n_out, float* out_dev, void* ws_dev,
               size_t ws_bytes, void* stream);

/* hy_quantize_rows_i8 of x [T][hidden] f32, then hy_gemm_i8: the 8-bit form of hy_lm_head_f32.  A
 * token with an infinity or NaN has NaN in all its outputs, other tokens are not touched by
 * it.  x aligned to 16 bytes; ws_dev: hy_linear_i8_ws bytes (which hold the codes). */
size_t hy_linear_i8_ws(uint32_t T, uint32_t hidden, uint32_t n_out);
int hy_linear_i8(const float* x_dev, const int8_t* w_dev, const float* w_scale_dev, const float* resid_dev, uint32_t T,
                 uint32_t hidden, uint32_t n_out, float* out_dev, void* ws_dev, size_t ws_bytes, void* stream);

/* ---- the cache --------------------------------------------------------------- */

/* A pool of pages (hy_paged_cache, type HY_TYPE_I8: elements are bytes, pointers and strides
 * multiples of 16) with scales.  Positions of a page fall into blocks of `block`
 * consecutive ones; the scale of block b of kv head g of page p is element
 * (p * n_kv_heads + g) * (page_size / block) + b of k_scale_dev / v_scale_dev. */
typedef struct {
    hy_paged_cache pool;
    float* k_scale_dev;
    float* v_scale_dev;
    uint32_t block;              /* a power of two, 8..page_size */
    uint64_t layer_scale_stride; /* floats from one layer's scales to the next (calls with a context;
                                  * looked at only where there are several layers) */
} hy_paged_cache_i8;

/* hy_rope_qknorm_paged with the write of codes.  A key's norm(rotate(k)) is computed in
 * 64 bits and rounded to f32 once, so that its code does not depend on the order of a sum.  The rows of
 * a call that fall into one block of one page have to be neighbours among the rows, in the order
 * of their positions and without gaps, as hy_paged_plan gives them.  A block whose first position
 * is among them begins anew: its scale is theirs, its positions that are not written become
 * 0.  In any other block the scale d' becomes the larger of what it was and d of the rows;
 * where it grows, the codes held become code * (d / d'), both rounded to f32, to the nearest
 * whole number, ties to even.  So tokens that came one by one are held at steps of up to d'
 * with an error of half a step per growth (about as many as the logarithm of the block's
 * length), and a row that is written again (a draft that was not taken) does not take
 * the growth back.  A block whose rows hold an infinity or NaN has a scale of NaN until it begins
 * anew.
 * Rows that break the order give codes and scales of no meaning in the blocks they name, and
 * touch nothing else. */
int hy_rope_qknorm_paged_i8(const float* qkv_dev, uint32_t n_rows, uint32_t n_heads, const hy_paged_cache_i8* cache,
                            const int32_t* positions_dev, const int32_t* slots_dev, float theta, const float* cos_dev,
                            const float* sin_dev, uint32_t n_pos, const float* q_norm_dev, const float* k_norm_dev,
                            float eps, float* q_dev, void* stream);

/* hy_paged_attention over such a cache: k_j and v_j are code * scale.  Products and sums have f32
 * accuracy, relative to the largest elements of q, of a key and of a value row; products of a
 * weight and its value's scale are taken to 2^-31 of the row's largest.  Scales are not negative;
 * keys' are of any size as long as scores stay in f32's range, values' from 2^-59 to 2^34 (below that
 * a value may count as 0, which is 2^-52 at most; larger ones are not defined).  A row that sees a
 * key of a block whose key or value scale is infinite or NaN is NaN; a key that a row does not
 * see does not touch it, whatever its block's scales.  ws_dev: hy_paged_attention_i8_ws bytes (0 for bad
 * arguments), aligned to 16 bytes, contents indifferent. */
size_t hy_paged_attention_i8_ws(uint32_t n_heads, const hy_paged_cache_i8* cache, const hy_paged_batch* batch);
int hy_paged_attention_i8(const float* q_dev, uint32_t n_heads, const hy_paged_cache_i8* cache,
                          const hy_paged_batch* batch, float scale, float* out_dev, void* ws_dev, size_t ws_bytes,
                          void* stream);

/* ---- the layer and the backbone ------------------------------------------------ */

/* Holds `layer`'s projections (hy_model_quantize_i8: every layer's, and the lm_head) in 8 bits
 * besides f32: the two calls below take those from then on, until the weights are loaded anew.
 * A graph keeps the form it was captured with: over 8 bits it goes on with the codes there are, whatever is
 * loaded behind it, until these calls are made again, which put the new ones in the same place.
 * Allocates, and waits for the device; not while a stream is captured. */
int hy_attn_quantize_i8(hy_attn_ctx* ctx, uint32_t layer);
int hy_model_quantize_i8(hy_model_ctx* ctx);

/* hy_attn_forward_paged and hy_model_forward_paged over a cache of 8 bits, with the products in
 * f32, or in 8 bits of weights that are held so.  Of several layers the pools lie as there,
 * the scales layer_scale_stride floats apart, at least as many as one layer has. */
int hy_attn_forward_paged_i8(hy_attn_ctx* ctx, uint32_t layer, const float* x_dev, const hy_paged_cache_i8* cache,
                             const hy_paged_batch* batch, const float* cos_dev, const float* sin_dev, uint32_t n_pos,
                             float* out_dev, void* ws_dev, size_t ws_bytes, void* stream);
int hy_model_forward_paged_i8(hy_model_ctx* ctx, const int32_t* ids_dev, const hy_paged_cache_i8* cache,
                              const hy_paged_batch* batch, float* logits_dev, void* ws_dev, size_t ws_bytes,
                              void* stream);

#ifdef __cplusplus
}
#endif
#endif
