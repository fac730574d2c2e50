/*
 * hy_paged.h -- C ABI of serving many requests on the MI355X (gfx950): a key / value cache
 * in pages, the tables that map requests to pages, attention of ragged batches of new
 * tokens over it, and the verification of drafted tokens.
 *
 * Conventions as hy_moe.h: plain pointers and sizes, "dev" = device (HBM) address,
 * `stream` = hipStream_t as void* (NULL: default stream), HY_OK or a negative hy_status
 * with hy_last_error() set; arguments are checked before anything is launched.  Calls
 * without a context run on the calling thread's current device (hy_set_device), which the
 * stream and all pointers belong to.  Every call only queues work on its stream: it
 * returns without waiting, allocates nothing, and can be captured into a graph.  Calls
 * that overlap in time, captured graphs among them, need workspaces of their own, and
 * contexts of their own where they take one.
 *
 * One step of a server: hy_paged_plan (tables, slots), hy_model_forward_paged (every
 * layer: hy_rope_qknorm_paged, hy_paged_attention), hy_verify_drafts (accepted tokens).
 * Request r brought new[r] rows, of a prompt or its last token and drafts.  With
 * status[r] = 0, cached[r] grows by the rows whose tokens were given (a prompt's), and by
 * 1 + accepted for those that were verified; with any other status its rows computed
 * nothing, cached[r] stays, and they come again.  No counterpart in the reference, whose KVCache
 * (src/hunyuan_image_gen.h:179-193) holds one sequence in one piece.
 */
#ifndef HY_PAGED_H
#define HY_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "hy_attn.h"
#include "hy_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* cache types besides HY_TYPE_F32 (ggml.h numbering) */
enum { HY_TYPE_F16 = 1, HY_TYPE_BF16 = 30 };

/* A pool of n_pages pages, each page_size positions of every kv head: the value d of kv
 * head g at position i of page p is element p * page_stride + g * head_stride +
 * i * token_stride + d of k_dev / v_dev.  All three strides 0: dense
 * [page][kv head][position][head_dim].  Pointers and strides are multiples of 16 bytes;
 * the elements of different (page, head, position) do not overlap. */
typedef struct {
    void* k_dev;
    void* v_dev;
    int32_t type;          /* HY_TYPE_F32, HY_TYPE_F16 or HY_TYPE_BF16 */
    uint32_t n_pages;      /* n_pages * page_size < 2^31 */
    uint32_t page_size;    /* a power of two, 8..4096 */
    uint32_t n_kv_heads;
    uint32_t head_dim;     /* 64 or 128 */
    uint64_t page_stride;  /* elements */
    uint64_t head_stride;
    uint64_t token_stride; /* 2^24 at most */
    uint64_t layer_stride; /* elements from one layer's pool to the next (calls with a context); pools of
                            * several layers lie side by side, or interleaved by page, head or
                            * position; looked at only where there are several */
} hy_paged_cache;

/* The requests of one step.  Request r has the token rows q_start[r] .. q_start[r + 1] - 1
 * and kv_len[r] keys, its new tokens among them as the last ones.  Row i of them sees the
 * keys 0 .. kv_len[r] - rows + i (causal), or the first seen_dev[row] keys (at most
 * kv_len[r]): an image's tokens see their whole span, 0 sees nothing.  Position j of
 * request r lies in page table[r][j / page_size]; positions in pages outside
 * 0..n_pages-1 hold no key.  Rows from q_start[n_req] on belong to nobody: calls leave
 * their outputs as they were. */
typedef struct {
    uint32_t n_req;                /* 1..4096 */
    uint32_t n_rows;               /* rows of the token arrays, 1..2^20 */
    uint32_t max_pages;            /* entries of a table row; max_pages * page_size <= 2^30 */
    uint32_t max_new;              /* the most rows a request has: it only chooses the kernel */
    const int32_t* q_start_dev;    /* [n_req + 1], ascending from 0 */
    const int32_t* kv_len_dev;     /* [n_req] */
    const int32_t* table_dev;      /* [n_req][max_pages] */
    const int32_t* positions_dev;  /* [n_rows], calls that write the cache */
    const int32_t* slots_dev;      /* [n_rows], calls that write the cache */
    const int32_t* seen_dev;       /* [n_rows] or NULL: causal */
} hy_paged_batch;

/* The tables of a step, from lengths in device memory.  Request r has cached[r] tokens
 * behind it and new[r] >= 0 coming, so it wants ceil((cached + new) / page_size) pages and
 * holds the first held[r] of its table row.  First, pages beyond what is wanted go back:
 * they are pushed on the stack free_dev (n_free entries, room for n_pages) in request
 * order, each request's in ascending position.  Then requests take what they lack from the
 * stack's end, in order; the first that finds too few, and all that lack pages after it,
 * get none.  Outputs:
 *   held_out [n_req], n_free_out [1]   may be held_dev and n_free_dev themselves
 *   q_start [n_req + 1]                sums of new (new outside 0..n_rows counts as 0),
 *                                      at most n_rows
 *   status [n_req]                     0 served, 1 no pages left, 2 wants more than
 *                                      max_pages, 3 lengths out of range (negative, held
 *                                      above max_pages, rows past n_rows)
 *   kv_len [n_req]                     cached + new; 0 unless served
 *   positions [n_rows], slots [n_rows] cached + i and page * page_size + offset of row i of
 *                                      a served request; 0 and -1 for other rows (slot -1
 *                                      also where the table names no page of the pool)
 * A request that is not served keeps its pages (status 3: as they are).  An ended request
 * is one of length 0: its pages go back.  Calling again with the same inputs gives the
 * same outputs.  All sizes as in hy_paged_batch. */
int hy_paged_plan(const int32_t* cached_dev, const int32_t* new_dev, uint32_t n_req, uint32_t n_rows,
                  uint32_t page_size, uint32_t max_pages, uint32_t n_pages, int32_t* table_dev,
                  const int32_t* held_dev, int32_t* held_out_dev, int32_t* free_dev, const int32_t* n_free_dev,
                  int32_t* n_free_out_dev, int32_t* q_start_dev, int32_t* kv_len_dev, int32_t* positions_dev,
                  int32_t* slots_dev, int32_t* status_dev, void* stream);

/* Rotary embedding, per-head RMSNorm and the write of the cache: for every row t with a
 * slot, q [n_rows][n_heads][head_dim] receives norm(rotate(q_t)) in f32, the cache
 * norm(rotate(k_t)) and v_t at the slot, rounded to its type.  qkv [n_rows][(n_heads +
 * 2 n_kv_heads) head_dim] is the projection's output.  Pair (2i, 2i + 1) turns by
 * positions[t] * theta^(-2i / head_dim) (the angle in 64 bits: positions may be large), or
 * by rows positions[t] of the tables cos_dev / sin_dev [n_pos][head_dim] (not NULL, as
 * hy_build_2d_rope writes them), or not at all (theta 0, no tables).  Norm as
 * attention_forward_cpu: x * (1 / sqrt(mean x^2 + eps)) * w; weights [head_dim], NULL: 1.
 * Rows with a slot outside the pool, or a position outside the tables, are skipped.  Two
 * rows with the same slot: either may be what is kept. */
int hy_rope_qknorm_paged(const float* qkv_dev, uint32_t n_rows, uint32_t n_heads, const hy_paged_cache* cache,
                         const int32_t* positions_dev, const int32_t* slots_dev, float theta, const float* cos_dev,
                         const float* sin_dev, uint32_t n_pos, const float* q_norm_dev, const float* k_norm_dev,
                         float eps, float* q_dev, void* stream);

/* out[t][h] = sum_j p_j v_j, p = softmax_j(scale q[t][h] . k_j) over the keys row t sees
 * (hy_paged_batch); zero where it sees none.  q, out [n_rows][n_heads][head_dim] f32;
 * query head h reads kv head h / (n_heads / n_kv_heads).  Products and sums have f32
 * accuracy whatever the cache's type, relative to the largest elements of q, of a key and
 * of a value row: one below 2^-16 of its vector's largest is taken to 2^-39 of that, values
 * to 2^-98 at least.  Small weights over f16 caches, and over the others in long chunks small
 * products of a weight and its value row, are taken to 2^-31 of the row's largest.  Values
 * up to 2^88 sum without overflow; scores past f32's range are not defined.
 * A key that a row does not see does not touch it, whatever it holds; an infinity or NaN in q
 * or in a key that a row sees makes the row NaN, one in a value makes that element infinite
 * or NaN (with a weight of 0 it may be left out).  ws_dev:
 * hy_paged_attention_ws bytes (0 for bad arguments; by the cache's and the batch's sizes,
 * 103 MB at most), aligned to 16 bytes, contents indifferent. */
size_t hy_paged_attention_ws(uint32_t n_heads, const hy_paged_cache* cache, const hy_paged_batch* batch);
int hy_paged_attention(const float* q_dev, uint32_t n_heads, const hy_paged_cache* cache, const hy_paged_batch* batch,
                       float scale, float* out_dev, void* ws_dev, size_t ws_bytes, void* stream);

/* The verification of drafted tokens by speculative sampling.  Request r's rows
 * q_start[r] .. q_start[r + 1] - 1 of ids are its last token and its drafts x_1 .. x_n;
 * row i of logits is the target's prediction of what follows row i, and row i of
 * draft_probs [n_rows][vocab] the distribution that x_{i+1} was drawn from (NULL: drafts
 * without probabilities, as certain).  With p = softmax(logits / temperature[r]) (NULL: 1),
 * in order: x_{i+1} is accepted if u_accept[row i] * q(x_{i+1}) < p(x_{i+1}).  At the first
 * refusal the next token is drawn from max(p - q, 0) / sum (from p where that is 0
 * everywhere), after n accepted drafts from p of the last row; drawn by inversion: the
 * lowest index whose running sum exceeds u_sample[r] times the whole.  n_rows * vocab <= 2^36.  Temperature 0 or
 * less: x is accepted if it is the largest logit (equal ones: the lowest index), which is
 * also the next token.  Numbers are computed in 64 bits.  Outputs:
 *   accepted [n_req]           accepted drafts; -1 for a request without rows or with more
 *                              than max_new
 *   tokens [n_req][max_new]    the accepted drafts, then the next token, then -1.  A row
 *                              that gives no distribution (a logit that is NaN or +inf, all
 *                              -inf) ends its request with next token -1.
 * Drafts outside 0..vocab-1 are refused.  u in [0, 1).  ws_dev: hy_verify_drafts_ws bytes
 * (0 for bad arguments), aligned to 16 bytes, contents indifferent.
 *
 * Every row after a request's first is taken for a draft.  Rows that are none (a prompt's but
 * its last) are kept apart by a q_start of this call's own, with two entries per request:
 * its start, and its start + such rows.  Results 2 r are theirs and mean nothing (-1 for more
 * than max_new rows); results 2 r + 1 are of the rows behind, -1 where there are none.  So
 * the last piece of a prompt has one row here, its last token, and gets the first new token. */
size_t hy_verify_drafts_ws(uint32_t n_req, uint32_t n_rows, uint32_t vocab);
int hy_verify_drafts(const float* logits_dev, const float* draft_probs_dev, const int32_t* ids_dev,
                     const int32_t* q_start_dev, uint32_t n_req, uint32_t n_rows, uint32_t max_new, uint32_t vocab,
                     const float* temperature_dev, const float* u_accept_dev, const float* u_sample_dev,
                     int32_t* accepted_dev, int32_t* tokens_dev, void* ws_dev, size_t ws_bytes, void* stream);

/* hy_attn_forward over a paged cache: out = o_proj(attention of the batch's rows), the
 * rows' keys and values written to `layer`'s pool first.  x, out [n_rows][hidden].  Rows
 * that belong to nobody get zeros; a row without a slot, or with a position outside the
 * tables, has a query of zeros.  1D rotary positions (rope_theta), or the tables of
 * hy_rope_qknorm_paged.  The cache's heads are the context's; n_rows <= max_tokens. */
int hy_attn_forward_paged(hy_attn_ctx* ctx, uint32_t layer, const float* x_dev, const hy_paged_cache* cache,
                          const hy_paged_batch* batch, const float* cos_dev, const float* sin_dev, uint32_t n_pos,
                          float* out_dev, void* ws_dev, size_t ws_bytes, void* stream);

/* hy_model_forward over a paged cache of num_layers pools: ids int32 [n_rows], logits
 * [n_rows][vocab]; 1D rotary positions.  HY_ERR_UNSUPPORTED for a model with drop_tokens:
 * an expert's capacity would be shared with the other requests and with rows of nobody. */
int hy_model_forward_paged(hy_model_ctx* ctx, const int32_t* ids_dev, const hy_paged_cache* cache,
                           const hy_paged_batch* batch, float* logits_dev, void* ws_dev, size_t ws_bytes,
                           void* stream);

#ifdef __cplusplus
}
#endif
#endif
