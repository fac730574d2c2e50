// hy_paged_part.hpp -- how the paged attention's work is cut between workers.
//
// A request's rows (token x query head of one kv head, token-major) fall into tiles of M; an
// item is a (request, kv head, tile) and its nominal length the keys that its last token sees
// if causal, plus what starting an item costs.  All items of a batch in a row (requests, then kv
// heads, then tiles) are cut into equal stretches, one per worker: however ragged the lengths,
// every worker has the same share.  Lengths are in device memory, so every work group sums them
// itself (part_sums).  An item inside one worker's stretch is written by it; one that is cut leaves
// a partial result per piece, joined afterwards (joining the pieces of a work group's waves in LDS
// first was tried: 32 requests of 24 rows 72.5 -> 70.4 us, one of 4 rows 14.1 -> 14.9).  A piece
// [x0, x1) of an item of nominal length W takes the key blocks from x0 B / W to x1 B / W
// (part_block) of the item's real B.
#pragma once
#include <limits.h>

#include <type_traits>

#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

struct PartShape {
    int M, m_shift;            // rows of a tile: 1 << m_shift
    int G, tau;                // query heads of a kv head; nominal tokens per tile, max(M / G, 1)
    int64_t rows_lo, rows_hi;  // requests with rows_lo < rows <= rows_hi belong to this launch
    int workers;
    int extra;                 // keys that starting an item is worth
    int unit;                  // nominal length of the shortest stretch, a power of two
    int snap;                  // a cut nearer than this to an item's end moves there
    size_t ws;                 // floats of the workspace before this launch's slots
};
inline PartShape part_shape(int m_shift, int G, int64_t rows_lo, int64_t rows_hi, int workers, int extra, int unit,
                            int snap, size_t ws) {
    const int M = 1 << m_shift;
    return {M, m_shift, G, M / G > 1 ? M / G : 1, rows_lo, rows_hi, workers, extra, unit, snap, ws};
}

// a value that all lanes share, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

struct PartReq {
    int start, n, kv;   // first row, rows (tokens), keys
    int tiles, full;    // tiles of its rows; those whose nominal tokens do not reach past the last
    int64_t base, head; // keys before its first token, and extra; nominal length of a head's tiles
    // nominal length of tiles 0 .. k - 1; I: what holds the request's.  f (f + 1) is formed without a
    // sign: tiles of one token reach 2^32 with it where half of it still fits I
    template <class I>
    __host__ __device__ __forceinline__ I upto(int tau, I k) const {
        const I f = k < (I)full ? k : (I)full;
        typedef typename std::make_unsigned<I>::type U;
        return k * (I)base + (I)tau * (I)((U)f * (U)(f + 1) / 2) + (k - f) * (I)n;
    }
};

// n / d for 0 <= n <= 2^20, 0 < d: n + 1/2 keeps 1 / (2 d) from the next whole number, the
// reciprocal is off by 2^-22 of the quotient
__device__ __forceinline__ int part_div(int n, int d) {
    return (int)(((float)n + 0.5f) * __builtin_amdgcn_rcpf((float)d));
}
// floor(x / n) for 0 <= x, 0 < n, the same for the wave: an estimate in f32, then a step either way
template <class I>
__device__ __forceinline__ int part_quotient(I x, I n) {
    int k = uniform((int)((float)x * __builtin_amdgcn_rcpf((float)n)));
    while ((I)k * n > x) k--;
    while (x - (I)k * n >= n) k++;
    return k;
}

__device__ __forceinline__ PartReq part_req(const PartShape& p, int start, int n, int kv) {
    PartReq q{start, n, kv, 0, part_div(n, p.tau), max(kv - n, 0) + p.extra, 0};
    const int64_t rows = (int64_t)n * p.G;
    if (rows > p.rows_lo && rows <= p.rows_hi) q.tiles = (int)((rows + p.M - 1) >> p.m_shift);
    // whole units: where stretches are one unit, short requests share no worker
    q.head = (q.upto<int64_t>(p.tau, q.tiles) + p.unit - 1) & ~(int64_t)(p.unit - 1);
    return q;
}

// What a work group of THREADS keeps of the batch in LDS: thread i has the per = ceil(n_req /
// THREADS) requests from i * per on; the sum of nominal lengths before them, and, of the
// first THREADS requests, row start, rows and keys.
template <int THREADS>
struct PartSums {
    int64_t pre[THREADS + 1];
    int64_t wave[THREADS / WAVE];
    int start[THREADS], n[THREADS], kv[THREADS];
};

__device__ __forceinline__ void part_load(const PagedAttnArgs& a, int r, int& start, int& n, int& kv) {
    const int s0 = a.q_start[r], s1 = a.q_start[r + 1], k = a.kv_len[r];
    start = min(max(s0, 0), a.n_rows);
    n = max(min(max(s1, 0), a.n_rows) - start, 0);
    kv = min(max(k, 0), a.max_pages << a.c.shift);
}

// inclusive sum over the lanes: shifts inside 16 lanes, then the rows' last lanes to those behind
// (vector operations: six steps of shuffles take 1 us)
__device__ __forceinline__ int64_t part_scan(int64_t v) {
    const auto step = [&](auto shr) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(shr)::value, 0xF, 0xF, false);
        const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), decltype(shr)::value, 0xF, 0xF, false);
        v += (int64_t)((uint64_t)(uint32_t)hi << 32 | lo);
    };
    step(std::integral_constant<int, 0x111>{});
    step(std::integral_constant<int, 0x112>{});
    step(std::integral_constant<int, 0x114>{});
    step(std::integral_constant<int, 0x118>{});
    const auto row_sum = [&](int l) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)v, l));
    };
    const int64_t r0 = row_sum(15), r1 = r0 + row_sum(31), r2 = r1 + row_sum(47);
    const int lane = threadIdx.x % WAVE;
    return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}

// fills s; returns the sum of all nominal lengths
template <int THREADS>
__device__ __forceinline__ int64_t part_sums(const PagedAttnArgs& a, const PartShape& p, PartSums<THREADS>& s) {
    const int tid = threadIdx.x, per = (a.n_req + THREADS - 1) / THREADS;
    int64_t mine = 0;
    for (int r = tid * per; r < min((tid + 1) * per, a.n_req); r++) {
        int start, n, kv;
        part_load(a, r, start, n, kv);
        mine += part_req(p, start, n, kv).head * a.c.nkv;
        if (r < THREADS) {
            s.start[r] = start;
            s.n[r] = n;
            s.kv[r] = kv;
        }
    }
    const int64_t v = part_scan(mine);
    if (tid % WAVE == WAVE - 1) s.wave[tid / WAVE] = v;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / WAVE; w++) {
        if (w < tid / WAVE) before += s.wave[w];
        total += s.wave[w];
    }
    s.pre[tid] = before + v - mine;
    if (tid == 0) s.pre[THREADS] = total;
    __syncthreads();
    return uniform(total);
}

__device__ __forceinline__ int64_t part_stretch(const PartShape& p, int64_t total) {
    // workers is a power of two
    return max((total + p.workers - 1) >> (31 - __builtin_clz(p.workers)), (int64_t)p.unit);
}

struct PartItem {
    PartReq q;
    int r, g, tile;
    int64_t at;  // where the item starts in the row of all items
    int len;     // its nominal length: the keys, at most 2^30, and the tokens
};

// kv head and tile of place y of a request
template <class I>
__device__ __forceinline__ void part_place(const PartShape& p, PartItem& it, I y) {
    it.g = part_quotient(y, (I)it.q.head);
    y -= (I)it.q.head * it.g;
    I t = 0;  // upto(t) <= y < upto(t + 1)
    if (it.q.tiles > 1) {
        // tiles of full size: t base + tau t (t + 1) / 2 = y
        const float b = (float)(I)it.q.base + 0.5f * p.tau, yf = (float)y;
        const float root = __builtin_amdgcn_sqrtf(b * b + 2.0f * p.tau * yf);
        t = min(uniform((int)(2.0f * yf * __builtin_amdgcn_rcpf(b + root))), it.q.tiles - 1);
        while (t > 0 && it.q.upto(p.tau, t) > y) t--;
        while (t + 1 < it.q.tiles && it.q.upto<I>(p.tau, t + 1) <= y) t++;  // the last one ends with its head
    }
    it.tile = (int)t;
    const I t0 = it.q.upto(p.tau, t);
    it.at += it.q.head * it.g + t0;
    it.len = (int)((t + 1 < it.q.tiles ? it.q.upto<I>(p.tau, t + 1) : (I)it.q.head) - t0);
}

// the item at place x (0 <= x < total), the same for the whole wave
template <int THREADS>
__device__ __forceinline__ PartItem part_find(const PagedAttnArgs& a, const PartShape& p, const PartSums<THREADS>& s,
                                              int64_t x) {
    // pre[lo] <= x < pre[lo + 1] (ties: the last): 64 of pre at once, then those between two
    constexpr int STEP = THREADS / WAVE;
    const int lane = threadIdx.x % WAVE;
    const int b = (__builtin_popcountll(__ballot(s.pre[lane * STEP] <= x)) - 1) * STEP;
    const int lo = b + __builtin_popcountll(__ballot(s.pre[b + lane % STEP] <= x && lane < STEP)) - 1;
    const int per = (a.n_req + THREADS - 1) / THREADS;
    PartItem it;
    it.r = lo * per;
    it.at = uniform(s.pre[lo]);
    for (;; it.r++) {
        int start, n, kv;
        if (it.r < THREADS) {
            start = s.start[it.r];
            n = s.n[it.r];
            kv = s.kv[it.r];
        } else {
            part_load(a, it.r, start, n, kv);
        }
        it.q = part_req(p, uniform(start), uniform(n), uniform(kv));
        if (x - it.at < it.q.head * a.c.nkv) break;
        it.at += it.q.head * a.c.nkv;
    }
    const int64_t y = x - it.at;
    if (it.q.head * a.c.nkv < 1ll << 31)  // 32 bits: a third of the instructions
        part_place<int>(p, it, (int)y);
    else
        part_place<int64_t>(p, it, y);
    return it;
}

// the block where a piece ending at place y of an item of nominal length len ends: rounded, but
// growing with y and the same for both who share the cut
__device__ __forceinline__ int part_block(int y, int len, int blocks) {
    return y >= len ? blocks : min(uniform((int)((float)y * ((float)blocks / (float)len))), blocks);
}

// A worker's piece of the item at place x, [p0, p1) of it: where its stretch begins and ends, each
// moved to the item's end that is nearer than p.snap (the neighbour moves it too).  x goes on to the
// next item, or to x_end.  False: nothing of the item is the worker's.
__device__ __forceinline__ bool part_piece(const PartShape& p, const PartItem& it, int64_t& x, int64_t x_end, int& p0,
                                           int& p1) {
    const auto cut = [&](int64_t at) {
        if (at - it.at >= it.len) return it.len;
        const int y = (int)(at - it.at);
        return y < p.snap ? 0 : it.len - y < p.snap ? it.len : y;
    };
    p0 = x == it.at ? 0 : cut(x);
    p1 = cut(x_end);
    x = p1 == it.len ? it.at + it.len : x_end;
    return p0 < p1;
}

// A score of -inf comes from an infinity in q or in the key (or, over f32 and bf16 caches, from
// products past f32's range): it becomes NaN, as one of +inf does in its weight, or the row would
// go on as if the key were masked, and one with no other score as if it saw nothing.  -inf has the
// largest bits but for NaNs', so the streams look for it by a maximum of whole numbers (0 to 2 %
// of their time; 1 to 3 % of the tiles', which mark such keys as they store them instead, 0 to 1 %).
constexpr uint32_t PA_MINUS_INF = 0xff800000u;
template <int N, class V>
__device__ __forceinline__ uint32_t top_bits(const V& s, uint32_t top = 0) {
#pragma unroll
    for (int v = 0; v < N; v++) top = max(top, __float_as_uint(s[v]));
    return top;
}
template <int N, class V>
__device__ __forceinline__ void minus_inf_to_nan(V& s) {
    asm volatile("");  // behind a branch, not done without one
#pragma unroll
    for (int v = 0; v < N; v++) s[v] = s[v] == -INFINITY ? __builtin_nanf("") : s[v];
}

// Attention of this lane's row over keys k0 .. k1 - 1, key by key in f32: what the kernels do
// again where their V holds infinities or NaNs.  A key of weight 0 does not touch the row.
// LPR lanes (l, l + 64 / LPR, ...) share a row, the i-th of a lane's HD / LPR dims is dim(i);
// set and get access the sums, m and l get the running maximum (base 2) and sum.
template <class E, int HD, int LPR, class Dim, class Set, class Get>
__device__ __forceinline__ void slow_rows(const PagedAttnArgs& a, const int* trow, int kv, int k0, int k1, int end,
                                          const float* q, const E* kg, const E* vg, Dim dim, Set set, Get get,
                                          float& m, float& l) {
    constexpr int N = HD / LPR;
    const float qscale = a.scale * 1.4426950408889634f;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) set(i, 0.0f);
#pragma unroll 1
    for (int key = k0; key < min(k1, kv); key++) {
        const int e = trow[key >> a.c.shift];
        if (e < 0 || e >= a.c.n_pages) continue;
        const int64_t at = e * a.c.page_stride + (key & ((1 << a.c.shift) - 1)) * a.c.token_stride;
        const float* qk = q;
        asm volatile("" : "+v"(qk));  // read again for every key, not kept in registers
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) s = fmaf(qk[dim(i)] * qscale, (float)kg[at + dim(i)], s);
#pragma unroll
        for (int d = 32; d >= 64 / LPR; d >>= 1) s += shfl_xor(s, d);
        if (s == -INFINITY) s = __builtin_nanf("");
        if (key >= end) s = -INFINITY;
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(s - ref);
        m = mn;
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float v = p * (float)vg[at + dim(i)];
            set(i, get(i) * alpha + (p != 0.0f ? v : 0.0f));
        }
    }
}

// Partial results: worker w's first piece, of an item begun before it, in slot 2 w, its last,
// of an item it begins and another ends, in 2 w + 1.  A slot: [M][hd] unnormalised output,
// [M] running maximum, [M] sum.
// The output lies by rows, or, from tiles of 256 rows, as their lanes hold it, so that a wave stores
// whole lines (prompts 64.4 -> 60.9 us; drafts' 53 for 56, but their joins of many pieces 17 for
// 11): per 32 rows, [n][64 lanes][4 dims], lane 32 h + row % 32, of d / 4 h the bit 1, n the
// others.
__device__ __forceinline__ int part_at(int hd, int row, int d) {
    const int m = d / 4;
    return row / 32 * 32 * hd + ((m >> 2 << 1 | (m & 1)) * 64 + 32 * (m >> 1 & 1) + row % 32) * 4;
}
__host__ __device__ __forceinline__ size_t part_slot_floats(int M, int hd) { return (size_t)M * (hd + 2); }

// What worker w leaves for the join: the item that it begins and others end.
struct PartJob {
    int n_piece;    // w's own and those of the workers after it; 0: no such item
    int n_live;     // rows
    int start;      // the request's first row
    int rho0;       // the tile's first row (token x head) of the request
    int g, pad[3];  // kv head
};
// floats of a launch's workspace: slots, then jobs
__host__ __device__ __forceinline__ size_t part_ws_floats(int workers, int M, int hd) {
    return workers * (2 * part_slot_floats(M, hd) + sizeof(PartJob) / 4);
}
__device__ __forceinline__ PartJob* part_jobs(const PagedAttnArgs& a, const PartShape& p, int hd) {
    return reinterpret_cast<PartJob*>(a.ws + p.ws + 2 * (size_t)p.workers * part_slot_floats(p.M, hd));
}
// the job that a piece [p0, p1) of an item makes of its worker
__device__ __forceinline__ PartJob part_job(const PartShape& p, const PartItem& it, int p0, int p1, int64_t stretch,
                                            int n_live) {
    PartJob j{0, n_live, it.q.start, it.tile * p.M, it.g, {}};
    if (p0 == 0 && p1 < it.len)  // the other pieces are a stretch each, the last one's rest aside
        j.n_piece = 2 + part_quotient(max(it.len - max(p.snap, 1) - p1, 0), (int)min(stretch, (int64_t)INT_MAX));
    return j;
}

// requests of few rows: PF_WORKERS waves, each for itself (hy_paged_attn.hip, hy_paged_wide.hip)
constexpr int PF_WAVES = 4, PF_GROUPS = 512, PF_WORKERS = PF_GROUPS * PF_WAVES;  // two work groups per CU
// The running maximum that weights are relative to is left behind while a block's scores do not
// pass it by more than PA_LAG (base 2): weights are up to 2^PA_LAG, and the sums are rescaled
// once or twice per row instead of at every new maximum.
constexpr float PA_LAG = 8.0f;
constexpr float PF_PSCALE = 64.0f;  // of the weights' f16 pieces: below 2^14 with PA_LAG
void launch_paged_wide(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s);

// requests of many rows: tiles of PM_TILE rows, PM_WORKERS work groups (hy_paged_many.hip)
constexpr int PM_TILE_SHIFT = 8, PM_TILE = 1 << PM_TILE_SHIFT, PM_WORKERS = 256;
void launch_paged_many(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s);

}  // namespace hy
