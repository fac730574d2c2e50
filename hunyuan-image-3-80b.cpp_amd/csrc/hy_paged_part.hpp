// hy_paged_part.hpp -- how the paged attention's work is cut between workers.
//
// A request's rows (token x query head of one kv head, token-major) fall into tiles of M; an
// item is a (request, kv head, tile) and its nominal length the keys that its last token sees
// if causal.  All items of a batch in a row (requests, then kv heads, then tiles) are cut into
// equal stretches, one per worker: however ragged the lengths, every worker has the same share.
// Lengths are in device memory, so every work group sums them itself (part_sums).  An item
// inside one worker's stretch is written by it; one that is cut leaves a partial result per
// piece, joined afterwards.  A piece [x0, x1) of nominal length W takes the key blocks
// floor(x0 B / W) .. floor(x1 B / W) - 1 of the item's real B.
#pragma once
#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

struct PartShape {
    int M;          // rows of a tile
    int64_t rows_lo, rows_hi;  // requests with rows_lo < rows <= rows_hi belong to this launch
    int workers;
    int min_keys;   // of a stretch
};

struct PartReq {
    int start, n, kv;   // first row, rows (tokens), keys
    int tiles, tau;     // tiles of its rows, nominal tokens per tile
    int64_t base, head; // keys before its first token; nominal length of a head's tiles
    // nominal length of tiles 0 .. k - 1
    __device__ __forceinline__ int64_t upto(int64_t k) const {
        const int64_t f = min(k, (int64_t)(n / tau));
        return k * base + (int64_t)tau * (f * (f + 1) / 2) + (k - f) * n;
    }
};

__device__ __forceinline__ PartReq part_req(const PagedAttnArgs& a, const PartShape& p, int r) {
    PartReq q;
    const int G = a.nh / a.c.nkv;
    const int s0 = min(max(a.q_start[r], 0), a.n_rows), s1 = min(max(a.q_start[r + 1], 0), a.n_rows);
    q.start = s0;
    q.n = max(s1 - s0, 0);
    q.kv = min(max(a.kv_len[r], 0), a.max_pages << a.c.shift);
    const int64_t rows = (int64_t)q.n * G;
    q.tiles = rows > p.rows_lo && rows <= p.rows_hi ? (int)((rows + p.M - 1) / p.M) : 0;
    q.tau = max(p.M / G, 1);
    q.base = max(q.kv - q.n, 0);
    q.head = q.upto(q.tiles);
    return q;
}

// Sums of the requests' nominal lengths: thread i of the THREADS holds the sum before its
// per = ceil(n_req / THREADS) consecutive ones in pre[i], the whole in pre[THREADS].
template <int THREADS>
__device__ __forceinline__ int64_t part_sums(const PagedAttnArgs& a, const PartShape& p, int64_t* pre) {
    const int tid = threadIdx.x, per = (a.n_req + THREADS - 1) / THREADS;
    int64_t s = 0;
    for (int r = tid * per; r < min((tid + 1) * per, a.n_req); r++) s += part_req(a, p, r).head * a.c.nkv;
    int64_t v = s;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const int64_t o = __shfl_up(v, d, WAVE);
        if (tid % WAVE >= d) v += o;
    }
    __shared__ int64_t wave_sum_s[THREADS / WAVE];
    if (tid % WAVE == WAVE - 1) wave_sum_s[tid / WAVE] = v;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / WAVE; w++) {
        if (w < tid / WAVE) before += wave_sum_s[w];
        total += wave_sum_s[w];
    }
    pre[tid] = before + v - s;
    if (tid == 0) pre[THREADS] = total;
    __syncthreads();
    return total;
}

// a value that all lanes share, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

__device__ __forceinline__ int64_t part_stretch(const PartShape& p, int64_t total) {
    return max((total + p.workers - 1) / p.workers, (int64_t)p.min_keys);
}

struct PartItem {
    PartReq q;
    int r, g, tile;
    int64_t at;   // where the item starts in the row of all items
    int64_t len;  // its nominal length
};

// the item at place x (0 <= x < total); uniform over the wave
template <int THREADS>
__device__ __forceinline__ PartItem part_find(const PagedAttnArgs& a, const PartShape& p, const int64_t* pre,
                                              int64_t x) {
    x = uniform(x);
    int lo = 0, hi = THREADS;  // pre[lo] <= x < pre[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (uniform(pre[mid]) <= x)
            lo = mid;
        else
            hi = mid;
    }
    const int per = (a.n_req + THREADS - 1) / THREADS;
    PartItem it;
    it.r = uniform(lo * per);
    it.at = uniform(pre[uniform(lo)]);
    it.q = part_req(a, p, it.r);
    while (x - it.at >= it.q.head * a.c.nkv) {
        it.at += it.q.head * a.c.nkv;
        it.r++;
        it.q = part_req(a, p, it.r);
    }
    it.g = (int)((x - it.at) / it.q.head);
    it.at += it.q.head * it.g;
    int t0 = 0, t1 = it.q.tiles;  // upto(t0) <= x - at < upto(t1)
    while (t1 - t0 > 1) {
        const int mid = (t0 + t1) / 2;
        if (it.q.upto(mid) <= x - it.at)
            t0 = mid;
        else
            t1 = mid;
    }
    it.tile = t0;
    it.at += it.q.upto(t0);
    it.len = it.q.upto(t0 + 1) - it.q.upto(t0);
    return it;
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
__host__ __device__ __forceinline__ size_t part_slot_floats(int M, int hd) { return (size_t)M * (hd + 2); }

// requests of many rows: tiles of PM_TILE rows, PM_WORKERS work groups (hy_paged_many.hip)
constexpr int PM_TILE = 256, PM_WORKERS = 256;
hipError_t launch_paged_many(const PagedAttnArgs& a, const PartShape& ps, hipStream_t s);

}  // namespace hy
