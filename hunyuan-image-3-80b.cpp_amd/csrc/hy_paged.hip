// hy_paged.hip -- the tables of a paged cache built from lengths, and the write into it:
//  * paged_plan_kernel: pages taken and given back, block tables, row offsets, positions and
//    slots of a step (hy_paged_plan);
//  * paged_append_kernel: rotary embedding + QK-norm of the projection's output, queries to
//    [rows][nh][hd], keys and values to their slots in the cache's type.
#include "hy_device.hpp"
#include "hy_paged.hpp"
#include "hy_paged_rotary.hpp"
#include "hy_paged_split.hpp"

namespace hy {

// ---------------------------------------------------------------- tables and slots
// One work group, a request (or PER consecutive ones) per thread: sums over requests (rows, pages
// given back, pages taken) by scans, then the pages and the rows one per thread, whose request a
// search in LDS finds.  All of it is latency: 8 requests 3.7 us, 1024 requests 7.8.  Rows beyond
// PL_ROWS go to a second launch over the whole chip (4.1 us; 16 000 rows in one work group: 40).
// Sums saturate at PL_CAP, which is past every bound that they are compared with.
constexpr int PL_CAP = (1 << 30) - 1, PL_ROWS = 4096;

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, PL_CAP); }  // of two up to PL_CAP

template <int CTRL, int ROWS>
__device__ __forceinline__ int sat_step(int v) {
    return sat_add(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false));
}
// inclusive sum over the lanes of a wave: shifts inside 16-lane rows, then the rows' last lanes
__device__ __forceinline__ int wave_scan(int v) {
    v = sat_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v = sat_step<0x112, 0xF>(v);
    v = sat_step<0x114, 0xF>(v);
    v = sat_step<0x118, 0xF>(v);
    v = sat_step<0x142, 0xA>(v);  // lane 15 to row 1, lane 47 to row 3
    return sat_step<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
}
// exclusive sum over the work group's threads; total: of all of them
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* part, int& total) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int s = wave_scan(v);
    if (lane == WAVE - 1) part[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / WAVE; w++) {
        const int p = part[w];
        before = w < wave ? sat_add(before, p) : before;
        total = sat_add(total, p);
    }
    // exclusive: the lane before's inclusive sum (a saturated one cannot be taken back by v)
    const int prev = __shfl_up(s, 1, WAVE);
    return sat_add(before, lane ? prev : 0);
}

// the last r < n with at[r] <= x (at ascending, at[0] <= x)
__device__ __forceinline__ int find_last(const int* at, int n, int x) {
    int lo = 0;
    for (int step = 1 << (31 - __builtin_clz(n)); step; step >>= 1)
        if (lo + step < n && at[lo + step] <= x) lo += step;
    return lo;
}

// position and slot of row t, of a request served with `cached` tokens (negative: not served)
__device__ __forceinline__ void plan_row(const PagedPlanArgs& a, int t, int r, int start, int cached) {
    int pos = 0, slot = -1;
    if (cached >= 0) {
        pos = cached + t - start;
        const int p = a.table[(int64_t)r * a.max_pages + (pos >> a.shift)];
        if (p >= 0 && p < a.n_pages) slot = (p << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
}

template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void paged_plan_kernel(PagedPlanArgs a, int rows_here) {
    constexpr int N = THREADS * PER;
    __shared__ int part[3][THREADS / WAVE];
    __shared__ int start_s[N], give_s[N], take_s[N], held_s[N], want_s[N], cached_s[N];
    __shared__ int used_s;
    const int tid = threadIdx.x, r0 = tid * PER, page = 1 << a.shift;
    int cached[PER], held[PER], add[PER], rows[PER], want[PER], status[PER];
    int sum = 0, total;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = min(r0 + i, a.n_req - 1);
        cached[i] = a.cached[r];
        add[i] = a.add[r];
        held[i] = a.held[r];
    }
    const int n_free = min(max(a.n_free[0], 0), a.n_pages);
    // every read of held and n_free is done before any write (they may be the outputs): the first scan
    // has a barrier
#pragma unroll
    for (int i = 0; i < PER; i++) {
        rows[i] = r0 + i < a.n_req && add[i] >= 0 && add[i] <= a.n_rows ? add[i] : 0;
        sum = sat_add(sum, rows[i]);
    }
    if (tid == 0) used_s = 0;
    int at = block_scan<THREADS>(sum, part[0], total);
    const int n_used = min(total, a.n_rows);
    int give_sum = 0, take_sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = r0 + i;
        const int64_t len = (int64_t)cached[i] + add[i], w = (len + page - 1) >> a.shift;
        const bool bad = cached[i] < 0 || add[i] < 0 || (int64_t)at + add[i] > a.n_rows || held[i] < 0 ||
                         held[i] > a.max_pages;
        status[i] = bad ? 3 : w > a.max_pages ? 2 : 0;
        want[i] = status[i] || r >= a.n_req ? held[i] : (int)w;  // refused requests keep what they have
        start_s[r] = min(at, a.n_rows);
        held_s[r] = held[i];
        want_s[r] = want[i];
        if (r < a.n_req) a.q_start[r] = min(at, a.n_rows);
        at = sat_add(at, rows[i]);
        give_sum = sat_add(give_sum, max(held[i] - want[i], 0));
        take_sum = sat_add(take_sum, max(want[i] - held[i], 0));
    }
    if (tid == 0) a.q_start[a.n_req] = n_used;
    int given, taken;
    int give = block_scan<THREADS>(give_sum, part[1], given), take = block_scan<THREADS>(take_sum, part[2], taken);
    const int avail = min(sat_add(n_free, given), a.n_pages);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = r0 + i, need = max(want[i] - held[i], 0);
        give_s[r] = give;
        take_s[r] = take;
        give = sat_add(give, max(held[i] - want[i], 0));
        take = sat_add(take, need);
        if (need && take > avail) {
            status[i] = 1;
        } else if (need) {
            atomicMax(&used_s, take);  // those that are served come before those that are not
        }
        cached_s[r] = status[i] == 0 ? cached[i] : -1;
        if (r < a.n_req) {
            a.status[r] = status[i];
            a.held_out[r] = status[i] == 0 ? want[i] : held[i];
            a.kv_len[r] = status[i] == 0 ? cached[i] + add[i] : 0;
        }
    }
    __syncthreads();
    const int used = used_s;
    if (tid == 0) a.n_free_out[0] = avail - used;
    if (given) {  // the same for all
        for (int e = tid; e < min(given, a.n_pages - n_free); e += THREADS) {
            const int r = find_last(give_s, a.n_req, e);
            a.free_[n_free + e] = a.table[(int64_t)r * a.max_pages + want_s[r] + e - give_s[r]];
        }
        __syncthreads();  // the stack is whole
    }
    for (int e = tid; e < used; e += THREADS) {
        const int r = find_last(take_s, a.n_req, e);
        a.table[(int64_t)r * a.max_pages + held_s[r] + e - take_s[r]] = a.free_[avail - 1 - e];
    }
    if (!rows_here) return;
    __syncthreads();  // the tables are whole
    for (int t = tid; t < a.n_rows; t += THREADS) {
        const int r = t < n_used ? find_last(start_s, a.n_req, t) : 0;
        plan_row(a, t, r, start_s[r], t < n_used ? cached_s[r] : -1);
    }
}

// the rows' positions and slots, from what the first launch wrote
__global__ __launch_bounds__(256) void paged_plan_rows_kernel(PagedPlanArgs a) {
    __shared__ int start_s[PG_MAX_REQ];
    for (int r = threadIdx.x; r < a.n_req; r += 256) start_s[r] = a.q_start[r];
    const int n_used = a.q_start[a.n_req], t = blockIdx.x * 256 + threadIdx.x;
    __syncthreads();
    if (t >= a.n_rows) return;
    const int r = t < n_used ? find_last(start_s, a.n_req, t) : 0;
    plan_row(a, t, r, start_s[r], t < n_used && a.status[r] == 0 ? a.cached[r] : -1);
}

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t s) {
    const int here = a.n_rows <= PL_ROWS;
    if (a.n_req <= 256 && a.n_rows <= 1024)
        hipLaunchKernelGGL((paged_plan_kernel<256, 1>), dim3(1), dim3(256), 0, s, a, here);
    else if (a.n_req <= 1024)
        hipLaunchKernelGGL((paged_plan_kernel<1024, 1>), dim3(1), dim3(1024), 0, s, a, here);
    else
        hipLaunchKernelGGL((paged_plan_kernel<1024, PG_MAX_REQ / 1024>), dim3(1), dim3(1024), 0, s, a, here);
    if (!here) hipLaunchKernelGGL(paged_plan_rows_kernel, dim3((a.n_rows + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- rotary + QK-norm + write
// The units of a row are its heads in memory order: nh query heads, nkv key heads, nkv value
// heads.  A work group takes a group of PA_STEPS * 64 / (HD / 4) units of four consecutive rows, a
// row per wave (neighbouring rows are neighbours in a page); HD / 4 lanes share a unit, 4 dims
// (16 bytes) each, and all loads of a wave go out before anything else.  Angles and norm:
// hy_paged_rotary.hpp.
// Bound by memory: 4096 rows of 48 heads of 128 (205 MB) 33 us in caches, 40 from memory (5.2 TB/s);
// 5 rows 4.4 us, all of it latency.
constexpr int PA_STEPS = 4;

template <class E, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int LPU = HD / 4, UNITS = PA_STEPS * WAVE / LPU;
    const int units = a.nh + 2 * a.c.nkv, groups = (units + UNITS - 1) / UNITS;
    const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int t = (int)(b / groups) * 4 + (int)threadIdx.x / WAVE, u0 = (int)(b % groups) * UNITS;
    if (t >= a.n_rows) return;
    const int l = threadIdx.x % WAVE, d = 4 * (l % LPU);
    const float* const row = a.qkv + (int64_t)t * units * HD + d;
    v4f_t x[PA_STEPS];
#pragma unroll
    for (int s = 0; s < PA_STEPS; s++)
        x[s] = *reinterpret_cast<const v4f_t*>(row + (int64_t)min(u0 + (s * WAVE + l) / LPU, units - 1) * HD);
    const int slot = a.slots[t], pos = a.positions[t];
    // What a layer goes on with comes from this call alone: a row of nobody has an attention of zeros,
    // a skipped one a query of zeros.
    const auto clear = [&](float* to) {
#pragma unroll
        for (int s = 0; s < PA_STEPS; s++) {
            const int u = u0 + (s * WAVE + l) / LPU;
            if (u < a.nh) *reinterpret_cast<v4f_t*>(to + ((int64_t)t * a.nh + u) * HD + d) = v4f_t{};
        }
    };
    if (a.merged && t >= a.row_end[0]) clear(a.merged);
    if (slot < 0 || (slot >> a.c.shift) >= a.c.n_pages || (a.rotate == 2 && (pos < 0 || pos >= a.n_pos))) {
        if (a.merged) clear(a.q);
        return;
    }
    float cs[2] = {1.0f, 1.0f}, sn[2] = {0.0f, 0.0f};
    if (u0 < a.nh + a.c.nkv) {  // not values alone
        if (a.rotate == 1) {
#pragma unroll
            for (int p = 0; p < 2; p++) rope_angle(pos, a.freq[d / 2 + p], sn[p], cs[p]);
        } else if (a.rotate == 2) {
            const v4f_t c = *reinterpret_cast<const v4f_t*>(a.cos_t + (int64_t)pos * HD + d);
            const v4f_t s = *reinterpret_cast<const v4f_t*>(a.sin_t + (int64_t)pos * HD + d);
            cs[0] = c[0], cs[1] = c[2], sn[0] = s[0], sn[1] = s[2];
        }
    }
    const v4f_t one = {1.0f, 1.0f, 1.0f, 1.0f};
    const v4f_t wq = a.q_norm ? *reinterpret_cast<const v4f_t*>(a.q_norm + d) : one;
    const v4f_t wk = a.k_norm ? *reinterpret_cast<const v4f_t*>(a.k_norm + d) : one;
    const int64_t cell = (int64_t)(slot >> a.c.shift) * a.c.page_stride +
                         (int64_t)(slot & ((1 << a.c.shift) - 1)) * a.c.token_stride + d;
#pragma unroll
    for (int s = 0; s < PA_STEPS; s++) {
        const int u = u0 + (s * WAVE + l) / LPU;
        v4f_t y;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            y[2 * p] = fmaf(x[s][2 * p], cs[p], -(x[s][2 * p + 1] * sn[p]));
            y[2 * p + 1] = fmaf(x[s][2 * p], sn[p], x[s][2 * p + 1] * cs[p]);
        }
        const float rms = head_rms<HD>(y, a.eps);
        if (u < a.nh) {
            *reinterpret_cast<v4f_t*>(a.q + ((int64_t)t * a.nh + u) * HD + d) = y * rms * wq;
        } else if (u < units) {
            const bool key = u < a.nh + a.c.nkv;
            const v4f_t z = key ? y * rms * wk : x[s];
            E* const pool = static_cast<E*>(key ? a.c.k : a.c.v);
            typedef E v4 __attribute__((ext_vector_type(4)));  // to nearest, ties to even
            *reinterpret_cast<v4*>(pool + cell + (u - a.nh - (key ? 0 : a.c.nkv)) * a.c.head_stride) =
                __builtin_convertvector(z, v4);
        }
    }
}

template <class E>
static void append(const PagedAppendArgs& a, hipStream_t s) {
    const int units = a.nh + 2 * a.c.nkv, per = PA_STEPS * WAVE * 4 / a.c.hd;
    // a launch has fewer than 2^32 threads along x
    const int64_t n = (int64_t)((a.n_rows + 3) / 4) * ((units + per - 1) / per), gx = n < 1 << 22 ? n : 1 << 22;
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));
    if (a.c.hd == 128)
        hipLaunchKernelGGL((paged_append_kernel<E, 128>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((paged_append_kernel<E, 64>), grid, dim3(256), 0, s, a);
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    if (a.c.type == HY_TYPE_F32)
        append<float>(a, s);
    else if (a.c.type == HY_TYPE_F16)
        append<_Float16>(a, s);
    else
        append<__bf16>(a, s);
    return hipGetLastError();
}

}  // namespace hy
