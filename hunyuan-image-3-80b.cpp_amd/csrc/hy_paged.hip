// hy_paged.hip -- the tables of a paged cache built from lengths, and the write into it:
//  * paged_plan_kernel: pages taken and given back, block tables, row offsets, positions and
//    slots of a step (hy_paged_plan);
//  * paged_append_kernel: rotary embedding + QK-norm of the projection's output, queries to
//    [rows][nh][hd], keys and values to their slots in the cache's type.
#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

// ---------------------------------------------------------------- tables and slots
// One work group, a request (or PER consecutive ones) per thread: sums over requests (rows, pages
// given back, pages taken) by scans, then the pages and the rows one per thread, whose request a
// search in LDS finds.  All of it is latency: 8 requests 6 us, 1024 requests 11.  Rows beyond
// PL_ROWS go to a second launch over the whole chip (16 000 rows in one work group: 40 us).
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
// One wave per (row, group of PA_HEADS heads), lane l the pair (2l, 2l + 1) of every head:
// the angle is formed once per wave.  An angle is kept as a fraction of a turn in 64 bits,
// position times turns per position minus its whole part, so a far position costs no
// accuracy; sine and cosine of the remaining |x| <= pi are f32.
constexpr int PA_HEADS = 4;

template <class E>
__device__ __forceinline__ void store_pair(E* p, float a, float b) {
    typedef E v2 __attribute__((ext_vector_type(2)));
    const v2 r = {(E)a, (E)b};  // to nearest, ties to even
    *reinterpret_cast<v2*>(p) = r;
}

template <class E>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const int heads = a.nh + a.c.nkv, hd = a.c.hd;
    const int groups = (heads + PA_HEADS - 1) / PA_HEADS;
    const int64_t wid = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + threadIdx.x / WAVE;
    if (wid >= (int64_t)a.n_rows * groups) return;
    const int t = (int)(wid / groups), h0 = (int)(wid % groups) * PA_HEADS, l = threadIdx.x % WAVE;
    const int slot = a.slots[t], pos = a.positions[t];
    if (slot < 0 || (slot >> a.c.shift) >= a.c.n_pages) return;
    if (a.rotate == 2 && (pos < 0 || pos >= a.n_pos)) return;
    if (2 * l >= hd) return;  // head_dim 64: half a wave (the sums below stay inside it)
    float cs = 1.0f, sn = 0.0f;
    if (a.rotate == 1) {
        double turn = (double)pos * a.freq[l];
        turn -= rint(turn);
        sincosf((float)(turn * 6.283185307179586), &sn, &cs);
    } else if (a.rotate == 2) {
        cs = a.cos_t[(int64_t)pos * hd + 2 * l];
        sn = a.sin_t[(int64_t)pos * hd + 2 * l];
    }
    const float* const row = a.qkv + (int64_t)t * (a.nh + 2 * a.c.nkv) * hd + 2 * l;
    const int64_t cell = (int64_t)(slot >> a.c.shift) * a.c.page_stride +
                         (int64_t)(slot & ((1 << a.c.shift) - 1)) * a.c.token_stride + 2 * l;
    for (int hh = h0; hh < min(h0 + PA_HEADS, heads); hh++) {
        const float2 x = *reinterpret_cast<const float2*>(row + (int64_t)hh * hd);
        const float y0 = x.x * cs - x.y * sn, y1 = x.x * sn + x.y * cs;
        float ss = y0 * y0 + y1 * y1;
        for (int d = hd / 4; d >= 1; d >>= 1) ss += shfl_xor(ss, d);
        const float rms = 1.0f / sqrtf(ss / (float)hd + a.eps);
        const float* const w = hh < a.nh ? a.q_norm : a.k_norm;
        const float w0 = w ? w[2 * l] : 1.0f, w1 = w ? w[2 * l + 1] : 1.0f;
        if (hh < a.nh) {
            *reinterpret_cast<float2*>(a.q + ((int64_t)t * a.nh + hh) * hd + 2 * l) =
                make_float2(y0 * rms * w0, y1 * rms * w1);
        } else {
            const int g = hh - a.nh;
            const float2 v = *reinterpret_cast<const float2*>(row + (int64_t)(hh + a.c.nkv) * hd);
            store_pair(static_cast<E*>(a.c.k) + cell + g * a.c.head_stride, y0 * rms * w0, y1 * rms * w1);
            store_pair(static_cast<E*>(a.c.v) + cell + g * a.c.head_stride, v.x, v.y);
        }
    }
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    const int64_t waves = (int64_t)a.n_rows * ((a.nh + a.c.nkv + PA_HEADS - 1) / PA_HEADS);
    // a launch has fewer than 2^32 threads along x
    const int64_t groups = (waves + 3) / 4, gx = groups < 1 << 22 ? groups : 1 << 22;
    const dim3 grid((unsigned)gx, (unsigned)((groups + gx - 1) / gx));
    if (a.c.type == HY_TYPE_F32)
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, s, a);
    else if (a.c.type == HY_TYPE_F16)
        hipLaunchKernelGGL(paged_append_kernel<_Float16>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(paged_append_kernel<__bf16>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace hy
