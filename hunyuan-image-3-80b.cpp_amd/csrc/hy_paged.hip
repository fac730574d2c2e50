// hy_paged.hip -- the tables of a paged cache built from lengths, and the write into it:
//  * paged_plan_kernel: pages taken and given back, block tables, row offsets, positions and
//    slots of a step (hy_paged_plan);
//  * paged_append_kernel: rotary embedding + QK-norm of the projection's output, queries to
//    [rows][nh][hd], keys and values to their slots in the cache's type.
#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

// ---------------------------------------------------------------- tables and slots
// One work group: every thread owns PL_PER consecutive requests, and the three sums over
// requests (rows, pages given back, pages taken) are scans over the threads' totals.
constexpr int PL_THREADS = 1024, PL_PER = PG_MAX_REQ / PL_THREADS;

// exclusive sum over the work group's threads; total: of all of them
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t& total) {
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    int64_t s = v;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const int64_t o = __shfl_up(s, d, WAVE);
        if (lane >= d) s += o;
    }
    __syncthreads();  // part may still be read
    if (lane == WAVE - 1) part[wave] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PL_THREADS / WAVE; w++) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + s - v;
}

__global__ __launch_bounds__(PL_THREADS) void paged_plan_kernel(PagedPlanArgs a) {
    __shared__ int64_t part[PL_THREADS / WAVE];
    const int tid = threadIdx.x;
    const int r0 = tid * PL_PER;
    const int page = 1 << a.shift;
    int cached[PL_PER], held[PL_PER], rows[PL_PER], status[PL_PER];
    int64_t add[PL_PER];
    int64_t sum = 0, total;
#pragma unroll
    for (int i = 0; i < PL_PER; i++) {
        const int r = r0 + i;
        const bool live = r < a.n_req;
        cached[i] = live ? a.cached[r] : 0;
        add[i] = live ? a.add[r] : 0;
        held[i] = live ? a.held[r] : 0;
        rows[i] = add[i] >= 0 && add[i] <= a.n_rows ? (int)add[i] : 0;
        sum += rows[i];
    }
    const int64_t n_free_in = a.n_free[0];
    // every read of held and n_free is done before any write (they may be the outputs)
    int64_t at = block_scan(sum, part, total);
    int want[PL_PER], start[PL_PER];
    int64_t give_sum = 0, take_sum = 0;
#pragma unroll
    for (int i = 0; i < PL_PER; i++) {
        const int r = r0 + i;
        const int64_t len = (int64_t)cached[i] + add[i], w = (len + page - 1) >> a.shift;
        const bool bad = cached[i] < 0 || add[i] < 0 || at + add[i] > a.n_rows || held[i] < 0 ||
                         held[i] > a.max_pages;
        status[i] = bad ? 3 : w > a.max_pages ? 2 : 0;
        want[i] = status[i] ? held[i] : (int)w;  // refused requests keep what they have
        start[i] = (int)min(at, (int64_t)a.n_rows);
        if (r < a.n_req) a.q_start[r] = start[i];
        at += rows[i];
        give_sum += max(held[i] - want[i], 0);
        take_sum += max(want[i] - held[i], 0);
    }
    if (tid == 0) a.q_start[a.n_req] = (int)min(total, (int64_t)a.n_rows);
    const int n_rows_used = (int)min(total, (int64_t)a.n_rows);
    int64_t given, taken;
    int64_t push = min(max(n_free_in, (int64_t)0), (int64_t)a.n_pages) + block_scan(give_sum, part, given);
    int64_t upto = block_scan(take_sum, part, taken);
    const int64_t avail = min(min(max(n_free_in, (int64_t)0), (int64_t)a.n_pages) + given, (int64_t)a.n_pages);
#pragma unroll
    for (int i = 0; i < PL_PER; i++) {
        int* row = a.table + (int64_t)(r0 + i) * a.max_pages;
        for (int k = want[i]; k < held[i]; k++, push++)
            if (push < a.n_pages) a.free_[push] = row[k];
    }
    __syncthreads();  // the stack is whole
    int64_t used = 0;
#pragma unroll
    for (int i = 0; i < PL_PER; i++) {
        const int r = r0 + i;
        if (r >= a.n_req) continue;
        const int need = max(want[i] - held[i], 0);
        upto += need;
        if (need && upto > avail) {
            status[i] = 1;
            want[i] = held[i];
        } else {
            used += need;
            int* row = a.table + (int64_t)r * a.max_pages;
            for (int k = 0; k < need; k++) row[held[i] + k] = a.free_[avail - 1 - (upto - need) - k];
        }
        a.status[r] = status[i];
        a.held_out[r] = status[i] == 0 ? want[i] : held[i];
        a.kv_len[r] = status[i] == 0 ? cached[i] + (int)add[i] : 0;
    }
    (void)block_scan(used, part, total);  // and a barrier: the tables are whole
    if (tid == 0) a.n_free_out[0] = (int)(avail - total);
#pragma unroll
    for (int i = 0; i < PL_PER; i++) {
        const int r = r0 + i;
        const int* row = a.table + (int64_t)r * a.max_pages;
        for (int k = 0; k < rows[i] && start[i] + k < n_rows_used; k++) {
            int pos = 0, slot = -1;
            if (status[i] == 0) {
                pos = cached[i] + k;
                const int p = row[pos >> a.shift];
                if (p >= 0 && p < a.n_pages) slot = (p << a.shift) + (pos & (page - 1));
            }
            a.positions[start[i] + k] = pos;
            a.slots[start[i] + k] = slot;
        }
    }
    for (int t = n_rows_used + tid; t < a.n_rows; t += PL_THREADS) {
        a.positions[t] = 0;
        a.slots[t] = -1;
    }
}

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(PL_THREADS), 0, s, a);
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
    const int64_t wid = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
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
    const dim3 grid((unsigned)((waves + 3) / 4));
    if (a.c.type == HY_TYPE_F32)
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, s, a);
    else if (a.c.type == HY_TYPE_F16)
        hipLaunchKernelGGL(paged_append_kernel<_Float16>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(paged_append_kernel<__bf16>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace hy
