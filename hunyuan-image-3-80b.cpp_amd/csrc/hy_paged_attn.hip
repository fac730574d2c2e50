// hy_paged_attn.hip -- attention of ragged batches of new tokens over a paged cache
// (hy_paged_attention): out = sum_j softmax_j(scale q . k_j) v_j over the keys a row sees.
#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

// request of a row: the last r with q_start[r] <= t (requests without rows in between have
// equal starts); -1 behind the last
__device__ __forceinline__ int row_request(const int* __restrict__ q_start, int n_req, int t) {
    int lo = 0, hi = n_req;  // q_start[lo] <= t < q_start[hi]
    if (t < q_start[0] || t >= q_start[n_req]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (q_start[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// One wave per (row, head), one key at a time, lane l two dims (or one) of it.
template <class E>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnArgs a) {
    const int64_t wid = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
    if (wid >= (int64_t)a.n_rows * a.nh) return;
    const int t = (int)(wid / a.nh), h = (int)(wid % a.nh), l = threadIdx.x % WAVE, hd = a.c.hd;
    const int r = row_request(a.q_start, a.n_req, t);
    if (r < 0) return;
    const int g = h / (a.nh / a.c.nkv);
    const int cap = a.max_pages << a.c.shift;
    const int kv = min(max(a.kv_len[r], 0), cap);
    const int end = min(a.seen ? a.seen[t] : kv - (a.q_start[r + 1] - t) + 1, kv);
    const bool two = hd == 128;
    const float* const q = a.q + ((int64_t)t * a.nh + h) * hd;
    const float q0 = q[l] * a.scale, q1 = two ? q[64 + l] * a.scale : 0.0f;
    const E* const kb = static_cast<const E*>(a.c.k) + g * a.c.head_stride + l;
    const E* const vb = static_cast<const E*>(a.c.v) + g * a.c.head_stride + l;
    float m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j = 0; j < end; j++) {
        const int page = a.table[(int64_t)r * a.max_pages + (j >> a.c.shift)];
        if (page < 0 || page >= a.c.n_pages) continue;
        const int64_t at = page * a.c.page_stride + (j & ((1 << a.c.shift) - 1)) * a.c.token_stride;
        float s = q0 * (float)kb[at] + (two ? q1 * (float)kb[at + 64] : 0.0f);
        s = wave_sum(s);
        const float mn = fmaxf(m, s);
        const float old = m == mn ? 1.0f : hy_expf(m - mn), p = s == mn ? 1.0f : hy_expf(s - mn);
        m = mn;
        sum = sum * old + p;
        o0 = o0 * old + p * (float)vb[at];
        if (two) o1 = o1 * old + p * (float)vb[at + 64];
    }
    float* const out = a.out + ((int64_t)t * a.nh + h) * hd + l;
    const float inv = m == -INFINITY ? 0.0f : 1.0f / sum;
    out[0] = o0 * inv;
    if (two) out[64] = o1 * inv;
}

size_t paged_attn_ws_bytes(int, int, int) { return 16; }

hipError_t launch_paged_attn(const PagedAttnArgs& a, int, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)a.n_rows * a.nh + 3) / 4));
    if (a.c.type == HY_TYPE_F32)
        hipLaunchKernelGGL(paged_attn_kernel<float>, grid, dim3(256), 0, s, a);
    else if (a.c.type == HY_TYPE_F16)
        hipLaunchKernelGGL(paged_attn_kernel<_Float16>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(paged_attn_kernel<__bf16>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace hy
