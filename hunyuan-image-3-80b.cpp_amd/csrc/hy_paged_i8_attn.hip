// hy_paged_i8_attn.hip -- attention of ragged batches over a paged cache of 8-bit integers
// (hy_paged_attention_i8): out = sum_j softmax_j(scale q . k_j) v_j, k_j and v_j codes times the scale of
// their block.
//
// The simple form: a wave per row and query head, key by key; lane l holds dims l and 64 + l.
#include "hy_device.hpp"
#include "hy_int8.hpp"
#include "hy_paged_part.hpp"

namespace hy {

template <int HD>
__global__ __launch_bounds__(256) void paged_i8_simple_kernel(PagedAttnI8Args g) {
    constexpr int N = HD / 64;
    const PagedAttnArgs& a = g.a;
    const int lane = threadIdx.x % WAVE;
    const int64_t at = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + threadIdx.x / WAVE;
    if (at >= (int64_t)a.n_rows * a.nh) return;
    const int row = (int)(at / a.nh), head = (int)(at % a.nh);
    int r = 0;  // the last request whose rows start at or before this one
    for (int step = 4096; step; step >>= 1)
        if (r + step < a.n_req && a.q_start[r + step] <= row) r += step;
    int start, n, kv;
    part_load(a, r, start, n, kv);
    if (row < start || row >= start + n) return;
    const int end = a.seen ? min(a.seen[row], kv) : kv - n + (row - start) + 1, kvh = head / (a.nh / a.c.nkv);
    const float* const q = a.q + ((int64_t)row * a.nh + head) * HD;
    float qv[N], o[N] = {}, m = -INFINITY, l = 0.0f;
    for (int i = 0; i < N; i++) qv[i] = q[lane + 64 * i] * (a.scale * 1.4426950408889634f);
    for (int j = 0; j < end; j++) {
        const int p = a.table[(int64_t)r * a.max_pages + (j >> a.c.shift)], in = j & ((1 << a.c.shift) - 1);
        if (p < 0 || p >= a.c.n_pages) continue;
        const int64_t cell = p * a.c.page_stride + kvh * a.c.head_stride + in * a.c.token_stride + lane;
        const int64_t b = (((int64_t)p * a.c.nkv + kvh) << (a.c.shift - g.bshift)) + (in >> g.bshift);
        const int8_t* const k = static_cast<const int8_t*>(a.c.k) + cell;
        const int8_t* const v = static_cast<const int8_t*>(a.c.v) + cell;
        float s = 0.0f;
        for (int i = 0; i < N; i++) s = fmaf(qv[i], (float)k[64 * i], s);
        s = wave_sum(s) * g.ks[b];
        if (s == -INFINITY) s = __builtin_nanf("");
        const float mn = fmaxf(m, s), alpha = __builtin_amdgcn_exp2f(m - mn);
        const float w = __builtin_amdgcn_exp2f(s - mn), vs = g.vs[b];
        m = mn;
        l = l * alpha + w;
        for (int i = 0; i < N; i++) o[i] = o[i] * alpha + w * ((float)v[64 * i] * (vs < INFINITY ? vs : __builtin_nanf("")));
    }
    for (int i = 0; i < N; i++)
        a.out[((int64_t)row * a.nh + head) * HD + lane + 64 * i] = l == 0.0f ? 0.0f : o[i] / l;
}

size_t paged_attn_i8_ws_bytes(int, int, int, int) { return 16; }

hipError_t launch_paged_attn_i8(const PagedAttnI8Args& a, int, hipStream_t s) {
    const int64_t n = ((int64_t)a.a.n_rows * a.a.nh + 3) / 4, gx = n < 1 << 22 ? n : 1 << 22;
    const dim3 grid((unsigned)gx, (unsigned)((n + gx - 1) / gx));  // fewer than 2^32 threads along x
    if (a.a.c.hd == 128)
        hipLaunchKernelGGL(paged_i8_simple_kernel<128>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(paged_i8_simple_kernel<64>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace hy
