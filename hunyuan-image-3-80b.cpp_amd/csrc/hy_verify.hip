// hy_verify.hip -- verification of drafted tokens (hy_verify_drafts): acceptance of each
// draft against the target's probability, and the next token by inversion of what is left.
//
// Every number is 64-bit: a token is decided by where u falls between two running sums of
// up to a few hundred thousand terms, and with n tokens of similar weight an error e of the
// sums moves n e of the decisions (f32: about one in a hundred at n = 10^5).
#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

// 2^y to 1e-14: whole part by ldexp, the rest |r| <= 1/2 by the series of e^(r ln 2) to
// degree 11 (remainder (0.347)^12 / 12! = 6e-15).  2^-inf = 0,
// and so is the masked logit of an infinite temperature, -inf times 0.
__device__ __forceinline__ double exp2_f64(double y) {
    if (!(y >= -1100.0)) return 0.0;
    const double n = rint(y), r = (y - n) * 0.6931471805599453;
    double p = 1.0 / 39916800;
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}

constexpr int VF_THREADS = 1024;

template <class T, class F>
__device__ __forceinline__ T block_fold(T v, T* part, F f) {
    for (int d = 32; d >= 1; d >>= 1) v = f(v, shfl_xor(v, d));
    __syncthreads();
    if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = v;
    __syncthreads();
    T r = part[0];
    for (int w = 1; w < VF_THREADS / WAVE; w++) r = f(r, part[w]);
    return r;
}

// One work group per request, row after row.
__global__ __launch_bounds__(VF_THREADS) void verify_kernel(VerifyArgs a) {
    __shared__ double pd[VF_THREADS / WAVE];
    __shared__ float pf[VF_THREADS / WAVE];
    __shared__ int pi[VF_THREADS / WAVE];
    __shared__ double run[VF_THREADS + 1];
    const int r = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const int lo = max(a.q_start[r], 0), hi = min(a.q_start[r + 1], a.n_rows), n = hi - lo;
    int* const out = a.tokens + (int64_t)r * a.max_new;
    if (n <= 0 || n > a.max_new) {
        for (int i = tid; i < a.max_new; i += VF_THREADS) out[i] = -1;
        if (tid == 0) a.accepted[r] = -1;
        return;
    }
    const float temp = a.temp ? a.temp[r] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    const double c = 1.4426950408889634 / (double)temp;
    int acc = 0, tok = -1;
    for (;; acc++) {
        const int row = lo + acc;
        const float* const l = a.logits + (int64_t)row * V;
        float mx = -INFINITY;
        int bad = 0;
        for (int i = tid; i < V; i += VF_THREADS) {
            const float x = l[i];
            bad |= !(x < INFINITY);
            mx = fmaxf(mx, x);
        }
        mx = block_fold(mx, pf, [](float x, float y) { return fmaxf(x, y); });
        bad = block_fold(bad, pi, [](int x, int y) { return x | y; });
        if (bad || mx == -INFINITY) break;  // no distribution
        const bool last = acc == n - 1;
        const int x = last ? -1 : a.ids[row + 1];
        if (greedy) {
            int best = V;
            for (int i = tid; i < V; i += VF_THREADS)
                if (l[i] == mx) best = min(best, i);
            best = block_fold(best, pi, [](int p, int q) { return min(p, q); });
            if (!last && x == best) continue;
            tok = best;
            break;
        }
        auto weight = [&](int i) { return exp2_f64(((double)l[i] - (double)mx) * c); };
        double z = 0.0;
        for (int i = tid; i < V; i += VF_THREADS) z += weight(i);
        z = block_fold(z, pd, [](double p, double q) { return p + q; });
        const float* const dr = a.draft && !last ? a.draft + (int64_t)row * V : nullptr;
        if (!last && x >= 0 && x < V) {
            const double q = dr ? (double)dr[x] : 1.0;
            if ((double)a.u_accept[row] * q < weight(x) / z) continue;
        }
        // draw: thread i owns the i-th stretch of the vocabulary
        const int per = (V + VF_THREADS - 1) / VF_THREADS;
        const int i0 = min(tid * per, V), i1 = min(i0 + per, V);
        for (int whole = last; whole < 2; whole++) {
            auto rest = [&](int i) {
                const double p = weight(i) / z;
                if (whole) return p;
                if (dr) return p > (double)dr[i] ? p - (double)dr[i] : 0.0;
                return i == x ? 0.0 : p;
            };
            double s = 0.0;
            for (int i = i0; i < i1; i++) s += rest(i);
            __syncthreads();
            run[tid + 1] = s;
            if (tid == 0) run[0] = 0.0;
            __syncthreads();
            if (tid == 0)
                for (int i = 1; i <= VF_THREADS; i++) run[i] += run[i - 1];
            __syncthreads();
            const double all = run[VF_THREADS], thr = (double)a.u_sample[r] * all;
            if (!(all > 0.0)) continue;
            int found = V, any = -1;
            double at = run[tid];
            if (run[tid + 1] > run[tid])
                for (int i = i0; i < i1; i++) {
                    const double v = rest(i);
                    at += v;
                    if (v > 0.0) {
                        any = i;
                        if (found == V && at > thr) found = i;
                    }
                }
            found = block_fold(found, pi, [](int p, int q) { return min(p, q); });
            any = block_fold(any, pi, [](int p, int q) { return max(p, q); });
            tok = found < V ? found : any;
            break;
        }
        break;
    }
    for (int i = tid; i < a.max_new; i += VF_THREADS) out[i] = i < acc ? a.ids[lo + i + 1] : i == acc ? tok : -1;
    if (tid == 0) a.accepted[r] = acc;
}

size_t verify_ws_bytes(int, int, int) { return 16; }

hipError_t launch_verify_drafts(const VerifyArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(verify_kernel, dim3((unsigned)a.n_req), dim3(VF_THREADS), 0, s, a);
    return hipGetLastError();
}

}  // namespace hy
