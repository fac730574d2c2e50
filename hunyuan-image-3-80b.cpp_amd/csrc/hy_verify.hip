// hy_verify.hip -- verification of drafted tokens (hy_verify_drafts): acceptance of each
// draft against the target's probability, and the next token by inversion of what is left.
//
// Rows are read in slices of VF_SLICE logits, one work group each:
//  * verify_rows_kernel: every row's slice: largest logit and its index, sum of weights;
//  * verify_rest_kernel: per request, joins its rows' slices, accepts drafts up to the first
//    refusal, and sums what is left to draw from over a slice of the row where that happened;
//  * verify_pick_kernel: per request, finds the slice that u falls into, and the token in it.
// Bound: the logits' bytes (one pass over all rows, one over a row per request), beside some 20
// 64-bit operations per logit.
//
// Every number is 64-bit: a token is decided by where u falls between two running sums of
// up to a few hundred thousand terms, and with n tokens of similar weight an error e of the
// sums moves n e of the decisions (f32: about one in a hundred at n = 10^5).
#include "hy_device.hpp"
#include "hy_paged.hpp"

namespace hy {

// 2^y: whole part n by ldexp, the rest |r| <= 1/2 by the series of e^(r ln 2) to degree 11, its
// powers of ln 2 in the coefficients (remainder (0.347)^12 / 12! = 6e-15).  y below -1100 and
// no number (the masked logit of an infinite temperature, -inf times 0): 0.
__device__ __forceinline__ double exp2_f64(double y) {
    y = fmax(y, -1100.0);
    const double n = rint(y), r = y - n;
    constexpr double L = 0.6931471805599453094, L2 = L * L, L4 = L2 * L2, L8 = L4 * L4;
    double p = L8 * L2 * L / 39916800;
    p = fma(p, r, L8 * L2 / 3628800);
    p = fma(p, r, L8 * L / 362880);
    p = fma(p, r, L8 / 40320);
    p = fma(p, r, L4 * L2 * L / 5040);
    p = fma(p, r, L4 * L2 / 720);
    p = fma(p, r, L4 * L / 120);
    p = fma(p, r, L4 / 24);
    p = fma(p, r, L2 * L / 6);
    p = fma(p, r, L2 / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// weight of a logit, 2^((l - m) c): the difference first, it is exact for logits near m of any size
__device__ __forceinline__ double weight(float l, double c, double m) { return exp2_f64(((double)l - m) * c); }

constexpr int VF_THREADS = 256, VF_VEC = 8, VF_SLICE = VF_THREADS * VF_VEC * 4;

typedef float f4_any_t __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

template <class T, class F>
__device__ __forceinline__ T wave_fold(T v, F f) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = f(v, shfl_xor(v, d));
    return v;
}
// over the work group; part: one T per wave
template <class T, class F>
__device__ __forceinline__ T block_fold(T v, T* part, F f) {
    v = wave_fold(v, f);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = v;
    __syncthreads();
    T r = part[0];
#pragma unroll
    for (int w = 1; w < VF_THREADS / WAVE; w++) r = f(r, part[w]);
    return r;
}

struct VfSlice {   // of a row
    double z;      // sum of 2^((l - m) c)
    float m;       // largest logit
    int arg;       // its lowest index
    int bad, pad;  // a NaN or +inf among the logits
};
struct VfRest {    // of a slice of the row to draw from
    double rest, all;  // sums of what is left of p after q, and of p
};
struct VfPick {    // of a request
    double z;
    float m;
    int accepted;  // drafts; -1: nothing to verify
    int row;       // to draw from; -1: none
    int tok;       // the next token, where it needs no drawing (row = -1)
    int x;         // the draft refused in it, -1: none was
    int pad;
};

__host__ __device__ __forceinline__ int vf_slices(int vocab) { return (vocab + VF_SLICE - 1) / VF_SLICE; }

// this thread's logits of slice s: element 4 (tid + VF_THREADS j) + i of it, fill past the end
__device__ __forceinline__ void load_slice(const float* row, int vocab, int s, float fill, f4_any_t (&x)[VF_VEC]) {
#pragma unroll
    for (int j = 0; j < VF_VEC; j++) {
        const int i = s * VF_SLICE + 4 * ((int)threadIdx.x + VF_THREADS * j);
        if (i + 4 <= vocab) {
            x[j] = *reinterpret_cast<const f4_any_t*>(row + i);
        } else {
#pragma unroll
            for (int n = 0; n < 4; n++) x[j][n] = i + n < vocab ? row[i + n] : fill;
        }
    }
}

// a request's rows [lo, hi), none where nothing can be verified
__device__ __forceinline__ bool vf_rows(const VerifyArgs& a, int r, int& lo, int& hi) {
    lo = max(a.q_start[r], 0);
    hi = min(a.q_start[r + 1], a.n_rows);
    return hi > lo && hi - lo <= a.max_new;
}

__global__ __launch_bounds__(VF_THREADS) void verify_rows_kernel(VerifyArgs a, VfSlice* __restrict__ out) {
    __shared__ float pf[VF_THREADS / WAVE];
    __shared__ int pi[VF_THREADS / WAVE];
    __shared__ double pd[VF_THREADS / WAVE];
    const int V = a.vocab, S = vf_slices(V), row = (int)(blockIdx.x / S), s = (int)(blockIdx.x % S);
    const float* const l = a.logits + (int64_t)row * V;
    f4_any_t x[VF_VEC];
    load_slice(l, V, s, -INFINITY, x);
    // the row's request, 64 starts at a time: the last r with q_start[r] <= row
    const int lane = threadIdx.x % WAVE;
    int r = 0;
    for (int step = 64; step >= 1; step = step > 1 && a.n_req > 64 ? 1 : 0) {
        if (step == 64 && a.n_req <= 64) step = 1;
        const int i = r + lane * step;
        r += (__builtin_popcountll(__ballot(i < a.n_req && a.q_start[min(i, a.n_req)] <= row)) - 1) * step;
        if (r < 0) return;
    }
    int lo, hi;
    if (!vf_rows(a, r, lo, hi) || row < lo || row >= hi) return;
    const float temp = a.temp ? a.temp[r] : 1.0f;
    float m = -INFINITY;
    int bad = 0;
#pragma unroll
    for (int j = 0; j < VF_VEC; j++)
#pragma unroll
        for (int n = 0; n < 4; n++) {
            bad |= !(x[j][n] < INFINITY);
            m = fmaxf(m, x[j][n]);
        }
    m = block_fold(m, pf, [](float p, float q) { return fmaxf(p, q); });
    bad = __syncthreads_or(bad);
    int arg = V;
    double z = 0.0;
    if (!(temp > 0.0f)) {  // the same for the work group, as all conditions here
#pragma unroll
        for (int j = VF_VEC - 1; j >= 0; j--)
#pragma unroll
            for (int n = 3; n >= 0; n--)
                if (x[j][n] == m) arg = s * VF_SLICE + 4 * ((int)threadIdx.x + VF_THREADS * j) + n;
        arg = block_fold(arg, pi, [](int p, int q) { return min(p, q); });
    } else if (m > -INFINITY && !bad) {
        const double c = 1.4426950408889634 / (double)temp;
#pragma unroll
        for (int j = 0; j < VF_VEC; j++)
#pragma unroll
            for (int n = 0; n < 4; n++) z += weight(x[j][n], c, (double)m);
        z = block_fold(z, pd, [](double p, double q) { return p + q; });
    }
    if (threadIdx.x == 0) out[(int64_t)row * S + s] = {z, m, arg, bad, 0};
}

__global__ __launch_bounds__(VF_THREADS) void verify_rest_kernel(VerifyArgs a, const VfSlice* __restrict__ part,
                                                                VfRest* __restrict__ rest, VfPick* __restrict__ pick) {
    constexpr int WAVES = VF_THREADS / WAVE;
    __shared__ VfPick found[WAVES];  // where a wave's row ends its request: row >= -1
    __shared__ int ends[WAVES];
    __shared__ double pd[WAVES];
    const int V = a.vocab, S = vf_slices(V), r = (int)(blockIdx.x / S), s = (int)(blockIdx.x % S);
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    int lo, hi;
    if (!vf_rows(a, r, lo, hi)) {
        if (s == 0 && threadIdx.x == 0) pick[r] = {0.0, 0.0f, -1, -1, -1, -1, 0};
        return;
    }
    const int n = hi - lo;
    const float temp = a.temp ? a.temp[r] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    const double c = 1.4426950408889634 / (double)temp;
    VfPick p;
    for (int i0 = 0;; i0 += WAVES) {  // a row per wave; the last row always ends the request
        const int i = i0 + wave, row = lo + min(i, n - 1);
        const VfSlice* const sl = part + (int64_t)row * S;
        const bool last = i >= n - 1;
        const int x = last ? -1 : a.ids[row + 1];
        float m = -INFINITY;
        int bad = 0, arg = V;
        for (int k = lane; k < S; k += WAVE) {
            const VfSlice v = sl[k];
            bad |= v.bad;
            if (v.m > m) {
                m = v.m;
                arg = v.arg;  // slices come in ascending order
            }
        }
        const float mm = wave_fold(m, [](float u, float v) { return fmaxf(u, v); });
        arg = wave_fold(m == mm ? arg : V, [](int u, int v) { return min(u, v); });
        bad = __any(bad);
        double z = 0.0;
        if (!greedy)
            for (int k = lane; k < S; k += WAVE) z += sl[k].z * exp2_f64(((double)sl[k].m - (double)mm) * c);
        z = wave_fold(z, [](double u, double v) { return u + v; });
        VfPick e = {z, mm, i, -1, -1, -1, 0};
        bool end = true;
        if (bad || mm == -INFINITY) {
            // no distribution
        } else if (greedy) {
            end = last || x != arg;
            e.tok = arg;
        } else {
            bool take = false;
            if (!last && x >= 0 && x < V) {
                const double q = a.draft ? (double)a.draft[(int64_t)row * V + x] : 1.0;
                const double w = weight(a.logits[(int64_t)row * V + x], c, (double)mm);
                take = (double)a.u_accept[row] * q < w / z;
            }
            end = !take;
            e.row = row;
            e.x = last ? -1 : x;
        }
        __syncthreads();  // the last round's are read
        if (lane == 0) {
            found[wave] = e;
            ends[wave] = end && i < n;
        }
        __syncthreads();
        int w = 0;
        while (w < WAVES && !ends[w]) w++;
        if (w < WAVES) {
            p = found[w];
            break;
        }
    }
    if (s == 0 && threadIdx.x == 0) pick[r] = p;
    if (p.row < 0) return;
    // what is left: p - q where positive (a draft without probabilities: p without it), all of p
    // for the row behind the last draft
    const bool refused = p.row < hi - 1;
    const float* const l = a.logits + (int64_t)p.row * V;
    f4_any_t x[VF_VEC], q[VF_VEC];
    load_slice(l, V, s, -INFINITY, x);
    if (a.draft && refused) load_slice(a.draft + (int64_t)p.row * V, V, s, 0.0f, q);
    const double m = (double)p.m, inv = 1.0 / p.z;
    double left = 0.0, all = 0.0;
#pragma unroll
    for (int j = 0; j < VF_VEC; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double v = weight(x[j][k], c, m) * inv;
            all += v;
            if (refused) {
                const int i = s * VF_SLICE + 4 * ((int)threadIdx.x + VF_THREADS * j) + k;
                if (a.draft)
                    left += v > (double)q[j][k] ? v - (double)q[j][k] : 0.0;
                else
                    left += i == p.x ? 0.0 : v;
            }
        }
    all = block_fold(all, pd, [](double u, double v) { return u + v; });
    left = block_fold(left, pd, [](double u, double v) { return u + v; });
    if (threadIdx.x == 0) rest[(int64_t)r * S + s] = {refused ? left : all, all};
}

__global__ __launch_bounds__(VF_THREADS) void verify_pick_kernel(VerifyArgs a, const VfRest* __restrict__ rest,
                                                                const VfPick* __restrict__ pick) {
    constexpr int WAVES = VF_THREADS / WAVE;
    __shared__ double runs[VF_VEC * WAVES];
    static_assert(VF_VEC * WAVES <= WAVE, "a run per lane");
    __shared__ int pi[WAVES];
    const int V = a.vocab, S = vf_slices(V), r = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const VfPick p = pick[r];
    const int lo = max(a.q_start[r], 0), hi = min(a.q_start[r + 1], a.n_rows);
    const float temp = a.temp ? a.temp[r] : 1.0f, u_sample = a.u_sample[r];
    int tok = p.tok;
    if (p.row >= 0) {
        const bool refused = p.row < hi - 1;
        const double c = 1.4426950408889634 / (double)temp;
        const VfRest* const rs = rest + (int64_t)r * S;
        // sums over the slices, in order; every wave for itself
        double left = 0.0, all = 0.0;
        for (int k = lane; k < S; k += WAVE) {
            left += rs[k].rest;
            all += rs[k].all;
        }
        left = wave_fold(left, [](double u, double v) { return u + v; });
        all = wave_fold(all, [](double u, double v) { return u + v; });
        const bool whole = !(left > 0.0);  // nothing is left: from p
        const double thr = (double)u_sample * (whole ? all : left);
        double before = 0.0;
        int s = -1, s_any = -1;  // the first slice whose running sum exceeds thr; the last one with any weight
        double s_before = 0.0, any_before = 0.0;
        for (int k0 = 0; k0 < S && s < 0; k0 += WAVE) {
            const int k = k0 + lane;
            const double v = k < S ? (whole ? rs[k].all : rs[k].rest) : 0.0;
            double run = v;
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const double o = __shfl_up(run, d, WAVE);
                if (lane >= d) run += o;
            }
            run += before;
            const unsigned long long over = __ballot(v > 0.0 && run > thr), any = __ballot(v > 0.0);
            if (any) {
                const int e = 63 - __builtin_clzll(any);
                s_any = k0 + e;
                any_before = __shfl(run - v, e, WAVE);
            }
            if (over) {
                const int e = __builtin_ctzll(over);
                s = k0 + e;
                s_before = __shfl(run - v, e, WAVE);
            }
            before = __shfl(run, WAVE - 1, WAVE);
        }
        if (s < 0) {  // u rounds to the whole
            s = s_any;
            s_before = any_before;
        }
        // in the slice: VF_VEC x WAVES runs of 4 x 64 tokens (load_slice's order), their sums, then
        // the lanes of the run that u falls into
        const float* const dr = a.draft && refused && !whole ? a.draft + (int64_t)p.row * V : nullptr;
        f4_any_t x[VF_VEC], q[VF_VEC];
        load_slice(a.logits + (int64_t)p.row * V, V, s, -INFINITY, x);
        if (dr) load_slice(dr, V, s, 0.0f, q);
        const double m = (double)p.m, inv = 1.0 / p.z;
        double sum[VF_VEC];
        auto left_of = [&](int j, int k) {
            const double v = weight(x[j][k], c, m) * inv;
            if (dr) return v > (double)q[j][k] ? v - (double)q[j][k] : 0.0;
            return refused && !whole && s * VF_SLICE + 4 * (tid + VF_THREADS * j) + k == p.x ? 0.0 : v;
        };
#pragma unroll
        for (int j = 0; j < VF_VEC; j++) {
            double u = 0.0;
#pragma unroll
            for (int k = 0; k < 4; k++) u += left_of(j, k);
            sum[j] = u;
        }
#pragma unroll
        for (int j = 0; j < VF_VEC; j++) {
            const double u = wave_fold(sum[j], [](double u, double v) { return u + v; });
            if (lane == 0) runs[j * WAVES + wave] = u;
        }
        __syncthreads();
        const double mine_run = lane < VF_VEC * WAVES ? runs[lane] : 0.0;  // a run per lane
        double run = mine_run;
#pragma unroll
        for (int d = 1; d < VF_VEC * WAVES; d <<= 1) {
            const double o = __shfl_up(run, d, WAVE);
            if (lane >= d) run += o;
        }
        const unsigned long long over = __ballot(mine_run > 0.0 && s_before + run > thr), some = __ballot(mine_run > 0.0);
        // no run: the sums of the slice and of its runs may round apart
        const int at = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        const double at_before = s_before + __shfl(run - mine_run, max(at, 0), WAVE);
        tok = -1;
        if (at >= 0 && at % WAVES == wave) {
            const int j = at / WAVES;
            f4_any_t xj = x[0], qj = q[0];
            double mine = sum[0];
#pragma unroll
            for (int k = 1; k < VF_VEC; k++)
                if (k == j) {
                    xj = x[k];
                    qj = q[k];
                    mine = sum[k];
                }
            x[0] = xj;
            q[0] = qj;
            double upto = mine;
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const double o = __shfl_up(upto, d, WAVE);
                if (lane >= d) upto += o;
            }
            double here = at_before + upto - mine;
            const int i0 = s * VF_SLICE + 4 * (tid + VF_THREADS * j);
            int found = V, any = -1;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                double v = weight(x[0][k], c, m) * inv;
                if (dr)
                    v = v > (double)q[0][k] ? v - (double)q[0][k] : 0.0;
                else if (refused && !whole && i0 + k == p.x)
                    v = 0.0;
                here += v;
                if (v > 0.0) {
                    any = i0 + k;
                    if (found == V && here > thr) found = i0 + k;
                }
            }
            found = wave_fold(found, [](int u, int v) { return min(u, v); });
            any = wave_fold(any, [](int u, int v) { return max(u, v); });
            tok = found < V ? found : any;
        }
        tok = block_fold(tok, pi, [](int u, int v) { return max(u, v); });
    }
    int* const out = a.tokens + (int64_t)r * a.max_new;
    for (int i = tid; i < a.max_new; i += VF_THREADS) out[i] = i < p.accepted ? a.ids[lo + i + 1] : i == p.accepted ? tok : -1;
    if (tid == 0) a.accepted[r] = p.accepted;
}

static size_t al16(size_t n) { return (n + 15) / 16 * 16; }

size_t verify_ws_bytes(int n_req, int n_rows, int vocab) {
    const size_t S = vf_slices(vocab);
    return al16(n_rows * S * sizeof(VfSlice)) + al16(n_req * S * sizeof(VfRest)) + al16(n_req * sizeof(VfPick));
}

hipError_t launch_verify_drafts(const VerifyArgs& a, hipStream_t s) {
    const size_t S = vf_slices(a.vocab);
    uint8_t* const ws = static_cast<uint8_t*>(a.ws);
    VfSlice* const part = reinterpret_cast<VfSlice*>(ws);
    VfRest* const rest = reinterpret_cast<VfRest*>(ws + al16(a.n_rows * S * sizeof(VfSlice)));
    VfPick* const pick = reinterpret_cast<VfPick*>(reinterpret_cast<uint8_t*>(rest) + al16(a.n_req * S * sizeof(VfRest)));
    hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)(a.n_rows * S)), dim3(VF_THREADS), 0, s, a, part);
    hipLaunchKernelGGL(verify_rest_kernel, dim3((unsigned)(a.n_req * S)), dim3(VF_THREADS), 0, s, a, part, rest, pick);
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)a.n_req), dim3(VF_THREADS), 0, s, a, rest, pick);
    return hipGetLastError();
}

}  // namespace hy
