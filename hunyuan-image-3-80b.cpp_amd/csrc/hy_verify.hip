// hy_verify.hip -- verification of drafted tokens (hy_verify_drafts): acceptance of each
// draft against the target's probability, and the next token by inversion of what is left.
//
// Rows are read in slices of VF_SLICE logits, one work group each:
//  * verify_rows_kernel: every row's slice: largest logit and its index, sum of the weights but
//    the draft's (a refused draft without probabilities leaves just these to draw from);
//  * verify_rest_kernel, for drafts with probabilities: per request, joins its rows' slices,
//    accepts drafts up to the first refusal, and sums what is left to draw from over a slice of
//    the row refused;
//  * verify_pick_kernel: per request, finds the slice that u falls into, and the token in it
//    (without probabilities it accepts first, the slices' sums are there already).
// Bound: the logits' bytes (one pass over all rows, one over a refused row and its draft's), beside
// some 20 64-bit operations per logit; few rows: the latency of the kernels' dependent reads.
// Vocabulary 133120, 226 rows of 64 requests (120 MB; 22 us at a copy's rate, and as long for the
// operations): rows 30 us, rest 13, pick 8; 20 rows of 4 requests: rows 6, pick 8.6.
//
// Every number is 64-bit: a token is decided by where u falls between two running sums of
// up to a few hundred thousand terms, and with n tokens of similar weight an error e of the
// sums moves n e of the decisions (f32: about one in a hundred at n = 10^5).
#include "hy_device.hpp"
#include "hy_paged.hpp"
#include "hy_paged_split.hpp"

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
// verify_pick_kernel: one work group per request, 256 threads 10.5 us, 512 8.6, 1024 10.0
constexpr int VP_THREADS = 512, VP_VEC = VF_SLICE / 4 / VP_THREADS;

typedef float f4_any_t __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

// f over the wave, the same bits in every lane: rotations by 8 .. 1 in 16 lanes, then rows and
// halves; vector operations, a shuffle takes the way through LDS
template <int CTRL, class T>
__device__ __forceinline__ T dpp(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, false);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
    }
}
template <class T, class F>
__device__ __forceinline__ T wave_fold(T v, F f) {
    v = f(v, dpp<0x128>(v));
    v = f(v, dpp<0x124>(v));
    v = f(v, dpp<0x122>(v));
    v = f(v, dpp<0x121>(v));
    if constexpr (sizeof(T) == 8) {
        const auto join = [](uint32_t lo, uint32_t hi) { return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo); };
        uint64_t u = __builtin_bit_cast(uint64_t, v);
        const auto l16 = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
        const auto h16 = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
        u = __builtin_bit_cast(uint64_t, f(join(l16[0], h16[0]), join(l16[1], h16[1])));
        const auto l32 = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
        const auto h32 = __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
        return f(join(l32[0], h32[0]), join(l32[1], h32[1]));
    } else {
        uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto g = [&](uint32_t p, uint32_t q) {
            return __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(T, p), __builtin_bit_cast(T, q)));
        };
        return __builtin_bit_cast(T, with_half(with_row(u, g), g));
    }
}
__device__ __forceinline__ double wave_sum(double v) {
    return wave_fold(v, [](double p, double q) { return p + q; });
}
__device__ __forceinline__ double read_lane(double v, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)u, l));
}
// inclusive sum over the lanes: shifts inside 16 lanes, then the rows' last lanes to those behind
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp<0x111>(v);
    v += dpp<0x112>(v);
    v += dpp<0x114>(v);
    v += dpp<0x118>(v);
    const int lane = threadIdx.x % WAVE;
    const double r0 = read_lane(v, 15), r1 = read_lane(v, 31), r2 = read_lane(v, 47);
    return v + (lane < 16 ? 0.0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2);
}
// over the work group; part: one T per wave
template <int THREADS, class T, class F>
__device__ __forceinline__ T block_fold(T v, T* part, F f) {
    v = wave_fold(v, f);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = v;
    __syncthreads();
    T r = part[0];
#pragma unroll
    for (int w = 1; w < THREADS / WAVE; w++) r = f(r, part[w]);
    return r;
}

struct VfSlice {   // of a row
    double z;      // sum of 2^((l - m) c), but the row's draft
    float m;       // largest logit
    int arg;       // its lowest index
    int bad, pad;  // a NaN or +inf among the logits
};
struct VfPick {    // of a request
    double z;
    float m;
    float lx;      // logit of x
    int accepted;  // drafts; -1: nothing to verify
    int row;       // to draw from; -1: none
    int tok;       // the next token, where it needs no drawing (row = -1)
    int x;         // the draft refused in it, -1: none was, or it is outside the vocabulary
    int refused, pad;
};

__host__ __device__ __forceinline__ int vf_slices(int vocab) { return (vocab + VF_SLICE - 1) / VF_SLICE; }

// this thread's logits of slice s: element 4 (tid + threads j) + i of it, fill past the end
template <int VEC>
__device__ __forceinline__ void load_slice(const float* row, int vocab, int s, float fill, f4_any_t (&x)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        const int i = s * VF_SLICE + 4 * ((int)threadIdx.x + VF_SLICE / 4 / VEC * j);
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
    constexpr int WAVES = VF_THREADS / WAVE;
    __shared__ VfSlice of_wave[WAVES];
    const int V = a.vocab, S = vf_slices(V), row = (int)(blockIdx.x / S), s = (int)(blockIdx.x % S);
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    f4_any_t x[VF_VEC];
    load_slice(a.logits + (int64_t)row * V, V, s, -INFINITY, x);
    int draft = a.ids[min(row + 1, a.n_rows - 1)];
    // the row's request, 64 starts at a time: the last r with q_start[r] <= row
    int r = 0;
    for (int step = a.n_req > 64 ? 64 : 1; step; step = step > 1) {
        const int i = r + lane * step;
        r += (__builtin_popcountll(__ballot(i < a.n_req && a.q_start[min(i, a.n_req)] <= row)) - 1) * step;
        if (r < 0) return;
    }
    int lo, hi;
    if (!vf_rows(a, r, lo, hi) || row < lo || row >= hi) return;
    const float temp = a.temp ? a.temp[r] : 1.0f;
    if (row == hi - 1) draft = -1;
    float m = -INFINITY;
    int bad = 0;
#pragma unroll
    for (int j = 0; j < VF_VEC; j++)
#pragma unroll
        for (int n = 0; n < 4; n++) {
            bad |= !(x[j][n] < INFINITY);
            m = fmaxf(m, x[j][n]);
        }
    m = wave_fold(m, [](float p, float q) { return fmaxf(p, q); });
    bad = __any(bad);
    int arg = V;
    double z = 0.0;
    if (!(temp > 0.0f)) {  // the same for the work group, as all conditions here
#pragma unroll
        for (int j = VF_VEC - 1; j >= 0; j--)
#pragma unroll
            for (int n = 3; n >= 0; n--)
                if (x[j][n] == m) arg = s * VF_SLICE + 4 * ((int)threadIdx.x + VF_THREADS * j) + n;
        arg = wave_fold(arg, [](int p, int q) { return min(p, q); });
    } else if (m > -INFINITY && !bad) {
        const double c = 1.4426950408889634 / (double)temp;
        if (draft >= 0 && draft / VF_SLICE == s) {
#pragma unroll
            for (int j = 0; j < VF_VEC; j++)
#pragma unroll
                for (int n = 0; n < 4; n++)
                    if (s * VF_SLICE + 4 * ((int)threadIdx.x + VF_THREADS * j) + n == draft) x[j][n] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < VF_VEC; j++)
#pragma unroll
            for (int n = 0; n < 4; n++) z += weight(x[j][n], c, (double)m);
        z = wave_sum(z);
    }
    if (lane == 0) of_wave[wave] = {z, m, arg, bad, 0};
    __syncthreads();
    if (threadIdx.x) return;
    VfSlice all = of_wave[0];
    for (int w = 1; w < WAVES; w++) {  // equal largest ones: the lowest index
        const VfSlice v = of_wave[w];
        all.bad |= v.bad;
        all.arg = v.m > all.m ? v.arg : v.m == all.m ? min(all.arg, v.arg) : all.arg;
        all.m = fmaxf(all.m, v.m);
    }
    if (temp > 0.0f) {
        const double c = 1.4426950408889634 / (double)temp;
        all.z = 0.0;
        for (int w = 0; w < WAVES; w++) all.z += of_wave[w].z * exp2_f64(((double)of_wave[w].m - (double)all.m) * c);
    }
    out[(int64_t)row * S + s] = all;
}

// Where request r, of rows lo .. hi - 1, ends: a row per wave, the last row always ends it.
// found, ends: one per wave.
template <int WAVES>
__device__ __forceinline__ VfPick vf_decide(const VerifyArgs& a, const VfSlice* part, int r, int lo, int hi,
                                            VfPick* found, int* ends) {
    const int V = a.vocab, S = vf_slices(V), lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, n = hi - lo;
    const float temp = a.temp ? a.temp[r] : 1.0f;
    const bool greedy = !(temp > 0.0f);
    const double c = 1.4426950408889634 / (double)temp;
    for (int i0 = 0;; i0 += WAVES) {
        const int i = i0 + wave, row = lo + min(i, n - 1);
        const VfSlice* const sl = part + (int64_t)row * S;
        const bool last = i >= n - 1;
        const int x = last ? -1 : a.ids[row + 1];
        const bool word = x >= 0 && x < V;
        const float lx = a.logits[(int64_t)row * V + (word ? x : 0)], u = a.u_accept[row];
        const float qx = a.draft ? a.draft[(int64_t)row * V + (word ? x : 0)] : 1.0f;
        const VfSlice none = {0.0, -INFINITY, V, 0, 0}, v0 = lane < S ? sl[lane] : none;
        float m = v0.m;
        int bad = v0.bad, arg = v0.arg;
        for (int k = lane + WAVE; k < S; k += WAVE) {
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
        VfPick e = {0.0, mm, lx, i, -1, -1, -1, !last, 0};
        bool end = true;
        if (bad || mm == -INFINITY) {
            // no distribution
        } else if (greedy) {
            end = last || x != arg;
            e.tok = arg;
        } else {
            double z = v0.z * exp2_f64(((double)v0.m - (double)mm) * c);
            for (int k = lane + WAVE; k < S; k += WAVE) z += sl[k].z * exp2_f64(((double)sl[k].m - (double)mm) * c);
            const double w = word ? weight(lx, c, (double)mm) : 0.0;
            z = wave_sum(z) + w;
            end = !(word && (double)u * (double)qx < w / z);
            e.z = z;
            e.row = row;
            e.x = word ? x : -1;
        }
        __syncthreads();  // the last rows' are read
        if (lane == 0) {
            found[wave] = e;
            ends[wave] = end && i < n;
        }
        __syncthreads();
        int w = 0;
        while (w < WAVES && !ends[w]) w++;
        if (w < WAVES) return found[w];
    }
}

__global__ __launch_bounds__(VF_THREADS) void verify_rest_kernel(VerifyArgs a, const VfSlice* __restrict__ part,
                                                                double* __restrict__ rest, VfPick* __restrict__ pick) {
    constexpr int WAVES = VF_THREADS / WAVE;
    __shared__ VfPick found[WAVES];
    __shared__ int ends[WAVES];
    __shared__ double pd[WAVES];
    const int V = a.vocab, S = vf_slices(V), r = (int)(blockIdx.x / S), s = (int)(blockIdx.x % S);
    int lo, hi;
    if (!vf_rows(a, r, lo, hi)) {
        if (s == 0 && threadIdx.x == 0) pick[r] = {0.0, 0.0f, 0.0f, -1, -1, -1, -1, 0, 0};
        return;
    }
    const VfPick p = vf_decide<WAVES>(a, part, r, lo, hi, found, ends);
    if (s == 0 && threadIdx.x == 0) pick[r] = p;
    if (p.row < 0 || !p.refused) return;
    // what is left: p - q where positive
    const double c = 1.4426950408889634 / (double)(a.temp ? a.temp[r] : 1.0f);
    f4_any_t x[VF_VEC], q[VF_VEC];
    load_slice(a.logits + (int64_t)p.row * V, V, s, -INFINITY, x);
    load_slice(a.draft + (int64_t)p.row * V, V, s, 0.0f, q);
    const double m = (double)p.m, inv = 1.0 / p.z;
    double left = 0.0;
#pragma unroll
    for (int j = 0; j < VF_VEC; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double v = weight(x[j][k], c, m) * inv;
            left += v > (double)q[j][k] ? v - (double)q[j][k] : 0.0;
        }
    left = block_fold<VF_THREADS>(left, pd, [](double u, double v) { return u + v; });
    if (threadIdx.x == 0) rest[(int64_t)r * S + s] = left;
}

// rest, pick: null without draft probabilities
__global__ __launch_bounds__(VP_THREADS) void verify_pick_kernel(VerifyArgs a, const VfSlice* __restrict__ part,
                                                                const double* __restrict__ rest,
                                                                const VfPick* __restrict__ pick) {
    constexpr int WAVES = VP_THREADS / WAVE;
    __shared__ double runs[VP_VEC * WAVES];
    static_assert(VP_VEC * WAVES <= WAVE, "a run per lane");
    __shared__ int pi[WAVES];
    __shared__ VfPick found[WAVES];
    __shared__ int ends[WAVES];
    const int V = a.vocab, S = vf_slices(V), r = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const float temp = a.temp ? a.temp[r] : 1.0f, u_sample = a.u_sample[r];
    int lo, hi;
    VfPick p = {0.0, 0.0f, 0.0f, -1, -1, -1, -1, 0, 0};
    const bool rows = vf_rows(a, r, lo, hi);
    if (pick)
        p = pick[r];
    else if (rows)
        p = vf_decide<WAVES>(a, part, r, lo, hi, found, ends);
    int tok = p.tok;
    if (p.row >= 0) {
        const double c = 1.4426950408889634 / (double)temp, m = (double)p.m, inv = 1.0 / p.z;
        const bool minus = p.refused && rest;  // p - q, else p (a refused draft: without it)
        const VfSlice* const sl = part + (int64_t)p.row * S;
        const double* const rs = rest + (int64_t)r * S;
        const int xs = p.x / VF_SLICE;         // its slice
        const double px = p.x >= 0 ? weight(p.lx, c, m) * inv : 0.0;
        auto without = [&](int k) { return sl[k].z * exp2_f64(((double)sl[k].m - m) * c) * inv; };
        // sums over the slices, in order; every wave for itself
        double left = 0.0;
        for (int k = lane; k < S; k += WAVE) left += minus ? rs[k] : without(k);
        left = wave_sum(left);
        const bool whole = !(left > 0.0);  // nothing is left: from p
        const double thr = (double)u_sample * (whole ? 1.0 : left);
        double before = 0.0;
        int s = -1, s_any = -1;  // the first slice whose running sum exceeds thr; the last one with any weight
        double s_before = 0.0, any_before = 0.0;
        for (int k0 = 0; k0 < S && s < 0; k0 += WAVE) {
            const int k = k0 + lane;
            double v = 0.0;
            if (k < S) v = whole ? without(k) + (p.x >= 0 && k == xs ? px : 0.0) : minus ? rs[k] : without(k);
            const double run = before + wave_scan(v);
            const unsigned long long over = __ballot(v > 0.0 && run > thr), any = __ballot(v > 0.0);
            if (any) {
                const int e = 63 - __builtin_clzll(any);
                s_any = k0 + e;
                any_before = read_lane(run - v, e);
            }
            if (over) {
                const int e = __builtin_ctzll(over);
                s = k0 + e;
                s_before = read_lane(run - v, e);
            }
            before = read_lane(run, WAVE - 1);
        }
        if (s < 0) {  // u rounds to the whole
            s = s_any;
            s_before = any_before;
        }
        // no weight anywhere: rows of no request, whose slices nobody wrote (row starts out of order)
        const bool none = s < 0;
        s = max(s, 0);
        // in the slice: VP_VEC x WAVES runs of 4 x 64 tokens (load_slice's order), their sums, then
        // the lanes of the run that u falls into
        const float* const dr = minus && !whole ? a.draft + (int64_t)p.row * V : nullptr;
        const int gone = whole || minus ? -1 : p.x;  // of a refused draft without probabilities
        f4_any_t x[VP_VEC], q[VP_VEC];
        load_slice(a.logits + (int64_t)p.row * V, V, s, -INFINITY, x);
        if (dr) load_slice(dr, V, s, 0.0f, q);
        double sum[VP_VEC];
        auto left_of = [&](const f4_any_t& lg, const f4_any_t& qs, int j, int k) {
            const double v = weight(lg[k], c, m) * inv;
            if (dr) return v > (double)qs[k] ? v - (double)qs[k] : 0.0;
            return s * VF_SLICE + 4 * (tid + VP_THREADS * j) + k == gone ? 0.0 : v;
        };
#pragma unroll
        for (int j = 0; j < VP_VEC; j++) {
            double u = 0.0;
#pragma unroll
            for (int k = 0; k < 4; k++) u += left_of(x[j], q[j], j, k);
            sum[j] = u;
        }
#pragma unroll
        for (int j = 0; j < VP_VEC; j++) {
            const double u = wave_sum(sum[j]);
            if (lane == 0) runs[j * WAVES + wave] = u;
        }
        __syncthreads();
        const double mine_run = lane < VP_VEC * WAVES ? runs[lane] : 0.0;  // a run per lane
        const double run = wave_scan(mine_run);
        const unsigned long long some = __ballot(mine_run > 0.0);
        const unsigned long long over = __ballot(mine_run > 0.0 && s_before + run > thr);
        // no run: the sums of the slice and of its runs may round apart
        const int at = none ? -1 : over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        const double at_before = s_before + read_lane(run - mine_run, max(at, 0));
        tok = -1;
        if (at >= 0 && at % WAVES == wave) {
            const int j = at / WAVES;
            f4_any_t xj = x[0], qj = q[0];
            double mine = sum[0];
#pragma unroll
            for (int k = 1; k < VP_VEC; k++)
                if (k == j) {
                    xj = x[k];
                    qj = q[k];
                    mine = sum[k];
                }
            double here = at_before + wave_scan(mine) - mine;
            const int i0 = s * VF_SLICE + 4 * (tid + VP_THREADS * j);
            int first = V, any = -1;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const double v = left_of(xj, qj, j, k);
                here += v;
                if (v > 0.0) {
                    any = i0 + k;
                    if (first == V && here > thr) first = i0 + k;
                }
            }
            first = wave_fold(first, [](int u, int v) { return min(u, v); });
            any = wave_fold(any, [](int u, int v) { return max(u, v); });
            tok = first < V ? first : any;
        }
        tok = block_fold<VP_THREADS>(tok, pi, [](int u, int v) { return max(u, v); });
    }
    int* const out = a.tokens + (int64_t)r * a.max_new;
    for (int i = tid; i < a.max_new; i += VP_THREADS)
        out[i] = i < p.accepted ? a.ids[lo + i + 1] : i == p.accepted ? tok : -1;
    if (tid == 0) a.accepted[r] = p.accepted;
}

static size_t al16(size_t n) { return (n + 15) / 16 * 16; }

size_t verify_ws_bytes(int n_req, int n_rows, int vocab) {
    const size_t S = vf_slices(vocab);
    return al16(n_rows * S * sizeof(VfSlice)) + al16(n_req * S * sizeof(double)) + al16(n_req * sizeof(VfPick));
}

hipError_t launch_verify_drafts(const VerifyArgs& a, hipStream_t s) {
    const size_t S = vf_slices(a.vocab);
    uint8_t* const ws = static_cast<uint8_t*>(a.ws);
    VfSlice* const part = reinterpret_cast<VfSlice*>(ws);
    double* rest = nullptr;
    VfPick* pick = nullptr;
    hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)(a.n_rows * S)), dim3(VF_THREADS), 0, s, a, part);
    if (a.draft) {
        rest = reinterpret_cast<double*>(ws + al16(a.n_rows * S * sizeof(VfSlice)));
        pick = reinterpret_cast<VfPick*>(reinterpret_cast<uint8_t*>(rest) + al16(a.n_req * S * sizeof(double)));
        hipLaunchKernelGGL(verify_rest_kernel, dim3((unsigned)(a.n_req * S)), dim3(VF_THREADS), 0, s, a, part, rest,
                           pick);
    }
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)a.n_req), dim3(VP_THREADS), 0, s, a, part, rest, pick);
    return hipGetLastError();
}

}  // namespace hy
