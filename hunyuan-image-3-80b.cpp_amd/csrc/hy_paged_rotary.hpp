// hy_paged_rotary.hpp -- rotary embedding and per-head RMSNorm of the cache writes, HD / 4 lanes per head
// with 4 dims each.
#pragma once
#include "hy_paged_split.hpp"

namespace hy {

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, false));
}

// Sine and cosine of position times freq (turns per position).  An angle is kept as a fraction of a
// turn in 64 bits, position times turns per position minus its whole part, so a far position costs no
// accuracy; sine and cosine are f32, of its f32 part, and turned by the rest.
__device__ __forceinline__ void rope_angle(int pos, double freq, float& sn, float& cs) {
    double turn = (double)pos * freq;
    turn = 2.0 * (turn - rint(turn));  // in half turns
    const float half = (float)turn, rest = (float)(turn - (double)half) * 3.14159265f;
    float s0, c0;
    sincospif(half, &s0, &c0);
    sn = fmaf(rest, c0, s0);
    cs = fmaf(-rest, s0, c0);
}

// 1 / sqrt(mean y^2 + eps) of a head, in all its lanes
template <int HD>
__device__ __forceinline__ float head_rms(v4f_t y, float eps) {
    float ss = (y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]);
    ss += dpp_f<0x128>(ss);  // rotations by 8 .. 1 in 16 lanes
    ss += dpp_f<0x124>(ss);
    ss += dpp_f<0x122>(ss);
    ss += dpp_f<0x121>(ss);
    if constexpr (HD == 128) ss = fadd_row(ss);
    // 1 / sqrt rounded once: the 64-bit estimate (2^-24) and a step of Newton's, fewer operations than
    // an f32 root and quotient
    const double ms = fma((double)ss, 1.0 / HD, (double)eps), e = __builtin_amdgcn_rsq(ms);
    return ms > 0.0 && ms < (double)INFINITY ? (float)fma(0.5 * e, fma(-ms * e, e, 1.0), e) : (float)e;
}

}  // namespace hy
