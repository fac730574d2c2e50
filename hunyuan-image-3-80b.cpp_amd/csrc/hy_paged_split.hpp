// hy_paged_split.hpp -- f32 values as two f16 pieces for the matrix cores, shared by the paged
// attention's kernels: x = hi + lo, each rounded to nearest, 2^-24 of x left out as long as the
// pieces are normal numbers (which the callers' powers of two see to).
#pragma once
#include "hy_lds.hpp"
#include "hy_split.hpp"

namespace hy {

typedef _Float16 v8h16_t __attribute__((ext_vector_type(8)));
typedef _Float16 v2h16_t __attribute__((ext_vector_type(2)));

// f(v, the same lane's of the other 32, or of the other 16 of its 32): vector operations, where
// a shuffle takes the way through LDS
template <class F>
__device__ __forceinline__ uint32_t with_half(uint32_t v, F f) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(r[0], r[1]);
}
template <class F>
__device__ __forceinline__ uint32_t with_row(uint32_t v, F f) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return f(r[0], r[1]);
}
__device__ __forceinline__ float fmax_half(float v) {
    return __uint_as_float(with_half(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ float fadd_half(float v) {
    return __uint_as_float(with_half(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
__device__ __forceinline__ float fmax_row(float v) {
    return __uint_as_float(with_row(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ float fadd_row(float v) {
    return __uint_as_float(with_row(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

// two floats, packed
__device__ __forceinline__ uint32_t pk_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f_t){a, b}, v2h16_t));
}
// Pieces of two floats; the remainders x - hi are rounded as they are formed (v_fma_mixlo_f16 / mixhi: hi's
// half times -1 plus x, one rounding).  The compiler has to write those itself: a matrix instruction may read
// a register two wait states after a vector instruction wrote it, and it sees to that for its own
// instructions, not for those of inline asm (whose last half was read before it was written).
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const v2h16_t h = __builtin_convertvector((v2f_t){a, b}, v2h16_t);
    hi = __builtin_bit_cast(uint32_t, h);
    float minus = -1.0f;
    asm("" : "+s"(minus));  // or the product becomes a subtraction, which has no such form
    lo = __builtin_bit_cast(uint32_t,
                            (v2h16_t){(_Float16)fmaf((float)h[0], minus, a), (_Float16)fmaf((float)h[1], minus, b)});
}

// 8-bit codes as f16, exactly: with its sign flipped and 0x64 above it a byte is 1024 + 128 + code.
// four codes of a dword, in their order
__device__ __forceinline__ uint32_t f16_less_1152(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h16_t, w) + (v2h16_t){(_Float16)-1152, (_Float16)-1152});
}
__device__ __forceinline__ void i8_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    lo = f16_less_1152(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
    hi = f16_less_1152(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
}
// byte d of a and of b
__device__ __forceinline__ uint32_t i8_pair(uint32_t a, uint32_t b, int d) {
    return f16_less_1152(__builtin_amdgcn_perm(b, a, 0x0c040c00u + 0x00010001u * d) ^ 0x64806480u);
}
// A scale of V: 2^ex mant, ex in -60 .. 34, and 2^-ex; mant in [1, 2) inside that range, NaN for an
// infinity or NaN.
struct I8Scale {
    float ex, inv, mant;
};
__device__ __forceinline__ I8Scale i8_scale(float d) {
    const int e = min(max((int)((__float_as_uint(d) >> 23) & 255) - 127, -60), 34);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    return {(float)e, inv, fmaf(d, 0.0f, d) * inv};
}

// the operand kinds of a cache type
template <class E>
struct PaType;
template <>
struct PaType<_Float16> {
    static constexpr int PIECES = 2;
    static __device__ __forceinline__ v4f_t mfma(v4i_t a, v4i_t b, v4f_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h16_t, a), __builtin_bit_cast(v8h16_t, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ v16f_t mfma(v4i_t a, v4i_t b, v16f_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h16_t, a), __builtin_bit_cast(v8h16_t, b), c,
                                                      0, 0, 0);
    }
    // two floats -> their pieces, packed
    static __device__ __forceinline__ void split(float a, float b, uint32_t (&p)[2]) {
        split_f16(a, b, p[0], p[1]);
    }
    static __device__ __forceinline__ bool odd(uint32_t w) {  // an infinity or NaN among the two
        return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
    }
};
template <>
struct PaType<__bf16> {
    static constexpr int PIECES = 3;
    static __device__ __forceinline__ v4f_t mfma(v4i_t a, v4i_t b, v4f_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_t, a), __builtin_bit_cast(v8bf_t, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ v16f_t mfma(v4i_t a, v4i_t b, v16f_t c) { return mfma_bf16(a, b, c); }
    static __device__ __forceinline__ void split(float a, float b, uint32_t (&p)[3]) {
        uint32_t lost = 0;
        const Split2 s = split2(a, b, lost);
#pragma unroll
        for (int i = 0; i < 3; i++) p[i] = s.p[i];
    }
    static __device__ __forceinline__ bool odd(uint32_t w) {
        return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
    }
};
template <>
struct PaType<float> {
    static constexpr int PIECES = 1;
    static __device__ __forceinline__ bool odd(uint32_t w) { return (w & 0x7F800000u) == 0x7F800000u; }
};

}  // namespace hy
