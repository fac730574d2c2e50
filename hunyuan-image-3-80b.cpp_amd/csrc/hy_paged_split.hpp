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
// pieces of two floats; the remainders x - hi are rounded as they are formed (v_fma_mixlo_f16 /
// mixhi: hi's half times -1 plus x, one rounding)
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pk_f16(a, b);
    asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(hi), "v"(a));
    asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(hi), "v"(b));
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
