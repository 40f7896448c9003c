// e4m3.h — numbers of 8 bits (one sign, four exponent, three mantissa bits) with a power of two that
// a block of them shares: value = code * 2^(power - 127), power 255 is NaN.  gfx950 converts
// code times power in one instruction, two codes at a time; it takes the power from the exponent
// bits of an FP32 number, 0 as 2^-127 and 255 as NaN too.
#ifndef CF_E4M3_H_
#define CF_E4M3_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cdna4.h"

namespace cdna4 {

typedef float f2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((__vector_size__(8))) int lds_i2_t;

// The power as the conversions take it.
__device__ __forceinline__ float power_bits(int power) { return __uint_as_float((uint32_t)power << 23); }

// Codes 0 and 1 (HI: 2 and 3) of a word.
template <bool HI> __device__ __forceinline__ f2_t codes_f32(uint32_t w, float power) {
    return __builtin_bit_cast(f2_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8((int)w, power, HI));
}
template <bool HI> __device__ __forceinline__ h2_t codes_f16(uint32_t w, float power) {
    return __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, power, HI));
}
template <bool HI> __device__ __forceinline__ b2_t codes_bf16(uint32_t w, float power) {
    return __builtin_bit_cast(b2_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, power, HI));
}
// Two values of at most 448 in size to the nearest codes, ties to even, into the low (HI: high) half of w.
template <bool HI> __device__ __forceinline__ uint32_t codes_of(uint32_t w, float a, float b) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)w, HI);
}

// The same as the type that the matrix cores take, 16 bits wide: B, with eight of them (codes of two
// words, each with its power) as one operand.
template <typename B> struct Codes;
template <> struct Codes<_Float16> {
    typedef h8_t eight_t;
    static __device__ __forceinline__ eight_t of(uint32_t lo, float plo, uint32_t hi, float phi) {
        const h2_t a = codes_f16<false>(lo, plo), b = codes_f16<true>(lo, plo), c = codes_f16<false>(hi, phi), d = codes_f16<true>(hi, phi);
        return eight_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    static __device__ __forceinline__ f4_t mfma(eight_t a, eight_t b, f4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Codes<__bf16> {
    typedef b8_t eight_t;
    static __device__ __forceinline__ eight_t of(uint32_t lo, float plo, uint32_t hi, float phi) {
        const b2_t a = codes_bf16<false>(lo, plo), b = codes_bf16<true>(lo, plo), c = codes_bf16<false>(hi, phi), d = codes_bf16<true>(hi, phi);
        return eight_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    static __device__ __forceinline__ f4_t mfma(eight_t a, eight_t b, f4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// ds_read_b64_tr_b8: in each 16-lane group, lane i receives byte i % 8 of the 8-byte chunks that
// lanes i / 8, 2 + i / 8, .., 14 + i / 8 address.  With lane j addressing X[row j / 2][8 (j % 2)],
// lane i gets column i of the eight rows.
__device__ __forceinline__ lds_i2_t ds_read_tr8(const uint8_t* p) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((CF_LDS lds_i2_t*)p);
}

// The nearest codes of two values over the power, ties to even, into half HI of w: what is over 464 in
// size, infinite or NaN becomes NaN.  One instruction, of a quarter of the usual rate.
typedef short s2_t __attribute__((ext_vector_type(2)));
template <bool HI> __device__ __forceinline__ s2_t codes_over(s2_t w, h2_t x, float power) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, x, power, HI);
}
template <bool HI> __device__ __forceinline__ s2_t codes_over(s2_t w, f2_t x, float power) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[0], x[1], power, HI);
}

// The least power whose 448 folds are not below x >= 0 (448 = 1.75 * 2^8); x = 0 and what is too small
// for any power: 0.
__device__ __forceinline__ int power_for(float x) {
    const uint32_t bits = __float_as_uint(x);
    return max((int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}

}  // namespace cdna4

#endif  // CF_E4M3_H_
