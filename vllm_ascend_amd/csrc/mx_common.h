// Microscaled 4-bit values (MXFP4): 32 values along a row share a power of two, held as one byte (exponent + 127), and have
// four bits each: sign, two bits of exponent, one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6), the first value of a byte in its
// low half.
//
// Quantisation of a block with the largest magnitude a: exponent e = floor(log2 a) - 2, at least -127, so that a / 2^e lies in
// [4, 8); codes are the values over 2^e rounded to the nearest that four bits hold, ties to the even code, magnitudes above 6
// to 6.  A block of zeros has e = -127; one with an infinity or NaN has the scale byte 255, which stands for NaN, and codes 0.
#pragma once

#include "moe355_common.h"

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

namespace moe355 {

// largest: the bits of the largest magnitude (as integers: magnitudes of binary32 numbers are ordered like their bits, and
// infinities and NaN come last).  The exponent field is floor(log2) + 127 for normal numbers and 0 for subnormal ones, whose
// scale is the smallest either way.
struct MxScale {
    uint32_t byte;
    float inverse;  // 2^-e: a normal number for every byte below 253, and no finite block has a larger one
    bool finite;
};
__device__ __forceinline__ MxScale mx_scale(uint32_t largest)
{
    const uint32_t field = largest >> 23;
    MxScale s;
    s.finite = field != 255;
    s.byte = field > 2 ? field - 2 : 0;
    s.inverse = __uint_as_float((254 - s.byte) << 23);
    if (!s.finite) s.byte = 255;
    return s;
}

// Eight values (already over 2^e) to codes.  v_cvt_scalef32_pk_fp4_f32 with a scale of 1 rounds to nearest even and saturates.
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8])
{
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], 1.0f, 3);
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// A block is four lanes with eight values each: its largest magnitude in all four of them.
__device__ __forceinline__ uint32_t mx_largest_of_quad(const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max_u32(m, __float_as_uint(v[j]) & 0x7fffffffu);
    m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true));   // quad_perm 1 0 3 2
    return max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}

__device__ __forceinline__ uint32_t mx_quantise8(const float (&v)[8], const MxScale& s)
{
    float scaled[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) scaled[j] = v[j] * s.inverse;
    return s.finite ? mx_codes8(scaled) : 0;
}

template <int DT>
__device__ __forceinline__ void load8(const void* p, float (&v)[8])
{
    if constexpr (DT == MOE355_DT_F32) {
        const v4f a = ((const v4f*)p)[0], b = ((const v4f*)p)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    } else {
        const v8u16 a = *(const v8u16*)p;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = half_to_f32<DT>(a[j]);
    }
}

// Eight values a thread, piece i of `pieces`, a block of 32 by four neighbouring lanes.  (Whole blocks: a multiple of four pieces.)
template <int DT>
__device__ __forceinline__ void mx_quant_piece(const char* x, int64_t i, int64_t pieces, uint32_t* codes, uint8_t* scale)
{
    if (i >= pieces) return;
    float v[8];
    load8<DT>(x + i * 8 * (DT == MOE355_DT_F32 ? 4 : 2), v);
    const MxScale s = mx_scale(mx_largest_of_quad(v));
    codes[i] = mx_quantise8(v, s);
    if ((threadIdx.x & 3) == 0) scale[i >> 2] = (uint8_t)s.byte;
}

}  // namespace moe355
