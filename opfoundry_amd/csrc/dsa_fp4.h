// dsa_fp4.h - the codes of DSA_KV_MXFP4 rows (include/dsa_mla.h) on the device.
// Included inside a kernel file's namespace, after dsa_lds.h.
#pragma once

constexpr int FP4_ROW = DSA_MLA_FP4_ROW_BYTES;       // 256 code bytes, 16 scale bytes, 64 bf16 RoPE values
constexpr int FP4_SCALE_OFF = 256, FP4_ROPE_OFF = 272;

// 8 e2m1 codes (a dword, the first value in the low half of the low byte) times 2^(e - 127) -> 8 bf16.
// Exact below 2^128: a code has two significant bits, the scale is a power of two and bf16 has fp32's exponents (and
// its values below the normal range, which byte 0 reaches).  From 2^128 on (codes 4 and 6 under byte 253, from 2 on
// under 254) it is infinity.  The instruction takes the scale's exponent field,
// and gives NaN where that is 255, whatever the code.  All 256 x 16 pairs were compared.
__device__ __forceinline__ u32x4 fp4_to_bf16(unsigned c, unsigned e) {
    const float s = __uint_as_float(e << 23);
    return u32x4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                 __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

// Two of them: values 2 SEL and 2 SEL + 1; `s` is the scale.
template <int SEL>
__device__ __forceinline__ unsigned fp4_pair(unsigned c, float s) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, SEL));
}

// e of the least power of two 2^e >= amax / 6 = amax / (1.5 * 2^2), at least -125, so that half of it, the
// least value a code stands for, is a normal bf16; 0 for 0.
__device__ __forceinline__ int fp4_exponent(float amax) {
    const unsigned bits = __float_as_uint(amax);
    if (bits == 0) return 0;
    return max(-125, (int)(bits >> 23) - 127 - 2 + ((bits & 0x7FFFFFu) > 0x400000u ? 1 : 0));
}
