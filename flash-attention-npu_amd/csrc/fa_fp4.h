// fa_fp4.h -- device code that the kernels over the 4-bit cache share: codes e2m1 (two
// to a byte, the even channel low) under a scale 2^(b - 127) for 32 channels. The
// hardware's conversions take the scale along, so a value comes out in one step, rounded to the
// nearest of the type: bf16 holds every one (two bits of significand), b = 255 gives NaN.
#pragma once
#include "fa_quant.h"

namespace fa {

constexpr int kGroup = 32;  // channels of a scale

// the scale that byte b stands for, as the conversions take it: its exponent field is b
__device__ __forceinline__ float fp4_scale(uint32_t b) { return __builtin_bit_cast(float, b << 23); }

// Eight codes (the nibbles of w, lowest first) as 16-bit values of DT
template <int DT>
__device__ __forceinline__ u32x4 fp4_widen8(uint32_t w, float s) {
    u32x4 o;
    if constexpr (DT == DT_FP16) {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3));
    } else {
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3));
    }
    return o;
}

}  // namespace fa
