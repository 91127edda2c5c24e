// gr_e4m3.h -- rows of 8-bit numbers with a power-of-two scale: bytes are e4m3 (sign, 4
// bits of exponent with bias 7, 3 of mantissa; 448 at most; 0x7f NaN), a row's scale is a
// byte b for 2^(b - 127), 255 for NaN (E8M0).
#pragma once
#include "gr_common.h"

template <bool Q8> struct gr_bytes { typedef unsigned short type; };
template <> struct gr_bytes<true> { typedef unsigned char type; };

// Two numbers of a word times a scale, as T: exact where T can hold them
// (v_cvt_scalef32_pk_{bf16,f16}_fp8, which takes the exponent of `scale`: checked for every
// byte and scale).
template <class T, bool HIGH>
__device__ __forceinline__ unsigned gr_from_e4m3(unsigned w, float scale) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HIGH));
  else
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}

// A scale byte as the float whose exponent the conversion takes.
__device__ __forceinline__ float gr_e8m0(unsigned sb) { return __builtin_bit_cast(float, sb << 23); }
