// gr_e4m3.h -- rows of 8-bit numbers with a power-of-two scale: bytes are e4m3 (sign, 4
// bits of exponent with bias 7, 3 of mantissa; 448 at most; 0x7f NaN), a row's scale is a
// byte b for 2^(b - 127), 255 for NaN (E8M0).
#pragma once
#include "gr_common.h"

template <bool Q8> struct gr_bytes { typedef unsigned short type; };
template <> struct gr_bytes<true> { typedef unsigned char type; };

// Two numbers of a word times a scale, as T: exact where T can hold them, the nearest
// number (to even) below its normal range (v_cvt_scalef32_pk_{bf16,f16}_fp8, which takes the
// exponent of `scale`: checked for every byte and scale).
template <class T, bool HIGH>
__device__ __forceinline__ unsigned gr_from_e4m3(unsigned w, float scale) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HIGH));
  else
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}

// Where lane l's 16 bytes of a cached row go in LDS as T: a row of D / 16 pieces is
// that many lanes wide, and a write of 16 bytes takes every second chunk of a row, so
// that 8 lanes side by side (128 bytes, what LDS takes at a time) are two half rows, of rows
// whose swizzles differ in the chunks' lowest bit: those that differ in bit 0 for keys
// (gr_paged_swz) and bit 2 for values (gr_swz_v8). (All 8 of one row: every write in two.)
template <int D>
__device__ __forceinline__ int gr_piece8(int lane) { return D == 128 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3; }
template <int D>
__device__ __forceinline__ int gr_key8(int lane) { return D == 128 ? ((lane >> 2) & 1) | ((lane >> 3) & 6) : lane >> 2; }
template <int D>
__device__ __forceinline__ int gr_value8(int lane) {
  return D == 128 ? (lane & 4) | ((lane >> 4) & 3) : (lane & 4) | ((lane >> 3) & 3) | ((lane >> 2) & 8);
}

// A scale byte, and byte `shift` / 8 of a word of four, as the float whose exponent the
// conversion takes. (Kept over a loop as loaded bytes, scales were masked to 8 bits in the
// iteration that asked for them, which waited for its loads: words need no mask.)
__device__ __forceinline__ float gr_e8m0_of(unsigned w, int shift) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ubfe(w, shift, 8) << 23);
}
__device__ __forceinline__ float gr_e8m0(unsigned sb) { return __builtin_bit_cast(float, sb << 23); }
