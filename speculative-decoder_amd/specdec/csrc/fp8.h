// The 8-bit row format that the projections read (quant.hip writes it,
// linear_fp8.hip multiplies it).
//
// A row of K values is cut into groups of 128; a group's scale is the least
// power of two s = 2^e, e >= -126, with max |y| <= 448 s over its finite
// values (448 is e4m3's largest), and its codes are y / s rounded once, to
// nearest even, to e4m3; infinities and NaN become NaN codes.  With a power
// of two y / s and s * code are exact, so the one error is e4m3's rounding,
// and the matrix unit takes the scale's exponent byte (e8m0: e + 127) with
// the operand, so scaling a product costs no instruction.
#pragma once

#include "common.h"

namespace specdec {

constexpr int kFp8Group = 128;

// codes of a row: whole groups; scales of a row: a multiple of four, so that
// the scales of four groups can be read as one word
inline __host__ __device__ int64_t fp8_code_cols(int64_t k) { return (k + kFp8Group - 1) / kFp8Group * kFp8Group; }
inline __host__ __device__ int64_t fp8_scale_cols(int64_t k) { return (k + 4 * kFp8Group - 1) / (4 * kFp8Group) * 4; }

constexpr unsigned kFp8ScaleOne = 127;  // the padding's scale

// The scale byte of a group whose largest finite |y| has the bits `amax`:
// with |y| = 1.f 2^E and 448 = 1.75 2^8, the least e is E - 8, or E - 7 where
// 1.f > 1.75.
__device__ __forceinline__ unsigned fp8_scale_byte(unsigned amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (unsigned)max(e, 1);
}

// 1 / scale, exactly
__device__ __forceinline__ float fp8_inverse(unsigned scale_byte) {
  return __uint_as_float((254u - scale_byte) << 23);
}

// four codes of values already divided by the scale (the conversion rounds to
// nearest even and turns infinities into NaN codes; finite values are within
// 448 here, so it never saturates)
__device__ __forceinline__ unsigned fp8_pack4(float a, float b, float c, float d) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
  return (unsigned)p;
}

// The largest of v >= 0 over each row of 16 lanes, in every lane of the row.
__device__ __forceinline__ float row16_max(float v) {
  v = dpp_max_step<0xB1>(v);
  v = dpp_max_step<0x4E>(v);
  v = dpp_max_step<0x141>(v);
  return dpp_max_step<0x140>(v);
}

}  // namespace specdec
