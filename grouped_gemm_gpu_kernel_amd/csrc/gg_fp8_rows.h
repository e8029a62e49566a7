// gg_fp8_rows.h -- 8-bit rows: float8 e4m3 numbers with a float scale for each
// block of 128 columns, made 8 columns a lane.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gg {

// 16 and 8 bytes that stand anywhere: the memory's instructions take any address, at the price of the lines that they touch.
typedef uint32_t Any16 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t Any8 __attribute__((ext_vector_type(2), aligned(1)));

constexpr int kFp8Block = 128;
constexpr float kFp8Largest = 448.0f;
constexpr float kFp8SmallestScale = 1.17549435e-38f;  // 2^-126: above it 1 / scale is finite

// Maximum over the 16 lanes of a row (DPP row rotations), of bits as unsigned numbers.
__device__ __forceinline__ uint32_t row_max16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
  return v;
}

// |v| as bits: compared as unsigned numbers these order like the magnitudes, with NaN above infinity, so that a
// maximum keeps a NaN (fmaxf drops it).
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

__device__ __forceinline__ float fp8_scale(uint32_t largest_bits) {
  const float s = __builtin_bit_cast(float, largest_bits) / kFp8Largest;
  return s < kFp8SmallestScale ? kFp8SmallestScale : s;  // a NaN stays
}

// What a block's values are divided by, a 448th of the block's largest magnitude, here as the scale and what its rounding left
// out: the quotient by an about equal reciprocal and one correction then rounds to the number of the exact quotient, but for
// ties closer than its last place.  (Against 64 bits 1500 of the 134 million numbers of a norm of 16384 rows of 8192 were the
// other neighbour with the rounded scale, none to two so.)  The smallest scale stands for itself; an infinite one leaves 0 of
// finite values and NaN of infinite ones.
struct Fp8Divisor {
  float scale, rest, inverse;
  __device__ __forceinline__ Fp8Divisor(float s, float largest)
      : scale(s == __builtin_inff() ? 0.0f : s), rest(0.0f), inverse(__builtin_amdgcn_rcpf(s)) {
    const float left = fmaf(-kFp8Largest, s, largest);
    if (fabsf(left) <= s * (kFp8Largest * 0x1p-22f)) rest = left * (1.0f / kFp8Largest);
  }
  __device__ __forceinline__ float operator()(float y) const {
    const float t = y * inverse;
    return fmaf(fmaf(-t, rest, fmaf(-t, scale, y)), inverse, t);
  }
};

// Four numbers: y / scale to the nearest of the type (steps of 2^-4).  |y / scale| is 448 and a rounding at most, which
// rounds to 448.
__device__ __forceinline__ uint32_t fp8_numbers(float a, float b, float c, float d, const Fp8Divisor& by) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(by(a), by(b), 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(by(c), by(d), v, true);
  return (uint32_t)v;
}

}  // namespace gg
