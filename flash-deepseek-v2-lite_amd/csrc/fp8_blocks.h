// Shared by the 8-bit kernels with block scales: the rounding of a block to e4m3.
//
// With a the largest |v| of a block of up to 128 columns (at least kLeast), its scale is a / 448 and its
// codes are the e4m3 values nearest to 448 v / a, ties to even.  The quotient is not taken by the rounded
// scale: values of bf16 often lie exactly half way between two codes, and there the scale's rounding
// would decide.
#pragma once

#include "common.h"

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;
// blocks with nothing larger are rounded as if this were their largest: reciprocals stay in range
constexpr uint32_t kLeastBits = (127u - 100u) << 23;  // 2^-100

// What rounds a block: am = a / 512 (exact) and its reciprocal.  448 v / a = (7/8 v) / am: 7/8 v is exact for
// bf16, v_rcp_f32 is off by an ulp, and one residual makes the quotient the nearest float, so that a v that
// lies on a code or half way between two gives exactly that.  A block with an infinity or a NaN has
// am = inf or NaN and every quotient is NaN.
struct Fp8Rounding {
  float am, ri;
  __device__ __forceinline__ explicit Fp8Rounding(uint32_t max_bits) {
    am = __uint_as_float(max_bits) * (1.f / 512.f);
    ri = __builtin_amdgcn_rcpf(am);
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float t = 0.875f * v, q = t * ri;
    return __builtin_fmaf(__builtin_fmaf(-q, am, t), ri, q);
  }
};

// a / 448, rounded once (NaN for a = inf: the block's values are NaN too)
__device__ __forceinline__ float fp8_scale(uint32_t max_bits) {
  constexpr float c = 1.f / kFp8Max;
  const float a = __uint_as_float(max_bits), q = a * c;
  return __builtin_fmaf(__builtin_fmaf(-q, kFp8Max, a), c, q);
}

// bits of |v|: as unsigned numbers they are ordered as the values are, NaN above infinity
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// four codes of quotients of at most 448 (1 + 2^-23): v_cvt_pk_fp8_f32 rounds to nearest even
__device__ __forceinline__ uint32_t fp8x4(float a, float b, float c, float d) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true));
}

// largest of a 16-lane row, in all its lanes (DPP: quad_perm xor 1 and 2, half mirror, mirror)
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, false)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, false)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, false)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xF, 0xF, false)));
  return v;
}
