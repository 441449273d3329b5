// SPDX-License-Identifier: Apache-2.0
// E4M3 codes of fp32 values: the conversions shared by the stores (fp8_kv.hip,
// rotary_store.hip).
#pragma once

#include "kvq_common.h"

namespace kvq {

constexpr float kE4M3Max = 448.0f;
constexpr float kScaleFloor = 1.0e-6f;  // the fp32 rounding of the literal 1e-6

// Four codes (element i in byte i), round to nearest even.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}

// The four codes of a word as fp32 (exact).
__device__ __forceinline__ void e4m3x4_f32(uint32_t w, float (&x)[4]) {
  typedef float f2v __attribute__((ext_vector_type(2)));
  const f2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f2v hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  x[0] = lo.x;
  x[1] = lo.y;
  x[2] = hi.x;
  x[3] = hi.y;
}

// The sign bits of four fp32 values at bit 7 of bytes 0..3.
__device__ __forceinline__ uint32_t sign_bytes(float a, float b, float c, float d) {
  // v_perm: bytes {a.b3, b.b3, 0, 0} and {0, 0, c.b3, d.b3}
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0703u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x07030c0cu);
  return (lo | hi) & 0x80808080u;
}

// Codes of e4m3fn(clamp(x / scale, -448, 448)), four elements a word.
//
// The IEEE quotient is needed only where it decides a code.  With
// y = RN(1/scale), t = RN(|x| * y) is within (2^-23 + 2^-48) |q| of the exact
// quotient q = |x| / scale, and RN(q) within 2^-24 |q| of q, so RN(q) lies
// within 3.03 * 2^-24 |q| of t: fewer than 7 steps of the fp32 bit pattern,
// also when a binade boundary between them halves the step.  Rounding to E4M3
// (like the clamp) is monotone, so when t - 8 steps and t + 8 steps give the
// same code as t, every value between them does, RN(q) included.  Otherwise
// (a code boundary within 8 steps: about 1 element in 60,000) the word is
// recomputed from the IEEE quotient.  The sign is applied to the magnitude's
// code, as round-to-nearest and the clamp are symmetric (-0 gives 0x80).
template <int VEC>
__device__ __forceinline__ void quantize_codes(const float (&x)[VEC], float scale,
                                               uint32_t (&codes)[VEC / 4]) {
  const float y = __fdiv_rn(1.0f, scale);
#pragma unroll
  for (int w = 0; w < VEC / 4; ++w) {
    float t[4], lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = fminf(fabsf(x[4 * w + i]) * y, kE4M3Max);
      const uint32_t b = __float_as_uint(t[i]);
      lo[i] = __uint_as_float(__builtin_elementwise_sub_sat(b, 8u));
      hi[i] = fminf(__uint_as_float(b + 8u), kE4M3Max);
    }
    uint32_t c = e4m3x4(t[0], t[1], t[2], t[3]);
    const uint32_t cl = e4m3x4(lo[0], lo[1], lo[2], lo[3]);
    const uint32_t ch = e4m3x4(hi[0], hi[1], hi[2], hi[3]);
    if (cl != c || ch != c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = fminf(__fdiv_rn(fabsf(x[4 * w + i]), scale), kE4M3Max);
      c = e4m3x4(t[0], t[1], t[2], t[3]);
    }
    codes[w] = c | sign_bytes(x[4 * w], x[4 * w + 1], x[4 * w + 2], x[4 * w + 3]);
  }
}

}  // namespace kvq
