// SPDX-License-Identifier: Apache-2.0
// Shared by the attention over pages of 8-bit codes with a scale for each block of `group`
// positions and kv head (block8*.hip).  Requests, what a row sees and partial results are
// those of the windowed attention (fp8_window.h); here the cache's scales are [pages,
// block_size / group, kv heads], and its codes E4M3 or INT8.
#pragma once

#include "fp8_window.h"

namespace kvq {

struct B8Cache : WinCache {
  FastDiv group;
  int int8;
  // (slot of position p, its scale's place for kv head 0)
  struct At {
    int64_t slot, scale;
  };
  __device__ __forceinline__ At at(int t, int p) const {
    const uint32_t i = bs.div(static_cast<uint32_t>(p));
    const uint32_t off = static_cast<uint32_t>(p) - i * bs.d;
    const int64_t pg = page(t, static_cast<int>(i));
    return At{pg * bs.d + off, (pg * (bs.d / group.d) + group.div(off)) * kvh};
  }
};

// A call: `win.cache` is `cache`'s part of it.
struct B8Call {
  WinCall win;
  B8Cache cache;
};

// INT8 codes as a pair of fp16, times 2^-9: with u = code + 128 as the fp16 subnormal
// u 2^-24, u 2^-24 * 2^15 - 2^-2 = code 2^-9, exact.  `x`: four codes, sign bits flipped.
constexpr float kInt8Unit = 0x1p-9f;
template <bool HI>
__device__ __forceinline__ uint32_t int8_pair(uint32_t x) {
  const w_h2 u = __builtin_bit_cast(w_h2, __builtin_amdgcn_perm(0u, x, HI ? 0x0c030c02u : 0x0c010c00u));
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_fma(u, w_h2{32768.0f16, 32768.0f16},
                                                      w_h2{-0.25f16, -0.25f16}));
}
// Eight codes as an operand: T's E4M3 pairs, or fp16 of INT8.
template <typename T, bool INT8>
__device__ __forceinline__ w_u4 b8_op8(uint32_t w0, uint32_t w1) {
  if constexpr (INT8) {
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    return w_u4{int8_pair<false>(w0), int8_pair<true>(w0), int8_pair<false>(w1),
                int8_pair<true>(w1)};
  } else {
    return code_op8<T>(w0, w1);
  }
}

// A query's eight elements in the type of the keys' operand: fp16 for INT8 codes, whose
// bf16 queries are scaled by a power of two for each row that brings the largest to
// [2^14, 2^15): exact down to 2^-31 of it (fp16 holds 8 bits down to 2^-17).
__device__ __forceinline__ uint32_t pair_bits_max(uint32_t m, uint32_t x) {
  const uint32_t lo = (x << 16) & 0x7fffffffu, hi = x & 0x7fff0000u;
  return max(m, max(lo, hi));  // fp32 bits of |bf16|
}
// 2^e with e = 14 - exponent of the row's largest, 1 for a row of nothing or not finite.
__device__ __forceinline__ float query_raise(uint32_t top) {
  const int e = static_cast<int>(top >> 23);
  if (e == 0 || e == 255) return 1.0f;
  const int r = 127 + 14 - (e - 127);
  return __uint_as_float(static_cast<uint32_t>(min(r, 253)) << 23);
}
__device__ __forceinline__ uint32_t raised_pair(uint32_t x, float raise) {
  return pack_pair(__uint_as_float(x << 16) * raise, __uint_as_float(x & 0xffff0000u) * raise, f16{});
}

// A value scale as the matrix kernels take it: log2 of its size for the softmax, its sign
// and what it leaves of the codes apart.  Sizes under 2^-90 count as 0; one that is not
// finite makes its rows NaN.
struct B8Value {
  float lv, iv, sign;
};
__device__ __forceinline__ B8Value b8_value(float vs) {
  const float size = fabsf(vs);
  if (size >= 0x1p-90f && size < INFINITY)
    return B8Value{__builtin_amdgcn_logf(size), __builtin_amdgcn_rcpf(size), vs < 0.0f ? -1.0f : 1.0f};
  if (size < INFINITY) return B8Value{-90.0f, 0x1p90f, 0.0f};
  return B8Value{0.0f, 1.0f, NAN};
}

// block8_decode.hip: requests of few rows; block8_chunk.hip: the others, both where
// b8_matrix applies.  _bytes: their partial results.
bool b8_decode_takes(const B8Call& call, int64_t b);
bool b8_tiles_only(const B8Call& call);
int64_t b8_decode_bytes(const B8Call& call, int* rc);
int b8_decode(const B8Call& call, void* workspace);
bool b8_chunk_takes(const B8Call& call, int64_t b);
int64_t b8_chunk_bytes(const B8Call& call, int* rc);
int b8_chunk(const B8Call& call, void* workspace);

// As win_matrix_geometry, and scales of whole groups of 16 positions.
inline bool b8_matrix(const B8Call& call) {
  const B8Cache& c = call.cache;
  return win_matrix_geometry(call.win.dtype, c.hq, c.kvh, c.d, static_cast<int>(c.bs.d)) &&
         c.group.d % 16 == 0 && aligned16(c.kd, c.vd);
}

}  // namespace kvq
