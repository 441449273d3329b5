// SPDX-License-Identifier: Apache-2.0
// A step's rows into 8-bit pages with the position rotation applied on the way: queries and
// keys rotated, keys and values quantized and scattered by slot, in one launch.
//
// Rotation of row x at position p by the table row (cos | sin)(p), rot / 2 of each:
//   y[a] = x[a] c - x[b] s,  y[b] = x[b] c + x[a] s
// for the pairs (a, b) = (i, i + rot / 2), or (2 i, 2 i + 1) where interleaved; dims from rot
// on pass through.  fp32, each product and sum rounded once; queries are rounded once to
// their type, keys not before they are quantized.
//
// Three destinations:
//   a scale for each token and head (E4M3; also the latent rows, one "head"):
//     scale = max(amax|y| / 448, 1e-6), code = e4m3(y / scale) as fp8_kv.hip;
//   a scale for each block of G slots and head (E4M3 or INT8), which its rows may reach in
//   several calls: S = s(amax of the new rows), or, where the first of them lies behind the
//   block's start, the larger of that and the old scale, the rows before them requantized
//   when it grows:
//     E4M3  s(a) = max(2^-20, the least 2^e with a <= 448 2^e): the codes float, so a power
//           of two loses nothing, and growth only moves their exponents (exact but for
//           subnormal codes);
//     INT8  s(a) = max(a / 127, 1e-6), code = rint(y / S), requantized rint(code old / S):
//           half a step of the new scale more at every growth (a block of 128 rows of one
//           size, a row a call: 4.5 growths, 1.30 times the error of one call, rms).
//   A scale only grows until a row at the block's start: what a token that is taken back did
//   to it stays.
// Maxima are over the bits of |y|: a NaN is the largest, so a row (block) that holds one, or
// an infinity, gets a scale of NaN and stays NaN.
//
// A lane holds 16 dims of a row as two runs of 8 that hold each other's pairs, so that a
// row is read once, rotated in registers and written as whole 64-byte runs; a group of
// d / 16 lanes holds a row.  Other geometry (dims or rotations off 16, unaligned rows): a
// wave a row, a lane up to four pairs, element by element.
// A block's new rows are one workgroup's (a head and side): maximum, then codes, rows past
// the first kKeep of a lane read twice (from L2).
//
// Bound by HBM: eight prompts of 14911 tokens, 40 + 16 heads of 128 (406 MB) 81 us, 5.0 TB/s; 12300
// latent rows of 512 with 128 heads of 64 (428 MB) 85 - 89 us, 5.0 - 4.8 TB/s.  Blocks of 128 in
// nine chunks (306 MB) 91 us, 3.4 TB/s: a block's maximum comes before its codes, rows past
// the kept ones are read again for them, and store_run asks for a row's slot, position, table
// row and elements one after the other.
#include <algorithm>

#include "fp8_codes.h"

namespace {

using namespace kvq;

enum Mode { kToken, kBlockE4M3, kBlockInt8 };

// Rows of the tokens: head h of token t at p + t * ts + h * hs.
struct Rows {
  const void* p;
  int64_t ts, hs;
};

struct Step {
  int64_t tokens;
  // rotation: none without a table
  const void *positions, *table;
  int64_t table_rows;
  int pos64, table_type, rot, inter;
  const void* slots;
  int slot64;
  int64_t num_slots;
  // what is stored: rows of keys (rotated) and values, or of one side alone (not rotated),
  // kvh heads of d
  Rows side[2];
  uint8_t* data[2];
  float* scale[2];
  int sides, kvh, d;
  FastDiv per_token;  // rows of a token: sides * kvh
  int shift;          // 2^shift lanes hold a row
  // blocks of `group` slots
  int64_t group;
  int group_shift;  // -1: no power of two
  int chunk;        // tokens of a workgroup
  int64_t store_blocks;
  // what is only rotated: `heads` rows of width, and then `extra` (0 or 1) row that goes to its
  // token's slot of `part`
  Rows query, extra_row;
  void* out;
  int64_t out_ts, out_hs;
  void* part;
  int heads, extra, width;
  FastDiv units, hgroups;  // 16-dim units of a row; a thread's heads are hgroups apart
};

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i]
              : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}
// Token t's slot, negative for padding and slots outside the cache.
__device__ __forceinline__ int64_t slot_of(const Step& s, int64_t t) {
  const int64_t x = index_at(s.slots, t, s.slot64);
  return x < s.num_slots ? x : -1;
}
// Token t's row of the table, negative outside it.
__device__ __forceinline__ int64_t place_of(const Step& s, int64_t t) {
  if (!s.table) return 0;
  const int64_t x = index_at(s.positions, t, s.pos64);
  return x < s.table_rows ? x : -1;
}
// Slot of a token whose rows are stored, else negative.
__device__ __forceinline__ int64_t live_slot(const Step& s, int64_t t) {
  const int64_t x = slot_of(s, t);
  return place_of(s, t) < 0 ? -1 : x;
}
__device__ __forceinline__ int64_t block_of(const Step& s, int64_t slot) {
  return s.group_shift >= 0 ? slot >> s.group_shift : slot / s.group;
}
__device__ __forceinline__ float table_at(const Step& s, int64_t i) {
  if (s.table_type == KVQ_DTYPE_F32) return static_cast<const float*>(s.table)[i];
  if (s.table_type == KVQ_DTYPE_F16) return to_f32(static_cast<const f16*>(s.table)[i]);
  return to_f32(static_cast<const bf16*>(s.table)[i]);
}
__device__ __forceinline__ void table8(const Step& s, int64_t i, float (&x)[8]) {
  if (s.table_type == KVQ_DTYPE_F32) {
    Raw8<float> r;
    r.load(static_cast<const float*>(s.table) + i);
    r.get(x);
  } else if (s.table_type == KVQ_DTYPE_F16) {
    Raw8<f16> r;
    r.load(static_cast<const f16*>(s.table) + i);
    r.get(x);
  } else {
    Raw8<bf16> r;
    r.load(static_cast<const bf16*>(s.table) + i);
    r.get(x);
  }
}

// ---- a lane's share of a row ---------------------------------------------------------

constexpr uint32_t kNotFinite = 0x7f800000u;  // bits of |x| from here on
constexpr int kGenPairs = 4;  // pairs of a lane where a wave holds a row: d <= 512

// FAST: 16 dims, x[0..7] from a, x[8..15] from b.  Otherwise pair lane + 64 j in x[2 j],
// x[2 j + 1].
template <bool FAST>
struct Share {
  static constexpr int N = FAST ? 16 : 2 * kGenPairs;
  float x[N];
};

// Where FAST unit u begins (its second run in b).
__device__ __forceinline__ int unit_at(const Step& s, bool rotate, int u, int& b) {
  if (rotate && !s.inter && 16 * u < s.rot) {
    b = 8 * u + s.rot / 2;
    return 8 * u;
  }
  b = 16 * u + 8;
  return 16 * u;
}
// The dims of pair p.
__device__ __forceinline__ int pair_at(const Step& s, bool rotate, int p, int& b) {
  if (rotate && !s.inter && 2 * p < s.rot) {
    b = p + s.rot / 2;
    return p;
  }
  b = 2 * p + 1;
  return 2 * p;
}

// Lane `lane` of the row's share of it; what lies past its end is 0.
template <typename T, bool FAST>
__device__ __forceinline__ void load_share(const Step& s, const T* row, int d, bool rotate, int lane,
                                           Share<FAST>& y) {
  if constexpr (FAST) {
    const bool on = 16 * lane < d;
    int b;
    const int a = unit_at(s, rotate, on ? lane : 0, b);
    Raw8<T> raw[2];
    raw[0].load(row + a);
    raw[1].load(row + b);
    float lo[8], hi[8];
    raw[0].get(lo);
    raw[1].get(hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y.x[i] = on ? lo[i] : 0.0f;
      y.x[8 + i] = on ? hi[i] : 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kGenPairs; ++j) {
      const int p = lane + 64 * j;
      int b;
      const int a = pair_at(s, rotate, p, b);
      const bool on = 2 * p < d;
      y.x[2 * j] = on ? to_f32(row[a]) : 0.0f;
      y.x[2 * j + 1] = on ? to_f32(row[b]) : 0.0f;
    }
  }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}
__device__ __forceinline__ void turn16(const Step& s, const float (&c)[8], const float (&n)[8],
                                       float (&x)[16]) {
  if (s.inter) {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[2 * i], x[2 * i + 1], c[i], n[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(x[i], x[8 + i], c[i], n[i]);
  }
}
// Rotates the share to table row `place`.
template <bool FAST>
__device__ __forceinline__ void rotate_share(const Step& s, int64_t place, int lane, Share<FAST>& y) {
  if constexpr (FAST) {
    if (16 * lane >= s.rot) return;
    float c[8], n[8];
    table8(s, place * s.rot + 8 * lane, c);
    table8(s, place * s.rot + s.rot / 2 + 8 * lane, n);
    turn16(s, c, n, y.x);
  } else {
#pragma unroll
    for (int j = 0; j < kGenPairs; ++j) {
      const int p = lane + 64 * j;
      if (2 * p < s.rot)
        turn(y.x[2 * j], y.x[2 * j + 1], table_at(s, place * s.rot + p),
             table_at(s, place * s.rot + s.rot / 2 + p));
    }
  }
}

// The largest |x| of the share, as bits.
template <bool FAST>
__device__ __forceinline__ uint32_t share_max(const Share<FAST>& y) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < Share<FAST>::N; ++i) m = max(m, __float_as_uint(y.x[i]) & 0x7fffffffu);
  return m;
}
template <int MASK>
__device__ __forceinline__ uint32_t xor_max(uint32_t m) {
  return max(m, __float_as_uint(lane_xor<MASK>(__uint_as_float(m))));
}
// Over groups of 2^shift lanes (uniform).
__device__ __forceinline__ uint32_t lanes_max(uint32_t m, int shift) {
  if (shift > 0) m = xor_max<1>(m);
  if (shift > 1) m = xor_max<2>(m);
  if (shift > 2) m = xor_max<4>(m);
  if (shift > 3) m = xor_max<8>(m);
  if (shift > 4) m = xor_max<16>(m);
  if (shift > 5) m = xor_max<32>(m);
  return m;
}

// A word of the codes rint(t[i]) within +-127.
__device__ __forceinline__ uint32_t int8_word(const float (&t)[4]) {
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = static_cast<int>(__builtin_amdgcn_fmed3f(rintf(t[i]), -127.0f, 127.0f));
    c |= (static_cast<uint32_t>(x) & 0xffu) << (8 * i);
  }
  return c;
}
// Codes rint(x / scale), byte i that of x[i].
// With t = RN(x RN(1 / scale)), |t| <= 127.1, t and RN(x / scale) lie within 127.1 * 3 * 2^-24
// < 2^-15 of each other, so they round alike unless t lies that near to a half: then the
// division decides.
template <int N>
__device__ __forceinline__ void int8_codes(const float (&x)[N], float scale, uint32_t (&codes)[N / 4]) {
  const float inv = __fdiv_rn(1.0f, scale);
#pragma unroll
  for (int w = 0; w < N / 4; ++w) {
    float t[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = x[4 * w + i] * inv;
      near = near || !(fabsf(t[i] - rintf(t[i])) < 0.5f - 0x1p-15f);
    }
    if (near) {
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = __fdiv_rn(x[4 * w + i], scale);
    }
    codes[w] = int8_word(t);
  }
}

template <int MODE, int N>
__device__ __forceinline__ void make_codes(const float (&x)[N], float scale, uint32_t (&codes)[N / 4]) {
  if constexpr (MODE == kToken) {
    quantize_codes<N>(x, scale, codes);
  } else if constexpr (MODE == kBlockInt8) {
    int8_codes<N>(x, scale, codes);
  } else {
    const float inv = __fdiv_rn(1.0f, scale);  // a power of two: the quotient is a product
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t[i] = __builtin_amdgcn_fmed3f(x[4 * w + i] * inv, -kE4M3Max, kE4M3Max);
      codes[w] = e4m3x4(t[0], t[1], t[2], t[3]);
    }
  }
}

template <bool FAST, int N>
__device__ __forceinline__ void put_codes(const Step& s, uint8_t* row, bool rotate, int lane,
                                          const uint32_t (&codes)[N / 4]) {
  if constexpr (FAST) {
    if (16 * lane >= s.d) return;
    int b;
    const int a = unit_at(s, rotate, lane, b);
    *reinterpret_cast<uint2*>(row + a) = make_uint2(codes[0], codes[1]);
    *reinterpret_cast<uint2*>(row + b) = make_uint2(codes[2], codes[3]);
  } else {
#pragma unroll
    for (int j = 0; j < kGenPairs; ++j) {
      const int p = lane + 64 * j;
      if (2 * p >= s.d) continue;
      int b;
      const int a = pair_at(s, rotate, p, b);
      row[a] = static_cast<uint8_t>(codes[j / 2] >> (16 * (j % 2)));
      row[b] = static_cast<uint8_t>(codes[j / 2] >> (16 * (j % 2) + 8));
    }
  }
}

// Keys (side 0 of two) are rotated, values are not.
__device__ __forceinline__ bool rotates(const Step& s, int side) {
  return s.table && s.sides == 2 && side == 0;
}
template <typename T>
__device__ __forceinline__ const T* source(const Step& s, int side, int64_t t, int h) {
  // (indexed by a constant: the argument stays out of scratch)
  const Rows& r = side ? s.side[1] : s.side[0];
  return static_cast<const T*>(r.p) + t * r.ts + h * r.hs;
}
__device__ __forceinline__ uint8_t* data_of(const Step& s, int side) {
  return side ? s.data[1] : s.data[0];
}
__device__ __forceinline__ float* scale_of(const Step& s, int side) {
  return side ? s.scale[1] : s.scale[0];
}

// ---- a scale for each token and head -------------------------------------------------

template <typename T, bool FAST>
__device__ __forceinline__ void store_tokens(const Step& s) {
  constexpr int N = Share<FAST>::N;
  const int lane = threadIdx.x & ((1 << s.shift) - 1);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> s.shift;
  if (row >= s.tokens * s.per_token.d) return;  // whole groups leave together
  const uint32_t t = s.per_token.div(static_cast<uint32_t>(row));
  int h = static_cast<int>(static_cast<uint32_t>(row) - t * s.per_token.d);
  const int side = h >= s.kvh ? 1 : 0;
  h -= side * s.kvh;
  const bool rotate = rotates(s, side);
  const int64_t slot = slot_of(s, t), place = place_of(s, t);
  Share<FAST> y;
  load_share<T, FAST>(s, source<T>(s, side, t, h), s.d, rotate, lane, y);
  if (slot < 0 || place < 0) return;
  if (rotate) rotate_share<FAST>(s, place, lane, y);
  const uint32_t top = lanes_max(share_max<FAST>(y), s.shift);
  float scale = __fdiv_rn(__uint_as_float(top), kE4M3Max);
  scale = top >= kNotFinite ? NAN : scale < kScaleFloor ? kScaleFloor : scale;
  uint32_t codes[N / 4];
  make_codes<kToken, N>(y.x, scale, codes);
  const int64_t at = slot * s.kvh + h;
  put_codes<FAST, N>(s, data_of(s, side) + at * s.d, rotate, lane, codes);
  if (lane == 0) scale_of(s, side)[at] = scale;
}

// ---- a scale for each block of slots and head ----------------------------------------

// s(a) of the bits of a >= 0.
template <int MODE>
__device__ __forceinline__ float block_scale(uint32_t top) {
  if (top >= kNotFinite) return NAN;
  if constexpr (MODE == kBlockInt8) {
    const float s = __fdiv_rn(__uint_as_float(top), 127.0f);
    return s < kScaleFloor ? kScaleFloor : s;
  } else {
    // 448 = 1.75 * 2^8
    const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(e, 127 - 20)) << 23);
  }
}

template <int MODE>
__device__ __forceinline__ uint32_t requantize(uint32_t w, float old, float scale) {
  float x[4];
  if constexpr (MODE == kBlockInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  } else {
    e4m3x4_f32(w, x);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __fdiv_rn(__fmul_rn(x[i], old), scale);
  return MODE == kBlockInt8 ? int8_word(x) : e4m3x4(x[0], x[1], x[2], x[3]);
}

// Rows of a lane that stay in registers between maximum and codes: the wave has to leave room
// for the waves that rotate queries beside it.  Nine chunks of 11503 tokens, 40 + 16 heads of
// 128 (306 MB), us a call with 16 tokens a workgroup: four rows in 166 registers 105, two in
// 128 (one more goes to scratch, bf16 and fp32) 97; 512 decodes 49 and 39.  One row, in 96
// registers: 114 and 57.
constexpr int kKeep = 2;

// The run of tokens that begins at t0 and shares its block.
template <typename T, bool FAST, int MODE>
__device__ __forceinline__ void store_run(const Step& s, int64_t t0, int side, int h, uint32_t* red) {
  constexpr int N = Share<FAST>::N;
  const int tid = threadIdx.x, lane64 = tid & 63;
  const int64_t slot0 = live_slot(s, t0), block = block_of(s, slot0);
  // its end, and the first slot of the block that it writes
  int64_t end = t0 + 1;
  int first = static_cast<int>(slot0 - block * s.group);
  for (;; end += 64) {
    const int64_t t = end + lane64;
    const int64_t x = t < s.tokens ? live_slot(s, t) : -1;
    const bool other = t >= s.tokens || (x >= 0 && block_of(s, x) != block);
    const uint64_t stop = __builtin_amdgcn_ballot_w64(other);
    const int n = stop ? __builtin_ctzll(stop) : 64;
    if (lane64 < n && x >= 0) first = min(first, static_cast<int>(x - block * s.group));
    if (stop) {
      end += n;
      break;
    }
  }
  if (end > t0 + 1) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) first = min(first, __shfl_xor(first, m, 64));
  }
  float* const scale_at = scale_of(s, side) + block * s.kvh + h;
  uint8_t* const data = data_of(s, side);
  const float old = first > 0 ? *scale_at : 0.0f;
  const bool rotate = rotates(s, side);
  const int lane = tid & ((1 << s.shift) - 1), each = 256 >> s.shift;  // rows at once
  const int64_t r0 = t0 + (tid >> s.shift);
  auto fetch = [&](int64_t t, Share<FAST>& y) {
    const int64_t place = place_of(s, t);
    load_share<T, FAST>(s, source<T>(s, side, t, h), s.d, rotate, lane, y);
    if (rotate) rotate_share<FAST>(s, place, lane, y);
  };
  Share<FAST> kept[kKeep];
  int64_t slots[kKeep];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    const int64_t t = r0 + j * each;
    slots[j] = t < end ? live_slot(s, t) : -1;
    if (slots[j] >= 0) {
      fetch(t, kept[j]);
      top = max(top, share_max<FAST>(kept[j]));
    }
  }
  for (int64_t t = r0 + kKeep * each; t < end; t += each) {
    if (live_slot(s, t) < 0) continue;
    Share<FAST> y;
    fetch(t, y);
    top = max(top, share_max<FAST>(y));
  }
  top = lanes_max(top, 6);
  if (lane64 == 0) red[tid >> 6] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  // (by their bits: a NaN stays the largest)
  const float scale = __uint_as_float(max(__float_as_uint(block_scale<MODE>(top)), __float_as_uint(old)));
  if (first > 0 && __float_as_uint(scale) != __float_as_uint(old)) {  // grown: uniform
    constexpr int W = FAST ? 16 : 4;
    const int units = s.d / W;
    for (int i = tid; i < first * units; i += 256) {
      const int row = i / units, u = i - row * units;
      uint8_t* p = data + ((block * s.group + row) * s.kvh + h) * s.d + W * u;
      if constexpr (FAST) {
        uint4 w = *reinterpret_cast<uint4*>(p);
        w.x = requantize<MODE>(w.x, old, scale);
        w.y = requantize<MODE>(w.y, old, scale);
        w.z = requantize<MODE>(w.z, old, scale);
        w.w = requantize<MODE>(w.w, old, scale);
        *reinterpret_cast<uint4*>(p) = w;
      } else {
        uint32_t* q = reinterpret_cast<uint32_t*>(p);
        *q = requantize<MODE>(*q, old, scale);
      }
    }
  }
  if (tid == 0) *scale_at = scale;
  auto put = [&](int64_t slot, const Share<FAST>& y) {
    uint32_t codes[N / 4];
    make_codes<MODE, N>(y.x, scale, codes);
    put_codes<FAST, N>(s, data + (slot * s.kvh + h) * s.d, rotate, lane, codes);
  };
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (slots[j] >= 0) put(slots[j], kept[j]);
  for (int64_t t = r0 + kKeep * each; t < end; t += each) {
    const int64_t slot = live_slot(s, t);
    if (slot < 0) continue;
    Share<FAST> y;
    fetch(t, y);
    put(slot, y);
  }
  __syncthreads();  // red is read, and the old scale
}

// A workgroup: the blocks whose first row in the call is one of its tokens, for a head and
// side.
template <typename T, bool FAST, int MODE>
__device__ __forceinline__ void store_blocks(const Step& s) {
  __shared__ uint32_t red[4];
  const uint32_t rest = s.per_token.div(blockIdx.x);
  int h = static_cast<int>(blockIdx.x - rest * s.per_token.d);
  const int side = h >= s.kvh ? 1 : 0;
  h -= side * s.kvh;
  const int64_t c0 = static_cast<int64_t>(rest) * s.chunk;
  const int lane = threadIdx.x & 63;
  const int64_t x = lane < s.chunk && c0 + lane < s.tokens ? live_slot(s, c0 + lane) : -1;
  const int64_t block = x < 0 ? -1 : block_of(s, x);
  // the block of the last token before it that is stored, among these or before them
  const uint64_t lives = __builtin_amdgcn_ballot_w64(x >= 0);
  if (!lives) return;
  const uint64_t below = lives & ((1ull << lane) - 1);
  int64_t before = __shfl(block, below ? 63 - __builtin_clzll(below) : lane, 64);
  if (!below) before = -1;
  for (int64_t end = c0; end > 0; end -= 64) {
    const int64_t p = end - 1 - lane;
    const int64_t y = p < 0 ? -1 : live_slot(s, p);
    const uint64_t found = __builtin_amdgcn_ballot_w64(y >= 0);
    if (!found) continue;
    const int64_t last = __shfl(y, __builtin_ctzll(found), 64);
    if (!below) before = block_of(s, last);
    break;
  }
  const bool start = x >= 0 && before != block;
  uint64_t starts = __builtin_amdgcn_ballot_w64(start);
  while (starts) {  // the same in every wave
    store_run<T, FAST, MODE>(s, c0 + __builtin_ctzll(starts), side, h, red);
    starts &= starts - 1;
  }
}

// ---- queries --------------------------------------------------------------------------

// FAST: a thread's 16 dims of HEADS heads of a token, whose cosines it loads once.
template <typename T, bool FAST, int HEADS>
__device__ __forceinline__ void rotate_rows(const Step& s, int64_t block) {
  const int all = s.heads + s.extra;
  auto from = [&](int64_t t, int h) {
    const Rows& r = s.query;
    return h < s.heads ? static_cast<const T*>(r.p) + t * r.ts + h * r.hs
                       : static_cast<const T*>(s.extra_row.p) + t * s.extra_row.ts;
  };
  // nullptr: nowhere
  auto to = [&](int64_t t, int h, int64_t place) -> T* {
    if (h < s.heads) return static_cast<T*>(s.out) + t * s.out_ts + h * s.out_hs;
    const int64_t slot = slot_of(s, t);
    return slot < 0 || place < 0 ? nullptr : static_cast<T*>(s.part) + slot * s.width;
  };
  if constexpr (FAST) {
    const int64_t item = block * 256 + threadIdx.x;
    const int hg = static_cast<int>(s.hgroups.d);
    if (item >= s.tokens * s.units.d * hg) return;
    const uint32_t rest = s.units.div(static_cast<uint32_t>(item));
    const int u = static_cast<int>(static_cast<uint32_t>(item) - rest * s.units.d);
    const uint32_t t = s.hgroups.div(rest);
    const int h0 = static_cast<int>(rest - t * s.hgroups.d);
    int b;
    const int a = unit_at(s, true, u, b);
    Raw8<T> lo[HEADS], hi[HEADS];
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      const T* row = from(t, min(h0 + j * hg, all - 1));
      lo[j].load(row + a);
      hi[j].load(row + b);
    }
    const int64_t place = place_of(s, t);
    float c[8], n[8];
    const bool on = 16 * u < s.rot;
    if (on && place >= 0) {
      table8(s, place * s.rot + 8 * u, c);
      table8(s, place * s.rot + s.rot / 2 + 8 * u, n);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = n[i] = NAN;  // outside the table
    }
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      const int h = h0 + j * hg;
      if (h >= all) break;
      float x[16], y[8];
      lo[j].get(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = y[i];
      hi[j].get(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 + i] = y[i];
      if (on) turn16(s, c, n, x);
      T* const row = to(t, h, place);
      if (!row) break;  // (the last)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
      store8(row + a, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[8 + i];
      store8(row + b, y);
    }
  } else {  // a wave a row
    const int64_t row = block * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= s.tokens * all) return;
    const int64_t t = row / all;
    const int h = static_cast<int>(row - t * all);
    Share<false> y;
    load_share<T, false>(s, from(t, h), s.width, true, lane, y);
    const int64_t place = place_of(s, t);
    if (place >= 0) rotate_share<false>(s, place, lane, y);
    T* const dst = to(t, h, place);
    if (!dst) return;
#pragma unroll
    for (int j = 0; j < kGenPairs; ++j) {
      const int p = lane + 64 * j;
      if (2 * p >= s.width) continue;
      int b;
      const int a = pair_at(s, true, p, b);
      const bool lost = place < 0 && 2 * p < s.rot;  // outside the table
      dst[a] = from_f32<T>(lost ? NAN : y.x[2 * j]);
      dst[b] = from_f32<T>(lost ? NAN : y.x[2 * j + 1]);
    }
  }
}

template <typename T, bool FAST, int MODE, int HEADS>
__global__ void __launch_bounds__(256, 4) rotary_store_kernel(Step s) {
  if (blockIdx.x >= s.store_blocks) {
    rotate_rows<T, FAST, HEADS>(s, static_cast<int64_t>(blockIdx.x) - s.store_blocks);
    return;
  }
  if constexpr (MODE == kToken)
    store_tokens<T, FAST>(s);
  else
    store_blocks<T, FAST, MODE>(s);
}

// ---- host -------------------------------------------------------------------------------

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Every row of 16-byte runs.
bool wide_rows(const Rows& r, int64_t bytes) {
  return on16(r.p) && r.ts * bytes % 16 == 0 && r.hs * bytes % 16 == 0;
}

template <typename T, bool FAST, int MODE>
int launch_heads(Step& s, hipStream_t stream) {
  const int all = s.heads + s.extra;
  int64_t rotate = 0;
  int heads = 1;
  if (all > 0) {
    if (FAST) {
      const int units = s.width / 16;
      // four heads a thread once that leaves threads enough for every CU
      if (s.tokens * all * units >= 4 * 256 * 1024) heads = 4;
      const int hg = (all + heads - 1) / heads;
      s.units = FastDiv::make(static_cast<uint32_t>(units));
      s.hgroups = FastDiv::make(static_cast<uint32_t>(hg));
      const int64_t items = s.tokens * units * hg;
      if (items > 0x7fffff00) return KVQ_ERR_INVALID;
      rotate = (items + 255) / 256;
    } else {
      rotate = (s.tokens * all + 3) / 4;
    }
  }
  const int64_t blocks = s.store_blocks + rotate;
  if (blocks == 0) return KVQ_OK;
  if (blocks > 0x7fffffff) return KVQ_ERR_INVALID;
  if (FAST && heads == 4)
    hipLaunchKernelGGL((rotary_store_kernel<T, FAST, MODE, 4>), dim3(static_cast<unsigned>(blocks)),
                       dim3(256), 0, stream, s);
  else
    hipLaunchKernelGGL((rotary_store_kernel<T, FAST, MODE, 1>), dim3(static_cast<unsigned>(blocks)),
                       dim3(256), 0, stream, s);
  KVQ_LAUNCH_CHECK();
  return KVQ_OK;
}

template <int MODE>
int launch_store(Step& s, int dtype, hipStream_t stream) {
  const int64_t bytes = dtype == KVQ_DTYPE_F32 ? 4 : 2;
  bool fast = s.d % 16 == 0 && s.rot % 16 == 0 && s.width % 16 == 0 && on16(s.table);
  for (int i = 0; i < s.sides; ++i) fast = fast && wide_rows(s.side[i], bytes) && on16(s.data[i]);
  if (s.heads > 0)
    fast = fast && wide_rows(s.query, bytes) && wide_rows(Rows{s.out, s.out_ts, s.out_hs}, bytes);
  if (s.extra > 0) fast = fast && wide_rows(s.extra_row, bytes) && on16(s.part);
  s.shift = 6;
  if (fast) {
    s.shift = 0;
    while ((16 << s.shift) < s.d) ++s.shift;
  }
  s.per_token = FastDiv::make(static_cast<uint32_t>(s.sides * s.kvh));
  const int64_t rows = s.tokens * s.sides * s.kvh;
  if (rows > 0x7fffffff) return KVQ_ERR_INVALID;
  if (MODE == kToken) {
    s.store_blocks = ((rows << s.shift) + 255) / 256;
  } else {
    // A workgroup takes the blocks that begin in its tokens one after another, and one that
    // finds none is time lost.  us a call at 1, 4, 16, 32 and 64 tokens: 11503 tokens of nine
    // chunks 271, 139, 94, 85 and 82 in blocks of 128, 324, 193, 111, 101 and 95 in blocks of
    // 16; 1100 decodes 77, 65, 88, 95 and 172, 1100 tokens of one chunk 32, 23, 22, 22 and 22.
    s.chunk = s.tokens <= 1024 ? 1 : (s.tokens <= 2048 ? 4 : 32);
    s.store_blocks = (s.tokens + s.chunk - 1) / s.chunk * s.sides * s.kvh;
  }
  KVQ_DISPATCH_FLOAT(dtype, T, {
    return fast ? launch_heads<T, true, MODE>(s, stream) : launch_heads<T, false, MODE>(s, stream);
  });
  return KVQ_ERR_INVALID;
}

bool index_type(int x) { return x == KVQ_INDEX_I32 || x == KVQ_INDEX_I64; }
bool float_type(int x) { return x == KVQ_DTYPE_F32 || x == KVQ_DTYPE_F16 || x == KVQ_DTYPE_BF16; }

// The rotation and the slots of a call.
int begin(Step& s, int64_t tokens, int dtype, const void* positions, int pos_type, const void* table,
          int table_dtype, int64_t table_rows, int rot, int interleaved, const void* slots,
          int slot_type, int64_t num_blocks, int block_size, int d, int width) {
  if (tokens < 0 || !float_type(dtype) || num_blocks <= 0 || block_size <= 0) return KVQ_ERR_INVALID;
  if (d <= 0 || d % 4 || d > 2 * 64 * kGenPairs) return KVQ_ERR_GEOMETRY;
  if (!slots || !index_type(slot_type)) return KVQ_ERR_INVALID;
  s.tokens = tokens;
  s.slots = slots;
  s.slot64 = slot_type == KVQ_INDEX_I64;
  s.num_slots = num_blocks * block_size;
  if (table) {
    if (!positions || !index_type(pos_type) || !float_type(table_dtype) || table_rows <= 0)
      return KVQ_ERR_INVALID;
    if (rot <= 0 || rot % 2 || rot > width || width % 2 || width > 2 * 64 * kGenPairs)
      return KVQ_ERR_GEOMETRY;
    s.positions = positions;
    s.pos64 = pos_type == KVQ_INDEX_I64;
    s.table = table;
    s.table_type = table_dtype;
    s.table_rows = table_rows;
    s.rot = rot;
    s.inter = interleaved != 0;
  }
  return KVQ_OK;
}

template <int MODE>
int store_keys(const void* query, int64_t query_stride, void* out_query, int64_t out_stride,
               const void* key, int64_t key_stride, const void* value, int64_t value_stride,
               int dtype, const void* positions, int pos_type, const void* cos_sin, int table_dtype,
               int64_t table_rows, int rot, int interleaved, const void* slot_mapping, int slot_type,
               int64_t num_tokens, int num_heads, int num_kv_heads, int head_size, void* k_data,
               float* k_scale, void* v_data, float* v_scale, int64_t num_blocks, int block_size,
               int group, void* stream) {
  if (num_tokens == 0) return KVQ_OK;
  Step s{};
  const int rc = begin(s, num_tokens, dtype, positions, pos_type, cos_sin, table_dtype, table_rows,
                       rot, interleaved, slot_mapping, slot_type, num_blocks, block_size, head_size,
                       head_size);
  if (rc != KVQ_OK) return rc;
  if (!key || !value || !k_data || !k_scale || !v_data || !v_scale || num_kv_heads <= 0 ||
      num_kv_heads > 65536 || group <= 0 || block_size % group || num_heads < 0 || num_heads > 65536)
    return KVQ_ERR_INVALID;
  const int64_t row = static_cast<int64_t>(num_kv_heads) * head_size;
  if (num_tokens > 1 && (key_stride < row || value_stride < row)) return KVQ_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(k_data) | reinterpret_cast<uintptr_t>(v_data)) & 3)
    return KVQ_ERR_GEOMETRY;  // a row's words
  if (num_heads > 0 && (!query || !out_query || !cos_sin)) return KVQ_ERR_INVALID;
  s.side[0] = Rows{key, key_stride, head_size};
  s.side[1] = Rows{value, value_stride, head_size};
  s.data[0] = static_cast<uint8_t*>(k_data);
  s.data[1] = static_cast<uint8_t*>(v_data);
  s.scale[0] = k_scale;
  s.scale[1] = v_scale;
  s.sides = 2;
  s.kvh = num_kv_heads;
  s.d = s.width = head_size;
  s.group = group;
  s.group_shift = -1;
  for (int i = 0; i < 31; ++i)
    if ((1 << i) == group) s.group_shift = i;
  s.heads = num_heads;
  s.query = Rows{query, query_stride, head_size};
  s.out = out_query;
  s.out_ts = out_stride;
  s.out_hs = head_size;
  return launch_store<MODE>(s, dtype, static_cast<hipStream_t>(stream));
}

}  // namespace

extern "C" int kvq_fp8_pth_rotary_store(
    const void* query, int64_t query_stride, void* out_query, int64_t out_stride, const void* key,
    int64_t key_stride, const void* value, int64_t value_stride, int dtype, const void* positions,
    int pos_type, const void* cos_sin, int table_dtype, int64_t table_rows, int rot, int interleaved,
    const void* slot_mapping, int slot_type, int64_t num_tokens, int num_heads, int num_kv_heads,
    int head_size, uint8_t* k_data, float* k_scale, uint8_t* v_data, float* v_scale,
    int64_t num_blocks, int block_size, void* stream) {
  return store_keys<kToken>(query, query_stride, out_query, out_stride, key, key_stride, value,
                            value_stride, dtype, positions, pos_type, cos_sin, table_dtype,
                            table_rows, rot, interleaved, slot_mapping, slot_type, num_tokens,
                            num_heads, num_kv_heads, head_size, k_data, k_scale, v_data, v_scale,
                            num_blocks, block_size, 1, stream);
}

extern "C" int kvq_block8_store(
    const void* query, int64_t query_stride, void* out_query, int64_t out_stride, const void* key,
    int64_t key_stride, const void* value, int64_t value_stride, int dtype, const void* positions,
    int pos_type, const void* cos_sin, int table_dtype, int64_t table_rows, int rot, int interleaved,
    const void* slot_mapping, int slot_type, int64_t num_tokens, int num_heads, int num_kv_heads,
    int head_size, int code_type, void* k_data, float* k_scale, void* v_data, float* v_scale,
    int64_t num_blocks, int block_size, int group, void* stream) {
  if (code_type != KVQ_CODES_E4M3 && code_type != KVQ_CODES_INT8) return KVQ_ERR_INVALID;
  const auto store = code_type == KVQ_CODES_INT8 ? store_keys<kBlockInt8> : store_keys<kBlockE4M3>;
  return store(query, query_stride, out_query, out_stride, key, key_stride, value, value_stride,
               dtype, positions, pos_type, cos_sin, table_dtype, table_rows, rot, interleaved,
               slot_mapping, slot_type, num_tokens, num_heads, num_kv_heads, head_size, k_data,
               k_scale, v_data, v_scale, num_blocks, block_size, group, stream);
}

extern "C" int kvq_fp8_latent_store(
    const void* query, int64_t query_stride, int64_t query_head_stride, void* out_query,
    int64_t out_stride, int64_t out_head_stride, const void* latent, int64_t latent_stride,
    const void* part, int64_t part_stride, int dtype, const void* positions, int pos_type,
    const void* cos_sin, int table_dtype, int64_t table_rows, int interleaved,
    const void* slot_mapping, int slot_type, int64_t num_tokens, int num_heads, int rank,
    int part_size, uint8_t* data, float* scale, void* rope, int64_t num_blocks, int block_size,
    void* stream) {
  if (num_tokens == 0) return KVQ_OK;
  Step s{};
  const int rc = begin(s, num_tokens, dtype, positions, pos_type, cos_sin, table_dtype, table_rows,
                       part_size, interleaved, slot_mapping, slot_type, num_blocks, block_size, rank,
                       part_size);
  if (rc != KVQ_OK) return rc;
  if (!latent || !part || !data || !scale || !rope || !cos_sin || num_heads < 0 || num_heads > 65536 ||
      (num_heads > 0 && (!query || !out_query)))
    return KVQ_ERR_INVALID;
  if (num_tokens > 1 && (latent_stride < rank || part_stride < part_size)) return KVQ_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(data) & 3) return KVQ_ERR_GEOMETRY;
  s.side[0] = Rows{latent, latent_stride, 0};
  s.data[0] = data;
  s.scale[0] = scale;
  s.sides = 1;
  s.kvh = 1;
  s.d = rank;
  s.group = 1;
  s.heads = num_heads;
  s.extra = 1;
  s.width = part_size;
  s.query = Rows{query, query_stride, query_head_stride};
  s.extra_row = Rows{part, part_stride, 0};
  s.out = out_query;
  s.out_ts = out_stride;
  s.out_hs = out_head_stride;
  s.part = rope;
  return launch_store<kToken>(s, dtype, static_cast<hipStream_t>(stream));
}
