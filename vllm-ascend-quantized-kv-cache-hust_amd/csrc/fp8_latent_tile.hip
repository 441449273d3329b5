// SPDX-License-Identifier: Apache-2.0
// Attention over latent rows that all heads share, on the matrix units, where a request has
// more columns than a small tile: decodes of many heads, and chunks.
//
// One workgroup of eight waves per tile of 64 columns (row, head), request and part of its
// positions, 64 positions at a time.  The latent is key and value at once, so a stage's codes,
// scales and position parts are read from memory once, by DMA into LDS (three stages of 41 KB
// at R = 512: one whose values are summed, the next, whose scores are formed, and one on its
// way).  What bounds it is the matrix units and the instructions that feed them: each code is
// converted to 16 bits on its way, as a key once per 32 columns, as a value once per 64.  So
// the waves are of two kinds, one of each on every SIMD, and one's products run while the
// other converts, exponentiates or waits:
//   four form scores, wave (p, c) of positions 32 p .. and columns 32 c .. of the NEXT stage:
//     S^T = C * Q^T in products of 32 x 32 x 16; A = codes in the query's type, exact, lane
//     (n, g) dims 32 w + 16 g .. of position n; B = the queries, all R + P dims of its columns
//     in registers (144 of them).  Then t = (S s_j + S_r) scale log2(e) + log2(s_j), S_r the
//     position parts' product, and with m the column's offset p' = 2^(t - m) = p s_j, within
//     fp16's range whatever the scales are, goes through LDS to the others.
//   four sum values, R / 4 dims of all 64 columns each: O^T += C^T * p'^T; A = codes in fp16,
//     exact, by the transposing reads of bytes (16 lanes read 8 rows of 16 bytes, lane s gets
//     column s).  They bring the stages too.
// m moves only when some column's maximum outgrows it by kOutgrow, which all waves learn with
// the weights and then settle together; it leaves the largest p' between 2^7 and 2^15, so p' is
// rounded by 2^-11 of itself, or, where fp16 is subnormal, by 2^-32 of the column's largest.
// The sum takes p' / s_j in fp32 before that rounding.  t is rounded before m is taken off: m
// then follows from scores as they are compared, and t - m stays under 16 also where scores
// have steps of 16 and more (the largest p' is 1 there).
// 16-byte chunk c of row t lies at c ^ t % 16, a position part's at c ^ t % 8, so that the rows
// of an operand are in different banks.
//
// (In 16 bits p' puts fp16 results up to 1.4 times as far off as their own rounding does, bf16
// ones 1.01.)
//
// 64 requests of 1000 - 8192 positions, 256 columns, R = 512, P = 64 (157 GFLOP): 207 us; five
// chunks of 100 - 1024 rows by 16 heads over 1111 - 6000 positions (444 GFLOP): 455 us, 0.98
// PFLOP/s.  The tiles of 32 columns of fp8_latent_mfma.hip take 306 and 693 for them; these
// tiles with all eight waves doing both kinds of work, half the dims of a score each, 270 and
// 535; with four such waves of 512 registers 270 and 520.
//
// Positions that a column does not see: weights by selection; in stages that some column
// does not wholly see, NaN codes become zeros in LDS before they count as values (a row that
// sees one is NaN by its score).
#include <algorithm>

#include "block8.h"
#include "fp8_latent.h"

namespace {

using namespace kvq;

constexpr int kWaves = 8;      // four that score, four that sum values
constexpr int kCols = 64;   // columns of a tile
constexpr int kStage = 64;  // positions
constexpr int kStages = 3;
// a column's maximum lies kRaise over its offset, and up to kOutgrow more before that moves
constexpr float kRaise = 7.0f, kOutgrow = 8.0f;
constexpr float kNone = -0x1p127f;  // the offset of a column that has seen nothing

typedef const __attribute__((address_space(4))) int32_t lat_ci32;
typedef const __attribute__((address_space(4))) int64_t lat_ci64;
typedef int lat_i2 __attribute__((ext_vector_type(2)));
typedef float lat_f16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) lat_i2* lat_lds2;
typedef const __attribute__((address_space(3))) w_u4* lat_cu4;
typedef const __attribute__((address_space(3))) w_f4* lat_cf4;

__device__ __forceinline__ lat_f16 mfma32(w_u4 a, w_u4 b, lat_f16 c, bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(w_b8, a),
                                                 __builtin_bit_cast(w_b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ lat_f16 mfma32(w_u4 a, w_u4 b, lat_f16 c, f16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(w_h8, a),
                                                __builtin_bit_cast(w_h8, b), c, 0, 0, 0);
}

template <int R, int PART>
struct LatLds {
  static constexpr int ROPE = kStage * R;                 // behind the codes: [kStage][PART]
  static constexpr int SCALE = ROPE + 2 * kStage * PART;  // [kStage] floats
  static constexpr int STAGE = SCALE + 512;  // (rows of codes on bounds of their size)
  static constexpr int PROW = 2 * kStage + 16;    // bytes of a column's p', padded
  static constexpr int PBUF = kCols * PROW;
  static constexpr int P = kStages * STAGE;       // two of [kCols][PROW]
  static constexpr int MAX = P + 2 * PBUF;        // [kCols][2] floats
  static constexpr int ROWS = MAX + kCols * 2 * 4;    // [4][4][32] floats of a scoring wave's rows
  static constexpr int FLAG = ROWS + 4 * 4 * 32 * 4;  // two of [4]
  static constexpr int BYTES = FLAG + 2 * 4 * 4;
};

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// A value that the compiler derives others from where they are needed, not ahead.
__device__ __forceinline__ uint32_t anew(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}
// The other half's value, x's lane ^ 32.
__device__ __forceinline__ float max_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <typename T, int R, int PART>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
latent_tile_kernel(WinArg, int count, LatentCache c, const T* __restrict__ query,
                   int64_t q_stride, int wide, float qscale, T* __restrict__ out, WinParts parts) {
  using L = LatLds<R, PART>;
  constexpr int KW = R / 32;     // 16-byte chunks of a row for a lane: two k-steps each
  constexpr int RS = PART / 16;  // k-steps of the position part
  constexpr int DB = R / 128;    // 32-dim blocks of a wave's dims
  constexpr int CH = R / 16;     // 16-byte chunks of a row
  constexpr int RPI = 64 / CH;   // rows a DMA instruction brings
  constexpr int RC = PART / 8;   // 16-byte chunks of a position part
  constexpr int CODE_DMAS = 16 / RPI, ROPE_DMAS = 16 * RC / 64;  // of a wave's 16 rows
  constexpr int PK = kStage / 16;  // k-steps of the values
  constexpr int AHEAD = 5;         // key chunks read ahead
  extern __shared__ __align__(16) char lds[];
  const WinReq r = win_req(count, blockIdx.x);
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, n = lane & 31, g = lane >> 5;
  const bool scorer = wave < 4;
  const int w4 = wave % 4;
  const int ph = w4 % 2, ch = w4 / 2;  // a scoring wave's 32 positions and 32 columns
  const int heads = c.hq, cols = r.n * heads;
  const int tiles = (cols + kCols - 1) / kCols;
  // tiles of a part lie 8 workgroups apart, on one XCD, whose L2 then holds its codes once
  int u = static_cast<int>(blockIdx.x) - r.first;
  const int set = u / (8 * tiles);
  u -= set * 8 * tiles;
  const int across = min(8, r.parts - 8 * set);
  const int tile = tiles - 1 - u / across, seg = 8 * set + u % across;
  const int col0 = kCols * tile;
  auto row_of = [&](int col) { return static_cast<int>(c.rep.div(static_cast<uint32_t>(col))); };
  const int base = r.len - r.n;  // position of the request's first row
  const int tile_last = base + row_of(min(col0 + kCols, cols) - 1);
  const int tile_first = base + row_of(col0);
  // the lane's column of group x, found where it is needed; one past the last sees nothing
  struct Col {
    bool live;
    int row, head, pos;
  };
  auto col_at = [&](int x) {
    const int col = static_cast<int>(anew(col0 + 32 * x + n));
    Col y;
    y.live = col < cols;
    y.row = row_of(y.live ? col : 0);
    y.head = (y.live ? col : 0) - y.row * heads;
    y.pos = y.live ? base + y.row : -1;
    return y;
  };
  const int stages = tile_last >= 0 ? (tile_last + kStage) / kStage : 0;
  const int s0 = static_cast<int>(static_cast<int64_t>(stages) * seg / r.parts);
  const int s1 = static_cast<int>(static_cast<int64_t>(stages) * (seg + 1) / r.parts);
  if (s0 >= s1) {  // uniform: a part without positions, or columns that see nothing
    for (int x = tid; x < kCols * (R / 4); x += 64 * kWaves) {
      const int col = col0 + x / (R / 4);
      if (col >= cols) break;
      const int i = row_of(col);
      const int64_t at = (static_cast<int64_t>(r.q0) + i) * heads + col - i * heads;
      if (r.parts > 1) {
        const int64_t part = r.part0 + static_cast<int64_t>(seg) * r.n * heads + col;
        if (x % (R / 4) == 0) *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{-INFINITY, 0.0f};
      } else {
        for (int e = 0; e < 4; ++e) out[at * R + 4 * (x % (R / 4)) + e] = from_f32<T>(0.0f);
      }
    }
    return;
  }

  // ---- a stage on its way: a summing wave brings 16 rows of it, all in one page ----
  const uint32_t lds0 = win_lds(lds);
  const int groups = (r.len + 15) / 16;
  auto place_of = [&](int stage) { return 16 * min(4 * stage + w4, groups - 1); };
  // the page of the wave's rows of a stage, asked for a stage ahead: it comes by a scalar load
  auto page_of = [&](int stage) -> int64_t {
    const int i = static_cast<int>(c.bs.div(static_cast<uint32_t>(place_of(stage))));
    const int64_t at =
        __builtin_amdgcn_readfirstlane(i < c.maxb ? i : static_cast<int>(c.maxb - 1));
    const int64_t e = static_cast<int64_t>(r.table) * c.maxb + at;
    return c.bt64 ? ((lat_ci64*)(const void*)c.table)[e]
                  : static_cast<int64_t>(((lat_ci32*)(const void*)c.table)[e]);
  };
  auto slot_of = [&](int stage, int64_t id) -> int64_t {
    const int64_t page = id < 0 ? 0 : (id >= c.nb ? c.nb - 1 : id);
    const uint32_t p = static_cast<uint32_t>(place_of(stage));
    return page * c.bs.d + (p - c.bs.div(p) * c.bs.d);
  };
  const uint32_t code_off = lane / CH * R + 16 * ((lane % CH) ^ (lane / CH));
  const uint32_t rope_off = lane / RC * 2 * PART + 16 * ((lane % RC) ^ (lane / RC % RC));
  constexpr int DMAS = CODE_DMAS + ROPE_DMAS + 1;
  auto issue = [&](int j, int64_t slot, uint32_t to) {
    if (j < CODE_DMAS)
      win_dma16(c.kd + slot * R + j * 1024, code_off ^ (16 * RPI * j), to + w4 * 16 * R + j * 1024);
    else if (j < CODE_DMAS + ROPE_DMAS)
      win_dma16(static_cast<const T*>(c.rope) + slot * PART + 512 * (j - CODE_DMAS), rope_off,
                to + L::ROPE + w4 * 32 * PART + 1024 * (j - CODE_DMAS));
    else if (j == DMAS - 1 && lane < 16)
      win_dma4(c.ks + slot, 4 * lane, to + L::SCALE + w4 * 64);
  };
  auto stage_at = [&](int slot3) { return lds0 + slot3 * L::STAGE; };
  auto is_edge = [&](int st) { return st * kStage + kStage - 1 > tile_first; };  // uniform
  auto stage_after = [](int at) { return at == kStages - 1 ? 0 : at + 1; };
  float* const smax = reinterpret_cast<float*>(lds + L::MAX);
  int* const flags = reinterpret_cast<int*>(lds + L::FLAG);
  // whether a maximum outgrew its column's offset in a stage: then all waves move the offsets
  auto outgrown = [&](int st) {
    const w_u4 flag = *(lat_cu4)(win_lds(flags) + st % 2 * 16);
    return __builtin_amdgcn_readfirstlane(flag[0] | flag[1] | flag[2] | flag[3]) != 0;
  };
  auto moved = [&](int x, float was) {
    const w_f2 y = *reinterpret_cast<const w_f2*>(smax + 2 * (32 * x + n));
    const float mx = fmaxf(y[0], y[1]);
    return mx - was > kRaise + kOutgrow ? mx - kRaise : was;
  };

  if (scorer) {
    // ---- scores and weights ----
    w_u4 q[2 * KW], qr[RS];
    {
      const Col y = col_at(ch);
      const T* qrow = query + (static_cast<int64_t>(r.q0) + y.row) * q_stride +
                      static_cast<int64_t>(y.head) * (R + PART);
      if (wide & 1) {
#pragma unroll
        for (int s = 0; s < 2 * KW; ++s)
          q[s] = load_op8(qrow + 32 * (s / 2) + 16 * g + 8 * (s % 2), true);
#pragma unroll
        for (int s = 0; s < RS; ++s) qr[s] = load_op8(qrow + R + 16 * s + 8 * g, true);
      } else {
#pragma unroll
        for (int s = 0; s < 2 * KW; ++s)
          q[s] = load_op8(qrow + 32 * (s / 2) + 16 * g + 8 * (s % 2), false);
#pragma unroll
        for (int s = 0; s < RS; ++s) qr[s] = load_op8(qrow + R + 16 * s + 8 * g, false);
      }
      if (!y.live) {
#pragma unroll
        for (int s = 0; s < 2 * KW; ++s) q[s] = w_u4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < RS; ++s) qr[s] = w_u4{0, 0, 0, 0};
      }
    }
    float m = kNone, l = 0.0f;
    const uint32_t k_row = 32 * ph + n;
    const uint32_t k_off = k_row * R + 16 * (g ^ (n % 16));
    const uint32_t r_off = L::ROPE + k_row * 2 * PART + 16 * (g ^ (n % RC));
    char* const p_write = lds + L::P + (32 * ch + n) * L::PROW + 2 * (32 * ph + 4 * g);
    float* const rows = reinterpret_cast<float*>(lds + L::ROWS) + w4 * 128;
    const uint32_t rows_lds = win_lds(rows);
    // of the stage whose weights come next: scores in the log2 domain, their largest, and the
    // sum
    float t[16], top, l_stage = 0.0f;
    bool odds = false;  // scales that the store does not write
    // the rows' constants, by way of the wave's own place
    auto row_values = [&](float scale) {
      const B8Value b = b8_value(scale);
      odds = !(scale >= 0x1p-90f && scale < INFINITY);
      rows[n] = scale * qscale;
      rows[32 + n] = b.lv;
      rows[64 + n] = b.iv;
      rows[96 + n] = b.sign;
      asm volatile("" ::: "memory");
    };
    auto row4 = [&](int which, int i) -> w_f4 {  // of rows 8 i + 4 g ..
      return *(lat_cf4)(rows_lds + 128 * which + 32 * i + 16 * g);
    };
    // all weights again, where there are masks, odd scales or another offset
    auto weigh_again = [&](int st, bool edge, char* to) {
      const int rel = (edge ? col_at(ch).pos : 0x7fffffff) - (edge ? st * kStage + 32 * ph + 4 * g : 0);
      l_stage = 0.0f;
      top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const w_f4 iv = row4(2, i);
        float pv[4];
        w_f4 sign = w_f4{1.f, 1.f, 1.f, 1.f};
        if (odds) sign = row4(3, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool on = 8 * i + e <= rel;
          float& x = t[4 * i + e];
          x = on ? x : -INFINITY;
          top = fmaxf(top, x);
          pv[e] = __builtin_amdgcn_exp2f(x - m);
          l_stage = __builtin_fmaf(pv[e], iv[e], l_stage);
          pv[e] = on ? pv[e] * sign[e] : 0.0f;
        }
        *reinterpret_cast<uint2*>(to + 16 * i) =
            make_uint2(pack_pair(pv[0], pv[1], f16{}), pack_pair(pv[2], pv[3], f16{}));
      }
    };
    lat_f16 sv, srv;
    w_u4 k[KW], kp[RS];
    float scale;
    w_f4 sq[4], lv[4], iv[4];
    auto scores_ahead = [&](uint32_t stage) {
      const uint32_t kr = stage + k_off;
#pragma unroll
      for (int w = 0; w < AHEAD; ++w) k[w] = *(lat_cu4)(kr ^ (32 * w));
      scale = *(const __attribute__((address_space(3))) float*)(stage + L::SCALE + 4 * k_row);
    };
    auto scores = [&](uint32_t stage) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sv[e] = srv[e] = 0.0f;
      const uint32_t kr = stage + k_off, rr = stage + r_off;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        if (w + AHEAD < KW)
          k[w + AHEAD] = *(lat_cu4)(kr ^ (32 * (w + AHEAD)));
        else if (w + AHEAD - KW < RS)
          kp[w + AHEAD - KW] = *(lat_cu4)(rr ^ (32 * (w + AHEAD - KW)));
        sv = mfma32(code_op8<T>(k[w][0], k[w][1]), q[2 * w], sv, T{});
        sv = mfma32(code_op8<T>(k[w][2], k[w][3]), q[2 * w + 1], sv, T{});
        if (w == KW / 2) row_values(scale);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sq[i] = row4(0, i);
        lv[i] = row4(1, i);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < RS; ++i) srv = mfma32(kp[i], qr[i], srv, T{});
    };
    // (In one run of instructions with the products: behind a branch the compiler has not always
    // kept the distance that their results need.)
    auto weigh = [&](char* to) {
      top = -INFINITY;
      l_stage = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& x = t[4 * i + e];
          x = __builtin_fmaf(sv[4 * i + e], sq[i][e],
                             __builtin_fmaf(srv[4 * i + e], qscale, lv[i][e]));
          top = fmaxf(top, x);
        }
        iv[i] = row4(2, i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float pv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[e] = __builtin_amdgcn_exp2f(t[4 * i + e] - m);
          l_stage = __builtin_fmaf(pv[e], iv[i][e], l_stage);
        }
        *reinterpret_cast<uint2*>(to + 16 * i) =
            make_uint2(pack_pair(pv[0], pv[1], f16{}), pack_pair(pv[2], pv[3], f16{}));
      }
    };
    // masks, and whether a maximum has outgrown its offset
    auto settle = [&](int st, char* to) {
      const bool edge = is_edge(st);
      odds = __any(odds);
      if (edge || odds) weigh_again(st, edge, to);
      const bool grown = __any(top - m > kRaise + kOutgrow);
      if (lane == 0) flags[st % 2 * 4 + w4] = grown;
    };

    lds_barrier();  // the first stage
    {
      scores_ahead(stage_at(0));
      scores(stage_at(0));
      char* const to = p_write + s0 % 2 * L::PBUF;
      weigh(to);
      settle(s0, to);
    }
    int at = 0;  // the stage's place in the ring
    for (int st = s0; st < s1; ++st) {
      lds_barrier();  // the weights are there, and the next stage
      const int next = st + 1 < s1 ? stage_after(at) : at;
      scores_ahead(stage_at(next));
      if (outgrown(st)) {
        const float mx = max_halves(top);
        if (g == 0) smax[2 * (32 * ch + n) + ph] = mx;
        lds_barrier();
        const float m_new = moved(ch, m);
        l *= __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        weigh_again(st, is_edge(st), p_write + st % 2 * L::PBUF);
        lds_barrier();
      }
      l += l_stage;
      if (is_edge(st)) lds_barrier();  // NaN codes are out of the values
      if (st + 1 < s1) {
        scores(stage_at(next));
        char* const to = p_write + (st + 1) % 2 * L::PBUF;
        weigh(to);
        settle(st + 1, to);
      }
      at = next;
    }
    lds_barrier();  // the maxima's place is read
    const float sum = sum_halves(l);
    if (g == 0) smax[2 * (32 * ch + n) + ph] = sum;
    lds_barrier();
    return;
  }

  // ---- values ----
  {
    const int64_t slot = slot_of(s0, page_of(s0));
#pragma unroll
    for (int j = 0; j < DMAS; ++j) issue(j, slot, stage_at(0));
  }
  if (s0 + 1 < s1) {
    const int64_t slot = slot_of(s0 + 1, page_of(s0 + 1));
#pragma unroll
    for (int j = 0; j < DMAS; ++j) issue(j, slot, stage_at(1));
    wait_vmcnt<DMAS>();
  } else {
    wait_vmcnt<0>();
  }
  lds_barrier();  // the first stage
  int64_t page = page_of(min(s0 + 2, s1 - 1));
  float m[2] = {kNone, kNone};
  lat_f16 o[DB][2];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][x][e] = 0.0f;
  const uint32_t v_row = 8 * g + n % 16 / 2;
  const uint32_t v_off = v_row * R + 16 * ((R / 64 * w4 + n / 16) ^ v_row) + 8 * (n % 2);
  const uint32_t p_read = lds0 + L::P + n * L::PROW + 16 * g;
  int at = 0;
  for (int st = s0; st < s1; ++st) {
    wait_vmcnt<0>();  // this wave's part of the next stage
    lds_barrier();    // everybody's; and the weights are there
    if (outgrown(st)) {
      lds_barrier();
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float m_new = moved(x, m[x]);
        const float alpha = __builtin_amdgcn_exp2f(m[x] - m_new);
        m[x] = m_new;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d][x] *= alpha;
      }
      lds_barrier();
    }
    if (is_edge(st)) {  // NaN codes count as zeros in the values
      char* const codes = lds + at * L::STAGE + w4 * 16 * R;
#pragma unroll
      for (int j = 0; j < CODE_DMAS; ++j) {
        w_u4* p = reinterpret_cast<w_u4*>(codes + j * 1024 + 16 * lane);
        w_u4 w = *p;
        const uint32_t odd = nan_codes(w[0]) | nan_codes(w[1]) | nan_codes(w[2]) | nan_codes(w[3]);
        if (odd) {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] &= ~((nan_codes(w[k]) >> 7) * 0xffu);
          *p = w;
        }
      }
      lds_barrier();
    }
    const bool more = st + 2 < s1;
    const int64_t slot = slot_of(min(st + 2, s1 - 1), page);
    const uint32_t to = stage_at(stage_after(stage_after(at)));
    const uint32_t vr = stage_at(at) + v_off, pr = p_read + st % 2 * L::PBUF;
    // the reads run ahead, past the DMA instructions between
    constexpr int STEPS = PK * DB, VA = 4;
    static_assert(DMAS <= 2 * STEPS, "DMA instructions between the steps");
    auto v_at = [&](int j) {
      return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (lat_lds2)((vr ^ (32 * (j % DB))) + 16 * (j / DB) * R));
    };
    w_u4 p[2][2];
    lat_i2 b[STEPS];
#pragma unroll
    for (int x = 0; x < 2; ++x) p[0][x] = *(lat_cu4)(pr + 32 * x * L::PROW);
#pragma unroll
    for (int j = 0; j < VA; ++j) b[j] = v_at(j);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int kk = j / DB, d = j % DB;
      if (j + VA < STEPS) b[j + VA] = v_at(j + VA);
      if (d == 0 && kk + 1 < PK) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          p[(kk + 1) % 2][x] = *(lat_cu4)(pr + 32 * x * L::PROW + 32 * (kk + 1));
      }
      const w_u4 a = code_op8<f16>(static_cast<uint32_t>(b[j][0]), static_cast<uint32_t>(b[j][1]));
#pragma unroll
      for (int x = 0; x < 2; ++x) o[d][x] = mfma32(a, p[kk % 2][x], o[d][x], f16{});
      if (more) {
        issue(j, slot, to);
        issue(j + STEPS, slot, to);
      }
    }
    at = stage_after(at);
    // (a scalar load in flight would make every wait for LDS one for all of it)
    page = page_of(min(st + 3, s1 - 1));
  }
  lds_barrier();
  lds_barrier();  // the sums are there

  // ---- results: o[d][x][e] is dim R/4 wave + 32 d + 8 (e / 4) + 4 g + e % 4 of the column ----
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const Col y = col_at(x);
    if (!y.live) continue;
    const w_f2 halves = *reinterpret_cast<const w_f2*>(smax + 2 * (32 * x + n));
    const float sum = halves[0] + halves[1];
    const int dim = R / 4 * w4 + 4 * g;
    if (r.parts > 1) {
      const int64_t part = r.part0 + (static_cast<int64_t>(seg) * r.n + y.row) * heads + y.head;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<w_f4*>(parts.o + part * R + dim + 32 * d + 8 * i) =
              w_f4{o[d][x][4 * i], o[d][x][4 * i + 1], o[d][x][4 * i + 2], o[d][x][4 * i + 3]};
      if (g == 0 && w4 == 0)  // a NaN score leaves m without it, but not l
        *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{sum != sum    ? INFINITY
                                                            : sum == 0.0f ? -INFINITY
                                                                          : m[x],
                                                            sum};
      continue;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* dst = out + ((static_cast<int64_t>(r.q0) + y.row) * heads + y.head) * R + dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = pack_pair(o[d][x][4 * i] * inv, o[d][x][4 * i + 1] * inv, T{});
        const uint32_t hi = pack_pair(o[d][x][4 * i + 2] * inv, o[d][x][4 * i + 3] * inv, T{});
        T* to = dst + 32 * d + 8 * i;
        if (wide & 2) {
          *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
        } else {
          uint16_t* d16 = reinterpret_cast<uint16_t*>(to);
          d16[0] = static_cast<uint16_t>(lo);
          d16[1] = static_cast<uint16_t>(lo >> 16);
          d16[2] = static_cast<uint16_t>(hi);
          d16[3] = static_cast<uint16_t>(hi >> 16);
        }
      }
  }
}

// ---- host -----------------------------------------------------------------------

constexpr LatentShape kShape{false, kCols, kStage, 6, 4, 6000000};

}  // namespace

namespace kvq {

int64_t latent_tile_bytes(const LatentCall& call, int* rc) {
  int64_t most = 0;
  *rc = latent_launches(call, kShape, [&](const WinArg&, int, int64_t, int64_t rows) -> int {
    most = std::max(most, win_parts_bytes(rows, call.cache.d));
    return KVQ_OK;
  });
  return most;
}

int latent_tile_attend(const LatentCall& call, void* workspace) {
  const WinCall& win = call.win;
  const LatentCache& c = call.cache;
  const int wide = (win.q_wide() ? 1 : 0) | (aligned16(win.out, nullptr) ? 2 : 0);
  return latent_launches(call, kShape, [&](const WinArg& arg, int count, int64_t units, int64_t rows) -> int {
    const WinParts parts{static_cast<float*>(workspace),
                         static_cast<float*>(workspace) + rows * c.d};
#define KVQ_LATENT(T, R, P)                                                                    \
  hipLaunchKernelGGL((latent_tile_kernel<T, R, P>), dim3(static_cast<unsigned>(units)),      \
                     dim3(64 * kWaves), (LatLds<R, P>::BYTES), win.stream, arg, count, c,      \
                     static_cast<const T*>(win.query), win.q_stride, wide, win.qscale,         \
                     static_cast<T*>(win.out), parts)
#define KVQ_LATENT_P(T, R)      \
  if (c.part == 64)             \
    KVQ_LATENT(T, R, 64);       \
  else                          \
    KVQ_LATENT(T, R, 32)
#define KVQ_LATENT_R(T)         \
  if (c.d == 512) {             \
    KVQ_LATENT_P(T, 512);       \
  } else {                      \
    KVQ_LATENT_P(T, 256);       \
  }
    if (win.dtype == KVQ_DTYPE_BF16) {
      KVQ_LATENT_R(bf16)
    } else {
      KVQ_LATENT_R(f16)
    }
#undef KVQ_LATENT_R
#undef KVQ_LATENT_P
#undef KVQ_LATENT
    KVQ_LAUNCH_CHECK();
    return rows > 0 ? launch_win_join(win, arg, count, parts) : KVQ_OK;
  });
}

}  // namespace kvq
