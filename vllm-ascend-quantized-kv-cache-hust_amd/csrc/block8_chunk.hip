// SPDX-License-Identifier: Apache-2.0
// Attention over pages with block scales for chunks: tiles of 128 or 256 rows (a row is one
// query of one head of a kv head's group), 64-position blocks, bound by the matrix units and
// the softmax beside them.
//
// Four chunks of 2048 rows over 10240 positions, 40 heads on 8 of 128 (1.546 TFLOP): 1630 us,
// 0.95 PFLOP/s, INT8 1687; the vector units are busy for 50% of it, the matrix units for 38%:
// a step converts and stages a block ahead of its products, and the softmax stands between
// them, so that the two kinds of work overlap across the SIMD's two waves only.
// (prefill_attn.hip, whose rows need no conversion and whose softmax runs beside the next
// block's products, reaches 1.0 - 1.15.)
//
// As fp8_window_chunk.hip: one workgroup of four or eight waves (chk_shape) per tile, kv head
// and segment of the tile's blocks.  Codes come from their pages into registers two blocks
// ahead, are converted once per workgroup (exact) and staged in LDS as 16-bit rows, keys in
// the query's type (INT8: in fp16 times 2^-9, bf16 queries raised by a power of two for each
// row into its range), values in fp16:
//   K [64][D]: 16-byte column x of row r at x ^ r % (D / 8), so that the 16 rows a
//     score operand reads sit in different banks;
//   V [64][D]: column x at x ^ (2 (r % 4) + 8 ((r / 4) % 2)) (the second term from
//     D = 128 on), likewise for the transposing reads of the value operand.
// A step converts and stages block i + 1 (or i + 2, ChkLds; loaded a step earlier), sends
// for the block after it, and computes block i; the SIMD's other wave fills its matrix
// units while this one does its softmax.
//
// The scales stay out of the operands: 16 positions share one, so a block has four of each
// side at most, kept beside its rows.  With ks' = k_scale * scale * log2(e), lv =
// log2(v_scale),
//   t = fma(S, ks', lv),  M = running max of t per row, less 7,  p' = 2^(t - M) = p v_scale,
//   O^T += V^T * p'^T (codes in fp16, p' rounded to fp16),
//   l += (sum of p' over the 16) / v_scale in fp32.
// Taking the maximum with the value scale in it keeps p' within fp16's range
// whatever the scales are.  M moves only when a row's maximum outgrows it by 8, so a
// row's largest p' lies between 2^7 and 2^15 (fp16 ends at 2^16): the rounding is 2^-11
// of p' at most, or, where fp16 is subnormal, 2^-32 of the row's largest; what is
// smaller than that counts in l alone, as l takes p' before its rounding.  (fp16 results lie
// up to 1.4 times as far off as their own rounding puts them, bf16 ones 1.01.)  Where t has
// steps of 16 and more, M is the maximum itself.
//
// Positions a row does not see: weights by selection; in blocks that some row does not
// wholly see, NaN codes of values (and rows of a scale that is not finite) are staged as
// zeros, and where some row does see one, a pass behind the others, over those blocks'
// pages, marks what sees them.
#include <algorithm>

#include "block8.h"

namespace {

using namespace kvq;

typedef short c_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) c_s4* c_lds4;

constexpr int kBlock = 64;      // positions
// a row's maximum lies kRaise over its offset M, and up to kOutgrow more before M moves
constexpr float kRaise = 7.0f, kOutgrow = 8.0f;

template <int D>
constexpr int chk_ng() { return D == 256 ? 1 : 2; }  // 16-row column groups of a wave
template <int D, int WAVES>
struct ChkLds {
  // blocks; with four, two steps run between barriers (D = 128: 1.60 for 1.66 ms)
  static constexpr int BUFS = D == 128 && WAVES == 8 ? 4 : 2;
  static constexpr int SIDE = kBlock * D * 2;
  static constexpr int SCALES = 2 * BUFS * SIDE;      // BUFS of [4][4] floats
  static constexpr int FLAG = SCALES + BUFS * 16 * 4;  // a NaN put aside that some row sees
  static constexpr int BYTES = FLAG + 16;
};

typedef const __attribute__((address_space(4))) int32_t chk_ci32;
typedef const __attribute__((address_space(4))) int64_t chk_ci64;

template <typename T, int D, int WAVES, bool INT8>
__global__ void __launch_bounds__(64 * WAVES)
__attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2)))
b8_chunk_kernel(WinArg, int count, B8Cache c, const T* __restrict__ query, int64_t q_stride,
                int wide, float qscale, T* __restrict__ out, WinParts parts) {
  using L = ChkLds<D, WAVES>;
  constexpr int NG = chk_ng<D>(), ROWS = 16 * NG, kTileRows = ROWS * WAVES;
  constexpr int KS = D / 32, DB = D / 16, PPR = D / 8, CH = D / 16;
  constexpr int INS = kBlock * CH / (64 * WAVES);  // 16-byte loads of a lane, block and side
  constexpr int RPI = 64 / CH;                     // rows of a wave's load
  // operands read from LDS one product ahead (D = 128: 1.73 for 1.83 ms; at 256 they
  // would spill, 197 for 100 us)
  constexpr bool AHEAD = D < 256;
  constexpr bool RAISE = INT8 && !std::is_same<T, f16>::value;
  using K = typename std::conditional<INT8, f16, T>::type;
  constexpr float kUnit = INT8 ? 1.0f / kInt8Unit : 1.0f;
  static_assert(INS >= 1 && RPI <= 16, "a wave's load stays inside a 16-position group");
  auto vswz = [](int r) { return 2 * (r % 4) + (PPR >= 16 ? 8 * ((r / 4) % 2) : 0); };
  extern __shared__ __align__(16) char lds[];

  const WinReq r = win_req(count, blockIdx.x);
  const int rep = static_cast<int>(c.rep.d), kvh = c.kvh;
  const int rows = r.n * rep;
  int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % kvh;
  u /= kvh;
  const int seg = u % r.parts;
  const int tiles = (rows + kTileRows - 1) / kTileRows;
  const int tile = tiles - 1 - u / r.parts;  // the longest first
  const int row0 = tile * kTileRows;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, n = lane & 15, kg = lane >> 4;
  auto query_of = [&](int row) { return static_cast<int>(c.rep.div(static_cast<uint32_t>(row))); };
  const int base = r.len - r.n;  // position of the request's first row
  const int last_row = min(row0 + kTileRows, rows) - 1;
  const int tile_first = base + query_of(row0), tile_last = base + query_of(last_row);
  const int wrow0 = row0 + wave * ROWS;
  const int wave_last = min(wrow0 + ROWS, rows) - 1;  // < wrow0: a wave without rows
  const int wave_first_pos = base + query_of(wrow0), wave_last_pos = base + query_of(wave_last);

  // the tile's blocks, of which this workgroup takes [blk0, nblk)
  WinSpan span{0, 0, 0};
  if (tile_last >= 0)
    span = WinSpan::of(tile_last + 1, tile_last - tile_first + 1, c.window, c.sinks, kBlock);
  const int blk0 = static_cast<int>(static_cast<int64_t>(span.groups) * seg / r.parts);
  const int nblk = static_cast<int>(static_cast<int64_t>(span.groups) * (seg + 1) / r.parts);
  auto at_block = [&](int i) { return span.pos(i, kBlock); };

  // the lane's row of column group g, found where it is needed (held, these would cost
  // registers that the blocks lack); a row past the last sees nothing
  struct Row {
    bool live;
    int i, head, pos;
  };
  auto row_at = [&](int g) {
    int row = wrow0 + 16 * g + n;
    asm volatile("" : "+v"(row));  // found anew
    Row x;
    x.live = row < rows;
    x.i = query_of(x.live ? row : 0);
    x.head = h * rep + (x.live ? row : 0) - x.i * rep;
    x.pos = x.live ? base + x.i : -1;
    return x;
  };

  // ---- staging ----
  // where 16-position group `grp` of block i and its scale are, from the table by scalar loads
  const int64_t per_page = c.bs.d / c.group.d;
  struct At {
    int64_t slot, scale;
  };
  auto place = [&](int i, int grp) -> At {
    const int p = at_block(i) + 16 * grp;
    const uint32_t pg = c.bs.div(static_cast<uint32_t>(p));
    const int64_t e = static_cast<int64_t>(r.table) * c.maxb +
                      __builtin_amdgcn_readfirstlane(static_cast<int>(
                          static_cast<int64_t>(pg) < c.maxb ? static_cast<int64_t>(pg)
                                                            : c.maxb - 1));
    const int64_t id = c.bt64 ? ((chk_ci64*)(const void*)c.table)[e]
                              : static_cast<int64_t>(((chk_ci32*)(const void*)c.table)[e]);
    const int64_t page = id < 0 ? 0 : (id >= c.nb ? c.nb - 1 : id);
    const uint32_t in = static_cast<uint32_t>(p) - pg * c.bs.d;
    return At{page * c.bs.d + in, (page * per_page + c.group.div(in)) * kvh + h};
  };
  // load a of this wave: rows RPI * (a * WAVES + wave) .., inside one 16-position group
  const int lrow = lane / CH, lch = lane % CH;
  const uint32_t lane_off = static_cast<uint32_t>(lrow * kvh) * D + 16u * lch;
  // scales by vector loads: a scalar load in flight would hold up every wait for LDS
  uint32_t lane_zero = 0;
  asm volatile("" : "+v"(lane_zero));
  // a block's codes and scales on their way to LDS
  struct Codes {
    w_u4 k[INS], v[INS];
    float ks[INS], vs[INS];
  };
  auto load = [&](int i) {
    Codes x;
#pragma unroll
    for (int a = 0; a < INS; ++a) {
      const int first = RPI * (a * WAVES + wave);
      const At at = place(i, first / 16);
      const int64_t row = (at.slot + first % 16) * kvh + h;
      x.k[a] = *reinterpret_cast<const w_u4*>(c.kd + row * D + lane_off);
      x.v[a] = *reinterpret_cast<const w_u4*>(c.vd + row * D + lane_off);
      x.ks[a] = (c.ks + at.scale)[lane_zero];
      x.vs[a] = (c.vs + at.scale)[lane_zero];
    }
    return x;
  };
  // whether some row of the tile may not see a position of block i
  auto edge = [&](int i) {
    const int p = at_block(i);
    return !(p + kBlock - 1 <= tile_first && (p > tile_last - c.window || p + kBlock - 1 < c.sinks));
  };
  auto put = [&](char* kb, char* vb, int which, int i, const Codes& x) {
    const bool cut = edge(i);  // uniform
#pragma unroll
    for (int a = 0; a < INS; ++a) {
      const int row = RPI * (a * WAVES + wave) + lrow;
      char* p = kb + row * (2 * D);
      *reinterpret_cast<w_u4*>(p + 16 * ((2 * lch) ^ (row % PPR))) =
          b8_op8<K, INT8>(x.k[a][0], x.k[a][1]);
      *reinterpret_cast<w_u4*>(p + 16 * ((2 * lch + 1) ^ (row % PPR))) =
          b8_op8<K, INT8>(x.k[a][2], x.k[a][3]);
      w_u4 v = x.v[a];
      const B8Value scale = b8_value(x.vs[a]);
      const bool lost = scale.sign != scale.sign;  // not finite
      uint32_t flip = 0, nan = 0;                  // of the fp16 pairs
      if (__any(scale.sign != 1.0f)) {             // (none that the store writes)
        flip = scale.sign < 0.0f ? 0x80008000u : 0u;
        nan = lost && !cut ? 0x7fff7fffu : 0u;
        if (scale.sign == 0.0f || (lost && cut)) {
#pragma unroll
          for (int k = 0; k < 4; ++k)  // NaN stays, times 0 too
            v[k] = INT8 || lost ? 0u : v[k] & (nan_codes(v[k]) >> 7) * 0xffu;
        }
      }
      if (cut) {
        uint32_t odd = lost ? 0x80u : 0u;
        if constexpr (!INT8)
          odd |= nan_codes(v[0]) | nan_codes(v[1]) | nan_codes(v[2]) | nan_codes(v[3]);
        const int at = at_block(i) + row;
        if (odd && at <= tile_last && (at > max(tile_first, 0) - c.window || at < c.sinks))
          *reinterpret_cast<uint32_t*>(lds + L::FLAG) = 1;
        if (!INT8 && odd) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] &= ~((nan_codes(v[k]) >> 7) * 0xffu);
        }
      }
      // odd rows store their second column first: the even columns of two rows would
      // share their banks
      p = vb + row * (2 * D);
      const int swap = row & 1;
      const uint32_t y[4] = {swap ? v[2] : v[0], swap ? v[3] : v[1], swap ? v[0] : v[2],
                             swap ? v[1] : v[3]};
      w_u4 z[2] = {b8_op8<f16, INT8>(y[0], y[1]), b8_op8<f16, INT8>(y[2], y[3])};
      if (__any((flip | nan) != 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          z[0][k] = (z[0][k] ^ flip) | nan;
          z[1][k] = (z[1][k] ^ flip) | nan;
        }
      }
      *reinterpret_cast<w_u4*>(p + 16 * ((2 * lch + swap) ^ vswz(row))) = z[0];
      *reinterpret_cast<w_u4*>(p + 16 * ((2 * lch + 1 - swap) ^ vswz(row))) = z[1];
      // of the group whose first row this load holds: [0][.] ks', [1][.] lv, [2][.] 1 / v_scale
      if (RPI * (a * WAVES + wave) % 16 == 0 && lane == 0) {
        float* d = reinterpret_cast<float*>(lds + L::SCALES) + which * 16 + row / 16;
        d[0] = x.ks[a] * (qscale * kUnit);
        d[4] = scale.lv;
        d[8] = scale.iv;
      }
    }
  };

  // a part without blocks, or rows that see nothing
  if (blk0 >= nblk) {  // uniform
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const Row y = row_at(g);
      if (!y.live) continue;
      const int64_t at = (static_cast<int64_t>(r.q0) + y.i) * c.hq + y.head;
      if (r.parts > 1) {
        const int64_t part = r.part0 + (static_cast<int64_t>(seg) * r.n + y.i) * c.hq + y.head;
        if (kg == 0) *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{-INFINITY, 0.0f};
      } else {
        for (int k = kg; k < D; k += 4) out[at * D + k] = from_f32<T>(0.0f);
      }
    }
    return;
  }

  // m of a row that has seen nothing: finite, so that 2^(t - m) needs no test for it
  constexpr float kNone = -0x1p127f;
  float m[NG], l[NG];
  w_f4 o[DB][NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    m[g] = kNone;
    l[g] = 0.0f;
#pragma unroll
    for (int j = 0; j < DB; ++j) o[j][g] = w_f4{0.f, 0.f, 0.f, 0.f};
  }
  w_u4 q[NG][KS];
  float lower[NG];  // what takes the raised queries' scores back
#pragma unroll
  for (int g = 0; g < NG; ++g) lower[g] = 1.0f;

  constexpr int AWAY = L::BUFS / 2;  // steps from a block's staging to its use
  auto kbuf = [&](int b) { return lds + b % L::BUFS * L::SIDE; };
  auto vbuf = [&](int b) { return lds + (L::BUFS + b % L::BUFS) * L::SIDE; };
  auto k_reads = [&](const char* sk, int grp, w_u4 (&a)[KS]) {
    const int row = 16 * grp + n;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      a[s] = *reinterpret_cast<const w_u4*>(sk + row * (2 * D) + 16 * ((4 * s + kg) ^ (row % PPR)));
  };
  auto k_mfmas = [&](const w_u4 (&a)[KS], w_f4 (&acc)[NG]) {
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int g = 0; g < NG; ++g) acc[g] = mfma_op(a[s], q[g][s], acc[g], K{});
  };
  // value operands of k-step ks (positions 32 ks ..), dim blocks DB / 2 * jh ..: lane s
  // of a 16-lane group addresses row keybase + s / 4, dims 16 j + 4 (s % 4) .., and
  // receives positions keybase .. + 3 of dim 16 j + s
  const int tr_row = lane % 16 / 4, tr_chunk = (lane % 4) / 2, tr_half = 8 * (lane % 2);
  auto v_reads = [&](const char* sv, int ks, int jh, w_u4 (&a)[DB / 2]) {
#pragma unroll
    for (int jj = 0; jj < DB / 2; ++jj) {
      const int j = jh * (DB / 2) + jj;
      c_s4 part[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int row = 32 * ks + 16 * hh + 4 * kg + tr_row;
        const int x = (2 * j + tr_chunk) ^ vswz(row);
        part[hh] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (c_lds4)(sv + row * (2 * D) + 16 * x + tr_half));
      }
      const uint2 lo = __builtin_bit_cast(uint2, part[0]), hi = __builtin_bit_cast(uint2, part[1]);
      a[jj] = w_u4{lo.x, lo.y, hi.x, hi.y};
    }
  };
  auto active = [&](int i) { return wrow0 <= wave_last && at_block(i) <= wave_last_pos; };

  if (tid == 0) *reinterpret_cast<uint32_t*>(lds + L::FLAG) = 0;
  __syncthreads();
  // prologue: the first AWAY blocks staged, the next one's codes on their way
  Codes first = load(blk0), next = first;
  if (AWAY > 1 && blk0 + 1 < nblk) next = load(blk0 + 1);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const Row y = row_at(g);
    const T* qrow = query + (static_cast<int64_t>(r.q0) + y.i) * q_stride +
                    static_cast<int64_t>(y.head) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[g][s] = load_op8(qrow + 32 * s + 8 * kg, wide & 1);
    if constexpr (RAISE) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) top = pair_bits_max(top, q[g][s][k]);
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
      const float raise = query_raise(top);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) q[g][s][k] = raised_pair(q[g][s][k], raise);
      lower[g] = 1.0f / raise;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
      if (!y.live) q[g][s] = w_u4{0, 0, 0, 0};
  }
  put(kbuf(0), vbuf(0), 0, blk0, first);
  if (AWAY > 1 && blk0 + 1 < nblk) put(kbuf(1), vbuf(1), 1, blk0 + 1, next);
  if (blk0 + AWAY < nblk) next = load(blk0 + AWAY);
  __syncthreads();

  // Step i, block i in buffer `cur`.
  auto step = [&](int cur, int i) {
    const char *kc = kbuf(cur), *vc = vbuf(cur);
    if (i + AWAY < nblk) put(kbuf(cur + AWAY), vbuf(cur + AWAY), (cur + AWAY) % L::BUFS, i + AWAY, next);
    if (i + AWAY + 1 < nblk) next = load(i + AWAY + 1);
    if (!active(i)) return;
    const int kb = at_block(i);
    const float* sc = reinterpret_cast<const float*>(lds + L::SCALES) + cur * 16;
    // operands are read a group ahead of their products where registers allow
    w_f4 s[4][NG];
    w_u4 a[AHEAD ? 2 : 1][KS];
    if (AHEAD) k_reads(kc, 0, a[0]);
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!AHEAD) k_reads(kc, k, a[0]);
      if (AHEAD && k < 3) k_reads(kc, k + 1, a[(k + 1) % 2]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < NG; ++g) s[k][g] = w_f4{0.f, 0.f, 0.f, 0.f};
      k_mfmas(a[AHEAD ? k % 2 : 0], s[k]);
    }
    // vector work goes before the other wave's products, which it leaves gaps for (2 - 3%
    // at head sizes 128 and 256; the other way round, nothing)
    __builtin_amdgcn_s_setprio(1);
    const w_f4 ks = *reinterpret_cast<const w_f4*>(sc), lv = *reinterpret_cast<const w_f4*>(sc + 4);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float a = RAISE ? ks[k] * lower[g] : ks[k];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[k][g][e] = __builtin_fmaf(s[k][g][e], a, lv[k]);
      }
    const bool full = kb + kBlock - 1 <= wave_first_pos &&
                      (kb > wave_last_pos - c.window || kb + kBlock - 1 < c.sinks);  // uniform
    if (!full) {
      asm volatile("");  // a branch, or every block pays the compares
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        // position kb + 16 k + 4 kg + e is seen when 16 k + e <= rel and (> old or < snk)
        const int pos = row_at(g).pos;
        const int rel = pos - kb - 4 * kg;
        const int old = max(pos, 0) - c.window - kb - 4 * kg, snk = c.sinks - kb - 4 * kg;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int x = 16 * (e / 4) + e % 4;
          const bool on = x <= rel && (x > old || x < snk);
          s[e / 4][g][e % 4] = on ? s[e / 4][g][e % 4] : -INFINITY;
        }
      }
    }
    float tmax[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      // med3(a, b, FLT_MAX) = max(a, b) without fmaxf's canonicalizing moves
      constexpr float kBig = 0x1.fffffep127f;
      float ta = __builtin_amdgcn_fmed3f(s[0][g][0], s[0][g][1], kBig);
      float tb = __builtin_amdgcn_fmed3f(s[2][g][0], s[2][g][1], kBig);
#pragma unroll
      for (int e = 2; e < 8; ++e) {
        ta = fmaxf(ta, s[e / 4][g][e % 4]);
        tb = fmaxf(tb, s[2 + e / 4][g][e % 4]);
      }
      tmax[g] = fmaxf(ta, tb);
    }
    if constexpr (NG == 2) {
      max_rows4_pair(tmax[0], tmax[1]);
    } else {
      tmax[0] = max_rows4(tmax[0]);
    }
    bool rescale = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) rescale = rescale || tmax[g] - m[g] > kRaise + kOutgrow;
    if (__any(rescale)) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float mn = tmax[g] - m[g] > kRaise + kOutgrow ? tmax[g] - kRaise : m[g];
        const float alpha = __builtin_amdgcn_exp2f(m[g] - mn);
        l[g] *= alpha;
#pragma unroll
        for (int j = 0; j < DB; ++j) o[j][g] *= alpha;
        m[g] = mn;
      }
    }
    w_u4 p[NG][2], v[AHEAD ? 2 : 1][DB / 2];
    if (AHEAD) v_reads(vc, 0, 0, v[0]);
    const w_f4 iv = *reinterpret_cast<const w_f4*>(sc + 8);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float pv[4], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[e] = __builtin_amdgcn_exp2f(s[k][g][e] - m[g]);
          sum += pv[e];
        }
        l[g] = __builtin_fmaf(sum, iv[k], l[g]);
        p[g][k / 2][2 * (k % 2)] = pack_pair(pv[0], pv[1], f16{});
        p[g][k / 2][2 * (k % 2) + 1] = pack_pair(pv[2], pv[3], f16{});
      }
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // k-step x / 2, half x % 2 of the dims
      if (!AHEAD) v_reads(vc, x / 2, x % 2, v[0]);
      if (AHEAD && x < 3) v_reads(vc, (x + 1) / 2, (x + 1) % 2, v[(x + 1) % 2]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int jj = 0; jj < DB / 2; ++jj)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          w_f4& acc = o[x % 2 * (DB / 2) + jj][g];
          acc = mfma_op(v[AHEAD ? x % 2 : 0][jj], p[g][x / 2], acc, f16{});
        }
    }
    __builtin_amdgcn_s_setprio(1);
  };
  int i = blk0;
  while (i < nblk) {
#pragma unroll
    for (int cur = 0; cur < L::BUFS; ++cur) {
      step(cur, i);
      if (++i >= nblk) break;
      if (cur % AWAY == AWAY - 1) __syncthreads();
    }
  }

  __syncthreads();
  if (*reinterpret_cast<const uint32_t*>(lds + L::FLAG)) {  // uniform
    for (i = blk0; i < nblk; ++i) {
      if (!edge(i)) continue;
      const int kb = at_block(i);
      for (int x = 0; x < kBlock && kb + x <= tile_last; ++x) {
        bool any = false;
#pragma unroll
        for (int g = 0; g < NG; ++g) any = any || c.sees(row_at(g).pos, kb + x);
        if (!__any(any)) continue;
        const At at = place(i, x / 16);
        const int64_t row = (at.slot + x % 16) * kvh + h;
        const uint32_t all = fabsf(c.vs[at.scale]) < INFINITY ? 0u : 0x80808080u;
#pragma unroll
        for (int j = 0; j < DB; ++j) {
          uint32_t odd = all;
          if constexpr (!INT8)
            odd |= nan_codes(*reinterpret_cast<const uint32_t*>(c.vd + row * D + 16 * j + 4 * kg));
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c.sees(row_at(g).pos, kb + x) && (odd >> (8 * e + 7)) & 1) o[j][g][e] = NAN;
        }
      }
    }
  }

  // ---- results: o[j][g][e] is dim 16 j + 4 kg + e of row 16 g + n ----
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float sum = sum_rows4(l[g]);
    const Row y = row_at(g);
    const int64_t at = (static_cast<int64_t>(r.q0) + y.i) * c.hq + y.head;
    if (r.parts > 1) {
      if (!y.live) continue;
      const int64_t part = r.part0 + (static_cast<int64_t>(seg) * r.n + y.i) * c.hq + y.head;
#pragma unroll
      for (int j = 0; j < DB; ++j)
        *reinterpret_cast<w_f4*>(parts.o + part * D + 16 * j + 4 * kg) = kUnit * o[j][g];
      // a NaN score reaches the sum but not the maximum
      if (kg == 0)
        *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{sum != sum    ? INFINITY
                                                                : sum == 0.0f ? -INFINITY
                                                                              : m[g],
                                                              sum};
      continue;
    }
    const float inv = sum == 0.0f ? 0.0f : kUnit / sum;
    T* dst = out + at * D;
    // two dim blocks' 8-byte pieces trade places between 16-lane groups: 16 bytes a lane
#pragma unroll
    for (int j = 0; j < DB; j += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto x = __builtin_amdgcn_permlane16_swap(
            pack_pair(o[j][g][2 * e] * inv, o[j][g][2 * e + 1] * inv, T{}),
            pack_pair(o[j + 1][g][2 * e] * inv, o[j + 1][g][2 * e + 1] * inv, T{}), false, false);
        w[0][e] = x[0];
        w[1][e] = x[1];
      }
      T* d8 = dst + 16 * (j + kg % 2) + 8 * (kg / 2);
      if (!y.live) continue;
      if (wide & 2) {
        *reinterpret_cast<uint4*>(d8) = make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
      } else {
        uint16_t* d16 = reinterpret_cast<uint16_t*>(d8);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t y = w[e / 2][e % 2];
          d16[2 * e] = static_cast<uint16_t>(y);
          d16[2 * e + 1] = static_cast<uint16_t>(y >> 16);
        }
      }
    }
  }
}

// ---- host -----------------------------------------------------------------------

// How a call runs: waves of a workgroup, rows of a tile.
struct ChkShape {
  int waves, rows;
};

int64_t chk_tiles(const B8Call& call, int64_t b, int rows) {
  if (call.win.qlens[b] <= 0 || !b8_chunk_takes(call, b)) return 0;
  return (call.win.qlens[b] * call.cache.rep.d + rows - 1) / rows;
}

// Head size 64: four waves of 32 rows, three workgroups a CU.  256: eight waves of 16.  128:
// eight waves of 32, which convert a block for 256 rows, or four, two workgroups a CU, where
// requests have few columns (row, head) to fill tiles with.
ChkShape chk_shape(const B8Call& call) {
  if (call.cache.d == 256) return {8, 128};
  if (call.cache.d == 64) return {4, 128};
  int64_t cols = 0, requests = 0;
  for (int64_t b = 0; b < call.win.batch; ++b)
    if (chk_tiles(call, b, 256) > 0) {
      cols += call.win.qlens[b] * call.cache.rep.d;
      ++requests;
    }
  return cols >= 512 * requests ? ChkShape{8, 256} : ChkShape{4, 128};
}

// The most blocks that a tile of request b has.
int64_t chk_blocks(const WinCall& win, int64_t b, int tile_rows) {
  const WinCache& c = win.cache;
  const int rows = static_cast<int>(
      std::min<int64_t>(win.qlens[b], (tile_rows + c.rep.d - 2) / c.rep.d + 1));
  return WinSpan::of(static_cast<int>(win.lens[b]), rows, c.window, c.sinks, kBlock).groups;
}

// Segments of a tile's blocks: what ends soonest, in blocks of one workgroup, when `groups`
// workgroups of `blocks` blocks share the CUs (two or more on one overlap to three fifths,
// where it has room for them), each a `segs`th as long, and the partial results (`bytes` of
// them a segment) go through memory and back: 3 blocks and one per 6 MB.
int64_t chk_segs(int64_t groups, int64_t blocks, int64_t cus, bool several, int64_t bytes) {
  auto time = [&](int64_t segs) {
    const int64_t each = (groups * segs + cus - 1) / cus;  // workgroups of a CU
    return each * ((blocks + segs - 1) / segs) * (each > 1 && several ? 3 : 5);
  };
  int64_t best = 1, cost = time(1);  // in fifths of a block
  for (int64_t segs = 2; segs <= 64 && segs * 4 <= blocks; ++segs) {
    const int64_t c = time(segs) + 5 * (3 + segs * bytes / 6000000);
    if (c < cost) {
      best = segs;
      cost = c;
    }
  }
  return best;
}

template <typename G>
int chk_launches(const B8Call& call, G&& go) {
  int cus = 0;
  const int rc = device_cu_count(&cus);
  if (rc != KVQ_OK) return rc;
  if (cus <= 0) cus = 256;
  const WinCall& win = call.win;
  const ChkShape shape = chk_shape(call);
  int64_t tiles = 0, blocks = 0;
  for (int64_t b = 0; b < win.batch; ++b) {
    const int64_t t = chk_tiles(call, b, shape.rows);
    tiles += t;
    if (t > 0) blocks = std::max(blocks, chk_blocks(win, b, shape.rows));
  }
  const int64_t groups = tiles * win.cache.kvh;
  const int64_t segs =
      chk_segs(groups, blocks, cus, shape.waves == 4, groups * shape.rows * win.cache.d * 8);
  return win_launches(
      win,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        const int64_t t = chk_tiles(call, b, shape.rows);
        if (t == 0) return false;
        parts = std::max<int64_t>(1, std::min(segs, chk_blocks(win, b, shape.rows) / 4));
        rows = win_part_rows(win, b, parts);
        units = t * parts * win.cache.kvh;
        return true;
      },
      [&](const WinArg& arg, int count, int64_t units, int64_t rows) -> int {
        return go(shape, arg, count, units, rows);
      });
}

}  // namespace

namespace kvq {

bool b8_chunk_takes(const B8Call& call, int64_t b) {
  return b8_matrix(call) && call.win.lens[b] > 0 && !b8_decode_takes(call, b);
}

int64_t b8_chunk_bytes(const B8Call& call, int* rc) {
  int64_t most = 0;
  *rc = chk_launches(call, [&](const ChkShape&, const WinArg&, int, int64_t, int64_t rows) -> int {
    most = std::max(most, win_parts_bytes(rows, call.cache.d));
    return KVQ_OK;
  });
  return most;
}

int b8_chunk(const B8Call& call, void* workspace) {
  const WinCall& win = call.win;
  const B8Cache& c = call.cache;
  const int wide = (win.q_wide() ? 1 : 0) | (aligned16(win.out, nullptr) ? 2 : 0);
  return chk_launches(call, [&](const ChkShape& shape, const WinArg& arg, int count, int64_t units,
                                int64_t rows) -> int {
    const WinParts parts{static_cast<float*>(workspace),
                         static_cast<float*>(workspace) + rows * c.d};
#define KVQ_B8_CHUNK_I(T, D, W, I)                                                             \
  hipLaunchKernelGGL((b8_chunk_kernel<T, D, W, I>), dim3(static_cast<unsigned>(units)),        \
                     dim3(64 * W), (ChkLds<D, W>::BYTES), win.stream, arg, count, c,           \
                     static_cast<const T*>(win.query), win.q_stride, wide, win.qscale,         \
                     static_cast<T*>(win.out), parts)
#define KVQ_B8_CHUNK(T, D, W)         \
  if (c.int8)                         \
    KVQ_B8_CHUNK_I(T, D, W, true);    \
  else                                \
    KVQ_B8_CHUNK_I(T, D, W, false)
#define KVQ_B8_CHUNK_D(T)             \
  if (c.d == 64) {                    \
    KVQ_B8_CHUNK(T, 64, 4);           \
  } else if (c.d == 256) {            \
    KVQ_B8_CHUNK(T, 256, 8);          \
  } else if (shape.waves == 8) {      \
    KVQ_B8_CHUNK(T, 128, 8);          \
  } else {                            \
    KVQ_B8_CHUNK(T, 128, 4);          \
  }
    if (win.dtype == KVQ_DTYPE_BF16) {
      KVQ_B8_CHUNK_D(bf16)
    } else {
      KVQ_B8_CHUNK_D(f16)
    }
#undef KVQ_B8_CHUNK_D
#undef KVQ_B8_CHUNK
#undef KVQ_B8_CHUNK_I
    KVQ_LAUNCH_CHECK();
    return rows > 0 ? launch_win_join(win, arg, count, parts) : KVQ_OK;
  });
}

}  // namespace kvq
