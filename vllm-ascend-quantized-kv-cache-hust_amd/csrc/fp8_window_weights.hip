// SPDX-License-Identifier: Apache-2.0
// Running attention weights of paged E4M3 positions, after the attention has left
// each (row, head)'s log-sum-exp: w_j += sum over rows and heads of 2^(t_j - lse).
//
// A wave holds the keys of 64 positions as score operands in registers, exact, the
// four waves of a workgroup 256 of one kv head, and the columns (row, head) of the
// head's group go through them 16 at a time:
//   S^T = K * Q^T (lane (g, n): bytes 64 w + 16 g .. of position n of a 16-position
//   group, so k-step 2 w + x takes dims 64 w + 16 g + 8 x ..), p = exp2(fma(S, ks', -lse)),
// summing p over columns in the lane, fp32; the 16 lanes of a position are added at
// the end.  Every position belongs to one wave and is summed in a fixed order.  Columns
// arrive in LDS by DMA, some groups ahead, for all four waves.
//
// Few columns: each code is read once, bound by HBM (keys only).  Many: bound by what a
// wave issues, vector work half of the time and matrix work a third of it, one after the
// other (3 prompts of 1.5K - 4.1K, 32 heads on 8 of 128: 158 us, of which the exponentials,
// one per (row, head, position), are a quarter by count).  The first positions are seen by every
// row and the last by few, so many columns are cut into segments, whose sums meet in
// win_weights_add_kernel.
//
// Requests of fewer than kScoreCols columns: from the scores their decode left
// (win_weights_scores_kernel), 4 bytes a column and position instead of the key.
#include <algorithm>

#include "fp8_window.h"

namespace {

using namespace kvq;

constexpr int kWaves = 4;
constexpr int kGroups = 4;                   // 16-position groups of a wave
constexpr int kSpan = 16 * kGroups * kWaves;  // positions of a workgroup
// Column groups of a segment, and workgroups of a request past which it is cut no
// further (long prompts have spans enough, and the sums would not stay small).  16, 64
// and 128 groups measured 5, 2 and 6% more on 3 prompts of 1.5K - 4.1K, 32 heads on 8.
constexpr int kSegTiles = 32;
constexpr int64_t kSegUnits = 8192;
// Column groups under way or in use, and the bytes of one: 16 rows of the query (16-byte
// column x of row c at x ^ c % 16, or % 8), then their log-sum-exps, a copy per wave.
template <int D>
constexpr int wgt_bufs() { return D == 256 ? 3 : 4; }
template <int D>
constexpr int wgt_buf_bytes() { return 32 * D + kWaves * 256; }
// DMA instructions of a wave and column group
template <int D>
constexpr int wgt_dmas() { return (D == 256 ? 2 : 1) + 1; }

typedef const __attribute__((address_space(4))) int32_t wgt_ci32;
typedef const __attribute__((address_space(4))) int64_t wgt_ci64;

// x summed over the 16 lanes of a row of lanes, in every one of them.
__device__ __forceinline__ float sum_row16(float x) {
  x += dpp_f32<kDppQuadXor1>(x);
  x += dpp_f32<kDppQuadXor2>(x);
  x += dpp_f32<kDppHalfMirror>(x);
  x += dpp_f32<kDppRowMirror>(x);
  return x;
}

// Groups of 16 columns with rows that may see a position of [j0, j0 + run): [lo, hi).
__device__ __forceinline__ void seeing_tiles(const WinReq& r, const WinCache& c, int j0, int run,
                                             int& lo, int& hi) {
  const int rep = static_cast<int>(c.rep.d), base = r.len - r.n;
  const int j1 = min(j0 + run, r.len);
  const int row_lo = max(j0 - base, 0);
  int row_hi = r.n;
  if (c.window != kNoWindow && j0 >= c.sinks) {
    // the last position to see j1 - 1 is j1 - 2 + window
    const int64_t last = static_cast<int64_t>(j1) - 1 + c.window - base;
    row_hi = static_cast<int>(last < r.n ? (last < 0 ? 0 : last) : r.n);
  }
  lo = row_lo * rep / 16;
  hi = (row_hi * rep + 15) / 16;
}

// Column groups of each of a request's segments.
__device__ __forceinline__ int seg_tiles(const WinReq& r, const WinCache& c) {
  const int tiles = (r.n * static_cast<int>(c.rep.d) + 15) / 16;
  return (tiles + r.parts - 1) / r.parts;
}

// A unit is a span of positions of one kv head (and a segment of their columns, of
// r.parts).
template <typename T, int D>
__global__ void __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(D == 256 ? 2 : D == 128 ? 3 : 4, D == 256 ? 2 : D == 128 ? 3 : 4)))
win_weights_kernel(WinArg, int count, WinCache c, const T* __restrict__ query, int64_t q_stride,
                   int wide, float qscale, const float* __restrict__ lse, const float* w_in,
                   float* w_out, int64_t w_cols, float* __restrict__ seg_sums) {
  constexpr int KS = D / 32, W = D / 64, NB = wgt_bufs<D>(), BYTES = wgt_buf_bytes<D>();
  constexpr int PPR = D / 8, RPI = 64 / PPR;  // 16-byte columns of a row, rows of a DMA
  __shared__ __align__(16) char bufs[NB * BYTES];
  __shared__ __align__(16) float s_sum[kSpan];
  const WinReq r = win_req(count, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh;
  u /= c.kvh;
  const int spans = (r.len + kSpan - 1) / kSpan;
  const int seg = u / spans;
  const int span0 = (u - seg * spans) * kSpan;
  const int j0 = span0 + 16 * kGroups * wave;  // the wave's first position
  const int rep = static_cast<int>(c.rep.d);
  const int cols = r.n * rep, base = r.len - r.n;
  int t_lo, t_hi;
  seeing_tiles(r, c, span0, kSpan, t_lo, t_hi);
  if (r.parts > 1) {
    const int per = seg_tiles(r, c);
    t_lo = max(t_lo, seg * per);
    t_hi = min(t_hi, (seg + 1) * per);
    if (t_lo >= t_hi) return;  // uniform over the workgroup
  }
  w_f4 acc[kGroups];
#pragma unroll
  for (int k = 0; k < kGroups; ++k) acc[k] = w_f4{0.f, 0.f, 0.f, 0.f};
  if (t_lo < t_hi) {  // uniform over the workgroup
    // ---- columns on their way ----
    const uint32_t lds0 = win_lds(bufs);
    auto swz = [](int col) { return col % (PPR < 16 ? PPR : 16); };
    // offset of column `col`'s query row, and its log-sum-exp's index
    auto column = [&](int col, int64_t& at) -> int64_t {
      const int x = min(col, cols - 1);  // (columns past the last see nothing)
      const int row = static_cast<int>(c.rep.div(static_cast<uint32_t>(x)));
      const int head = h * rep + x - row * rep;
      at = (static_cast<int64_t>(r.q0) + row) * c.hq + head;
      return (static_cast<int64_t>(r.q0) + row) * q_stride + static_cast<int64_t>(head) * D;
    };
    constexpr int INSTS = 16 / RPI;  // DMAs of the rows: waves 0 and 1 have a double at D = 64
    // where 16 columns are whole rows, a group's addresses are the group before's plus a
    // constant, and a lane's offset from them stays the same
    const bool regular = (wide & 1) && 16 % rep == 0 && q_stride < (1 << 24);  // uniform
    constexpr int PER_WAVE = (INSTS + kWaves - 1) / kWaves;
    uint32_t lane_off[PER_WAVE], lane_lse;
    const char* row_base = nullptr;
    const float* lse_base = nullptr;
    int64_t row_step = 0, lse_step = 0;
    if (regular) {
#pragma unroll
      for (int k = 0; k < PER_WAVE; ++k) {
        const int col = RPI * ((kWaves * k + wave) % INSTS) + lane / PPR;
        const int row = static_cast<int>(c.rep.div(static_cast<uint32_t>(col)));
        lane_off[k] = 2u * (static_cast<uint32_t>(row) * static_cast<uint32_t>(q_stride) +
                            static_cast<uint32_t>(col - row * rep) * D) +
                      16u * ((lane % PPR) ^ swz(col));
      }
      const int row = static_cast<int>(c.rep.div(static_cast<uint32_t>(n)));
      lane_lse = 4u * static_cast<uint32_t>(row * c.hq + n - row * rep);
      const int64_t row0 = r.q0 + static_cast<int64_t>(t_lo) * (16 / rep);
      row_base = reinterpret_cast<const char*>(query + row0 * q_stride +
                                               static_cast<int64_t>(h) * rep * D);
      lse_base = lse + row0 * c.hq + h * rep;
      row_step = 2 * (16 / rep) * q_stride;
      lse_step = (16 / rep) * c.hq;
    }
    // (called for t_lo, t_lo + 1, .. in turn)
    auto issue = [&](int t, int b) {
      if (regular && 16 * t + 15 < cols) {  // uniform
#pragma unroll
        for (int k = 0; k < PER_WAVE; ++k)
          win_dma16(row_base, lane_off[k],
                    lds0 + b * BYTES + 1024 * ((kWaves * k + wave) % INSTS));
        win_dma4(lse_base, lane_lse, lds0 + b * BYTES + 32 * D + 256 * wave);
        row_base += row_step;
        lse_base += lse_step;
        return;
      }
      int64_t at;
#pragma unroll
      for (int k = 0; k < PER_WAVE; ++k) {
        const int i = (kWaves * k + wave) % INSTS;
        const int col = RPI * i + lane / PPR, x = (lane % PPR) ^ swz(col);
        const T* src = query + column(16 * t + col, at) + 8 * x;
        if (wide & 1) {
          const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds0 + b * BYTES + 1024 * i);
          asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                       :
                       : "v"(src), "{m0}"(m0)
                       : "memory");
        } else {
          *reinterpret_cast<w_u4*>(bufs + b * BYTES + 1024 * i + 16 * lane) = load_op8(src, false);
        }
      }
      column(16 * t + n, at);
      const uint32_t m0 =
          __builtin_amdgcn_readfirstlane(lds0 + b * BYTES + 32 * D + 256 * wave);
      asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off"
                   :
                   : "v"(lse + at), "{m0}"(m0)
                   : "memory");
    };

    // ---- keys ----
    w_u4 key[kGroups][KS];
    w_f4 ks[kGroups];
    {
      w_u4 raw[kGroups][W];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        // groups past the end read the last one (masked)
        const int p = min(j0 + 16 * k, (r.len - 1) & ~15);
        const uint32_t pg = c.bs.div(static_cast<uint32_t>(p));
        const int64_t e = static_cast<int64_t>(r.table) * c.maxb +
                          __builtin_amdgcn_readfirstlane(static_cast<int>(
                              static_cast<int64_t>(pg) < c.maxb ? static_cast<int64_t>(pg)
                                                                : c.maxb - 1));
        const int64_t id = c.bt64 ? ((wgt_ci64*)(const void*)c.table)[e]
                                  : static_cast<int64_t>(((wgt_ci32*)(const void*)c.table)[e]);
        const int64_t page = id < 0 ? 0 : (id >= c.nb ? c.nb - 1 : id);
        const int64_t row = (page * c.bs.d + (static_cast<uint32_t>(p) - pg * c.bs.d)) * c.kvh + h;
        const uint32_t lane_row = static_cast<uint32_t>(n * c.kvh);
#pragma unroll
        for (int w = 0; w < W; ++w)
          raw[k][w] = *reinterpret_cast<const w_u4*>(c.kd + row * D + lane_row * D + 64 * w +
                                                     16 * kg);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ks[k][i] = (c.ks + row)[static_cast<uint32_t>((4 * kg + i) * c.kvh)];
      }
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          key[k][2 * w] = code_op8<T>(raw[k][w][0], raw[k][w][1]);
          key[k][2 * w + 1] = code_op8<T>(raw[k][w][2], raw[k][w][3]);
        }
        ks[k] *= qscale;
      }
    }
    // landed: from here on only the DMAs are outstanding
#pragma unroll
    for (int k = 0; k < kGroups; ++k) asm volatile("" : "+v"(ks[k]));
    wait_vmcnt<0>();
#pragma unroll
    for (int b = 0; b < NB - 1; ++b)
      if (t_lo + b < t_hi) issue(t_lo + b, b);

    // groups that see some of the wave's positions, and those that see all of them
    constexpr int RUN = 16 * kGroups;
    int s_lo = t_hi, s_hi = t_hi;
    if (j0 < r.len) seeing_tiles(r, c, j0, RUN, s_lo, s_hi);
    int w_lo = t_hi, w_hi = t_hi;
    if (j0 + RUN <= r.len) {
      // row(16 t) >= j0 + RUN - 1 - base, 16 t + 15 < cols, row(16 t + 15) < j0 + window - base
      w_lo = (max(j0 + RUN - 1 - base, 0) * rep + 15) / 16;
      w_hi = cols / 16;
      if (c.window != kNoWindow && j0 + RUN - 1 >= c.sinks) {
        const int64_t last = static_cast<int64_t>(j0) + c.window - base;  // rows before it
        w_hi = static_cast<int>(min(static_cast<int64_t>(w_hi), last <= 0 ? 0 : last * rep / 16));
      }
    }
    int buf = 0;
    for (int t = t_lo; t < t_hi; ++t) {
      if (t + NB - 2 < t_hi && (wide & 1)) {
        wait_vmcnt<(NB - 2) * wgt_dmas<D>()>();
      } else {
        wait_vmcnt<0>();
      }
      // group t is in LDS, and every wave is done with group t - 1, whose place the next
      // DMA takes
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (t + NB - 1 < t_hi) issue(t + NB - 1, buf == 0 ? NB - 1 : buf - 1);
      const char* cb = bufs + buf * BYTES;
      buf = buf + 1 == NB ? 0 : buf + 1;
      if (t < s_lo || t >= s_hi) continue;  // uniform over the wave
      const bool whole = t >= w_lo && t < w_hi;
      w_u4 q[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i)
        q[i] = *reinterpret_cast<const w_u4*>(
            cb + n * (2 * D) + 16 * ((8 * (i / 2) + 2 * kg + i % 2) ^ swz(n)));
      const float off = *reinterpret_cast<const float*>(cb + 32 * D + 256 * wave + 4 * n);
      w_f4 s[kGroups];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) s[k] = w_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int k = 0; k < kGroups; ++k) s[k] = mfma_op(key[k][i], q[i], s[k], T{});
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[k][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][e], ks[k][e], -off));
      if (!whole) {
        asm volatile("");  // a branch
        const int pos =
            16 * t + n < cols
                ? base + static_cast<int>(c.rep.div(static_cast<uint32_t>(16 * t + n)))
                : -1;
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[k][e] = c.sees(pos, j0 + 16 * k + 4 * kg + e) ? s[k][e] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kGroups; ++k) acc[k] += s[k];
    }
  }
  // lane 0 of each 16 leaves positions 16 k + 4 kg + e
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    w_f4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = sum_row16(acc[k][e]);
    if (n == 0) *reinterpret_cast<w_f4*>(s_sum + 16 * kGroups * wave + 16 * k + 4 * kg) = x;
  }
  __syncthreads();
  const int j = span0 + static_cast<int>(threadIdx.x);
  static_assert(kSpan == 64 * kWaves, "a thread a position");
  if (j >= r.len) return;
  const float sum = s_sum[threadIdx.x];
  if (r.parts > 1) {
    seg_sums[r.part0 + (static_cast<int64_t>(seg) * c.kvh + h) * r.len + j] = sum;
  } else {
    const int64_t at = (static_cast<int64_t>(r.wrow) * c.kvh + h) * w_cols + j;
    w_out[at] = (j < base ? w_in[at] : 0.0f) + sum;
  }
}

// The segments' sums of a position, in their order.  A unit is a span of a head.
__global__ void __launch_bounds__(kSpan)
win_weights_add_kernel(WinArg, int count, WinCache c, const float* w_in, float* w_out,
                       int64_t w_cols, const float* __restrict__ seg_sums) {
  const WinReq r = win_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh, span0 = u / c.kvh * kSpan;
  const int j = span0 + static_cast<int>(threadIdx.x);
  if (j >= r.len) return;
  int lo, hi;
  seeing_tiles(r, c, span0, kSpan, lo, hi);
  float sum = 0.0f;
  const int per = seg_tiles(r, c);
  for (int s = lo / per; s * per < hi; ++s)
    sum += seg_sums[r.part0 + (static_cast<int64_t>(s) * c.kvh + h) * r.len + j];
  const int64_t at = (static_cast<int64_t>(r.wrow) * c.kvh + h) * w_cols + j;
  w_out[at] = (j < r.len - r.n ? w_in[at] : 0.0f) + sum;
}

// From the decode's scores.  A unit is 1024 positions of one kv head, four a thread.
constexpr int kScoreSpan = 1024;
__global__ void __launch_bounds__(256)
win_weights_scores_kernel(WinArg, int count, WinCache c, const float* __restrict__ lse,
                          const float* __restrict__ scores, const float* w_in, float* w_out,
                          int64_t w_cols) {
  const WinReq r = win_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh, j0 = u / c.kvh * kScoreSpan + 4 * static_cast<int>(threadIdx.x);
  if (j0 >= r.len) return;
  const int rep = static_cast<int>(c.rep.d), cols = r.n * rep, base = r.len - r.n;
  const int64_t padded = (r.len + 15) & ~15;
  // part0: where the request's scores are, in units of 16
  const float* src = scores + 16 * static_cast<int64_t>(r.part0) + h * cols * padded + j0;
  w_f4 sum = w_f4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < r.n; ++i) {
    const float* off = lse + (static_cast<int64_t>(r.q0) + i) * c.hq + h * rep;
    bool on[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) on[e] = c.sees(base + i, j0 + e);
    if (!(on[0] || on[1] || on[2] || on[3])) continue;  // (their scores may be unwritten)
    for (int k = 0; k < rep; ++k) {
      const w_f4 t = *reinterpret_cast<const w_f4*>(src + (i * rep + k) * padded);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(t[e] - off[k]);
        sum[e] += on[e] ? p : 0.0f;
      }
    }
  }
  const int64_t at = (static_cast<int64_t>(r.wrow) * c.kvh + h) * w_cols + j0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j0 + e < r.len) w_out[at + e] = (j0 + e < base ? w_in[at + e] : 0.0f) + sum[e];
}

}  // namespace

namespace kvq {

bool win_weights_takes(const WinCall& call, int64_t b) {
  const WinCache& c = call.cache;
  return win_matrix_geometry(call.dtype, c.hq, c.kvh, c.d, static_cast<int>(c.bs.d)) &&
         aligned16(c.kd, c.vd) && call.lens[b] > 0;
}

namespace {

template <typename G>
int wgt_launches(const WinCall& call, const WinScores& scores, G&& go) {
  const WinCache& c = call.cache;
  return win_launches(
      call,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        if (!win_weights_takes(call, b) || (scores.on && win_decode_scores(call, b))) return false;
        const int64_t tiles = (call.qlens[b] * c.rep.d + 15) / 16;
        const int64_t spans = (call.lens[b] + kSpan - 1) / kSpan * c.kvh;
        parts = std::min((tiles + kSegTiles - 1) / kSegTiles,
                         std::max<int64_t>(1, kSegUnits / spans));
        units = spans * parts;
        rows = parts > 1 ? parts * c.kvh * call.lens[b] : 0;
        return true;
      },
      go);
}

}  // namespace

int64_t win_weights_bytes(const WinCall& call, const WinScores& scores, int* rc) {
  int64_t most = 0;
  *rc = wgt_launches(call, scores, [&](const WinArg&, int, int64_t, int64_t rows) -> int {
    most = std::max(most, rows * static_cast<int64_t>(sizeof(float)));
    return KVQ_OK;
  });
  return most;
}

int win_weights(const WinCall& call, const WinScores& scores, void* workspace) {
  const WinCache& c = call.cache;
  const int wide = call.q_wide() ? 1 : 0;
  float* sums = static_cast<float*>(workspace);
  if (scores.on) {
    int64_t scored = 0;
    const int rc = win_launches(
        call,
        [&](int64_t b, int64_t& units, int64_t&, int64_t&) {
          units = (call.lens[b] + kScoreSpan - 1) / kScoreSpan * c.kvh;
          return win_decode_scores(call, b);
        },
        [&](const WinArg& plan, int count, int64_t units, int64_t) -> int {
          WinArg arg = plan;
          for (int i = 0; i < count; ++i) {
            arg.r[i].part0 = static_cast<int32_t>(scored);
            scored += win_score_units(call, arg.r[i].table);
          }
          hipLaunchKernelGGL(win_weights_scores_kernel, dim3(static_cast<unsigned>(units)),
                             dim3(256), 0, call.stream, arg, count, c, call.lse, call.scores,
                             call.w_in, call.w_out, call.w_cols);
          KVQ_LAUNCH_CHECK();
          return KVQ_OK;
        });
    if (rc != KVQ_OK) return rc;
  }
  return wgt_launches(call, scores, [&](const WinArg& arg, int count, int64_t units, int64_t rows) -> int {
#define KVQ_WIN_WGT(T, D)                                                                     \
  hipLaunchKernelGGL((win_weights_kernel<T, D>), dim3(static_cast<unsigned>(units)),          \
                     dim3(64 * kWaves), 0, call.stream, arg, count, c,                        \
                     static_cast<const T*>(call.query), call.q_stride, wide, call.qscale,     \
                     call.lse, call.w_in, call.w_out, call.w_cols, sums)
#define KVQ_WIN_WGT_D(T)                                                                   \
  if (c.d == 64) KVQ_WIN_WGT(T, 64); else if (c.d == 128) KVQ_WIN_WGT(T, 128);             \
  else KVQ_WIN_WGT(T, 256)
    if (call.dtype == KVQ_DTYPE_BF16) {
      KVQ_WIN_WGT_D(bf16);
    } else {
      KVQ_WIN_WGT_D(f16);
    }
#undef KVQ_WIN_WGT_D
#undef KVQ_WIN_WGT
    KVQ_LAUNCH_CHECK();
    if (rows == 0) return KVQ_OK;
    // the requests with several segments, a workgroup per span and head
    WinArg add;
    int n = 0;
    int64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
      if (arg.r[i].parts == 1) continue;
      add.r[n] = arg.r[i];
      add.r[n++].first = static_cast<int32_t>(blocks);
      blocks += (static_cast<int64_t>(arg.r[i].len) + kSpan - 1) / kSpan * c.kvh;
    }
    if (blocks > 0x7fffffff) return KVQ_ERR_INVALID;
    hipLaunchKernelGGL(win_weights_add_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kSpan), 0,
                       call.stream, add, n, c, call.w_in, call.w_out, call.w_cols, sums);
    KVQ_LAUNCH_CHECK();
    return KVQ_OK;
  });
}

}  // namespace kvq
