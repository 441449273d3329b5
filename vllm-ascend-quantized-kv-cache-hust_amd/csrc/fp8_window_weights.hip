// SPDX-License-Identifier: Apache-2.0
// Running attention weights of paged E4M3 positions, after the attention has left
// each (row, head)'s log-sum-exp: w_j += sum over rows and heads of 2^(t_j - lse).
//
// A wave holds the keys of a run of positions (128 of them, 64 at head size 256) as
// score operands in registers, exact, and takes the columns (row, head) of the kv
// head's group through them 16 at a time:
//   S^T = K * Q^T (lane (g, n): bytes D/4 g .. of position n of a 16-position group,
//   so k-step s takes dims D/4 g + 8 s ..), p = exp2(fma(S, ks', -lse)),
// summing p over columns in the lane, fp32; the 16 lanes of a position are added at
// the end.  Every position belongs to one workgroup and is summed in a fixed order.
//
// Few columns: a wave per run, each code read once: bound by HBM (keys only).  Many
// (SPLIT): the four waves of a workgroup share a run and take every fourth column
// group, joined in LDS: bound by the exponentials, one per (row, head, position).  The
// first positions are seen by every row and the last by few, so long requests' columns
// are cut into segments of kSegTiles groups, whose sums meet in win_weights_add_kernel
// (3 prompts of 1.5K - 4.1K, 32 heads on 8: 354 us uncut).
#include <algorithm>

#include "fp8_window.h"

namespace {

using namespace kvq;

constexpr int kWaves = 4;
constexpr int kSplitCols = 64;  // columns from which a workgroup's waves share a run
constexpr int kSegTiles = 128;  // column groups of a segment

template <int D>
constexpr int run_groups() { return D == 256 ? 4 : 8; }

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
  hi = j0 < r.len ? (row_hi * rep + 15) / 16 : 0;
}

// A unit is a workgroup's run(s) of one kv head (and a segment of their columns, of
// r.parts): RUN positions if SPLIT, 4 RUN if not.
template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
win_weights_kernel(WinArg, int count, WinCache c, const T* __restrict__ query, int64_t q_stride,
                   int wide, float qscale, const float* __restrict__ lse, const float* w_in,
                   float* w_out, int64_t w_cols, float* __restrict__ seg_sums) {
  constexpr int NGRP = run_groups<D>(), RUN = 16 * NGRP, KS = D / 32, W = D / 64;
  __shared__ float s_scale[kWaves][RUN];
  __shared__ float s_sum[kWaves][RUN];
  const WinReq r = win_req(count, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh;
  u /= c.kvh;
  constexpr int SPAN = SPLIT ? RUN : kWaves * RUN;
  const int spans = (r.len + SPAN - 1) / SPAN;
  const int seg = u / spans;
  const int wg0 = (u - seg * spans) * SPAN;
  const int j0 = wg0 + (SPLIT ? 0 : wave * RUN);  // the wave's first position
  const int rep = static_cast<int>(c.rep.d);
  const int cols = r.n * rep, base = r.len - r.n;
  int t_lo, t_hi;
  seeing_tiles(r, c, j0, RUN, t_lo, t_hi);
  if (SPLIT && r.parts > 1) {
    t_lo = max(t_lo, seg * kSegTiles);
    t_hi = min(t_hi, (seg + 1) * kSegTiles);
    if (t_lo >= t_hi) return;  // uniform over the workgroup
  }
  float* sums = s_sum[wave];

  w_f4 acc[NGRP];
#pragma unroll
  for (int k = 0; k < NGRP; ++k) acc[k] = w_f4{0.f, 0.f, 0.f, 0.f};
  if (t_lo < t_hi) {  // wave-uniform
    // ---- keys ----
    w_u4 key[NGRP][KS];
    {
      w_u4 raw[NGRP][W];
      float sc[NGRP];
#pragma unroll
      for (int k = 0; k < NGRP; ++k) {
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
          raw[k][w] = *reinterpret_cast<const w_u4*>(c.kd + row * D + lane_row * D + (D / 4) * kg +
                                                     16 * w);
        sc[k] = (c.ks + row)[lane_row];
      }
#pragma unroll
      for (int k = 0; k < NGRP; ++k) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          key[k][2 * w] = code_op8<T>(raw[k][w][0], raw[k][w][1]);
          key[k][2 * w + 1] = code_op8<T>(raw[k][w][2], raw[k][w][3]);
        }
        if (kg == 0) s_scale[wave][16 * k + n] = sc[k] * qscale;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // ---- columns ----
    struct Cols {
      w_u4 q[KS];
      float lse;
      int pos;
    };
    auto load = [&](int t) {
      Cols x;
      const int col = 16 * t + n;
      const bool live = col < cols;
      const int row = static_cast<int>(c.rep.div(static_cast<uint32_t>(live ? col : 0)));
      const int head = h * rep + (live ? col : 0) - row * rep;
      const int64_t at = static_cast<int64_t>(r.q0) + row;
      const T* qrow = query + at * q_stride + static_cast<int64_t>(head) * D + (D / 4) * kg;
#pragma unroll
      for (int s = 0; s < KS; ++s) x.q[s] = load_op8(qrow + 8 * s, wide & 1);
      x.lse = lse[at * c.hq + head];
      x.pos = live ? base + row : -1;
      return x;
    };
    constexpr int STEP = SPLIT ? kWaves : 1;
    int t = t_lo + (SPLIT ? wave : 0);
    Cols now{};
    if (t < t_hi) now = load(t);
    for (; t < t_hi; t += STEP) {
      Cols next = now;
      if (t + STEP < t_hi) next = load(t + STEP);
      const int pos_lo = base + static_cast<int>(c.rep.div(static_cast<uint32_t>(16 * t)));
      const int pos_hi =
          base + static_cast<int>(c.rep.div(static_cast<uint32_t>(min(16 * t + 15, cols - 1))));
      const bool whole = 16 * t + 15 < cols && j0 + RUN <= r.len && j0 + RUN - 1 <= pos_lo &&
                         (j0 > pos_hi - c.window || j0 + RUN - 1 < c.sinks);  // uniform
#pragma unroll
      for (int k = 0; k < NGRP; ++k) {
        w_f4 s = w_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) s = mfma_op(key[k][i], now.q[i], s, T{});
        const w_f4 ks = *reinterpret_cast<const w_f4*>(&s_scale[wave][16 * k + 4 * kg]);
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], ks[e], -now.lse));
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            p[e] = c.sees(now.pos, j0 + 16 * k + 4 * kg + e) ? p[e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[k][e] += p[e];
        if (k % 2) __builtin_amdgcn_sched_barrier(0);  // two groups at a time: registers
      }
      now = next;
    }
  }
  // lane 0 of each 16 leaves positions 16 k + 4 kg + e
#pragma unroll
  for (int k = 0; k < NGRP; ++k) {
    w_f4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = sum_row16(acc[k][e]);
    if (n == 0) *reinterpret_cast<w_f4*>(sums + 16 * k + 4 * kg) = x;
  }
  __syncthreads();
  const int64_t dst = (static_cast<int64_t>(r.wrow) * c.kvh + h) * w_cols;
  for (int x = threadIdx.x; x < (SPLIT ? RUN : kWaves * RUN); x += 64 * kWaves) {
    const int j = wg0 + x;
    if (j >= r.len) break;
    float sum;
    if constexpr (SPLIT) {
      sum = (s_sum[0][x] + s_sum[1][x]) + (s_sum[2][x] + s_sum[3][x]);
      if (r.parts > 1) {
        seg_sums[r.part0 + (static_cast<int64_t>(seg) * c.kvh + h) * r.len + j] = sum;
        continue;
      }
    } else {
      sum = s_sum[x / RUN][x % RUN];
    }
    w_out[dst + j] = (j < base ? w_in[dst + j] : 0.0f) + sum;
  }
}

// The segments' sums of a position, in their order.  A unit is 256 positions of a head.
template <int D>
__global__ void __launch_bounds__(256)
win_weights_add_kernel(WinArg, int count, WinCache c, const float* w_in, float* w_out,
                       int64_t w_cols, const float* __restrict__ seg_sums) {
  const WinReq r = win_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh, j = u / c.kvh * 256 + static_cast<int>(threadIdx.x);
  if (j >= r.len) return;
  constexpr int RUN = 16 * run_groups<D>();
  int lo, hi;
  seeing_tiles(r, c, j / RUN * RUN, RUN, lo, hi);
  float sum = 0.0f;
  for (int s = lo / kSegTiles; s * kSegTiles < hi; ++s)
    sum += seg_sums[r.part0 + (static_cast<int64_t>(s) * c.kvh + h) * r.len + j];
  const int64_t at = (static_cast<int64_t>(r.wrow) * c.kvh + h) * w_cols + j;
  w_out[at] = (j < r.len - r.n ? w_in[at] : 0.0f) + sum;
}

}  // namespace

namespace kvq {

bool win_weights_takes(const WinCall& call, int64_t b) {
  const WinCache& c = call.cache;
  return win_matrix_geometry(call.dtype, c.hq, c.kvh, c.d, static_cast<int>(c.bs.d)) &&
         aligned16(c.kd, c.vd) && call.lens[b] > 0;
}

namespace {

// Launches of the requests whose columns a workgroup's waves share, or of the others.
template <typename G>
int wgt_launches(const WinCall& call, int split, G&& go) {
  const WinCache& c = call.cache;
  const int64_t run = 16 * (c.d == 256 ? 4 : 8) * (split ? 1 : kWaves);
  return win_launches(
      call,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        const int64_t cols = call.qlens[b] * c.rep.d;
        if (!win_weights_takes(call, b) || (cols >= kSplitCols) != (split != 0)) return false;
        parts = split ? ((cols + 15) / 16 + kSegTiles - 1) / kSegTiles : 1;
        units = (call.lens[b] + run - 1) / run * c.kvh * parts;
        rows = parts > 1 ? parts * c.kvh * call.lens[b] : 0;
        return true;
      },
      go);
}

}  // namespace

int64_t win_weights_bytes(const WinCall& call, int* rc) {
  int64_t most = 0;
  *rc = wgt_launches(call, 1, [&](const WinArg&, int, int64_t, int64_t rows) -> int {
    most = std::max(most, rows * static_cast<int64_t>(sizeof(float)));
    return KVQ_OK;
  });
  return most;
}

int win_weights(const WinCall& call, void* workspace) {
  const WinCache& c = call.cache;
  const int wide = call.q_wide() ? 1 : 0;
  float* sums = static_cast<float*>(workspace);
  for (int split = 0; split < 2; ++split) {
    const int rc = wgt_launches(
        call, split, [&](const WinArg& arg, int count, int64_t units, int64_t rows) -> int {
#define KVQ_WIN_WGT(T, D, S)                                                                  \
  hipLaunchKernelGGL((win_weights_kernel<T, D, S>), dim3(static_cast<unsigned>(units)),       \
                     dim3(64 * kWaves), 0, call.stream, arg, count, c,                        \
                     static_cast<const T*>(call.query), call.q_stride, wide, call.qscale,     \
                     call.lse, call.w_in, call.w_out, call.w_cols, sums)
#define KVQ_WIN_WGT_S(T, D) \
  if (split) KVQ_WIN_WGT(T, D, true); else KVQ_WIN_WGT(T, D, false)
#define KVQ_WIN_WGT_D(T)                                                                  \
  if (c.d == 64) { KVQ_WIN_WGT_S(T, 64); } else if (c.d == 128) { KVQ_WIN_WGT_S(T, 128); } \
  else { KVQ_WIN_WGT_S(T, 256); }
          if (call.dtype == KVQ_DTYPE_BF16) {
            KVQ_WIN_WGT_D(bf16);
          } else {
            KVQ_WIN_WGT_D(f16);
          }
#undef KVQ_WIN_WGT_D
#undef KVQ_WIN_WGT_S
#undef KVQ_WIN_WGT
          KVQ_LAUNCH_CHECK();
          if (rows == 0) return KVQ_OK;
          // the requests with several segments, a workgroup per 256 positions and head
          WinArg add;
          int n = 0;
          int64_t blocks = 0;
          for (int i = 0; i < count; ++i) {
            if (arg.r[i].parts == 1) continue;
            add.r[n] = arg.r[i];
            add.r[n++].first = static_cast<int32_t>(blocks);
            blocks += (static_cast<int64_t>(arg.r[i].len) + 255) / 256 * c.kvh;
          }
          if (blocks > 0x7fffffff) return KVQ_ERR_INVALID;
#define KVQ_WIN_ADD(D)                                                                          \
  hipLaunchKernelGGL((win_weights_add_kernel<D>), dim3(static_cast<unsigned>(blocks)), dim3(256), \
                     0, call.stream, add, n, c, call.w_in, call.w_out, call.w_cols, sums)
          if (c.d == 256)
            KVQ_WIN_ADD(256);
          else
            KVQ_WIN_ADD(128);
#undef KVQ_WIN_ADD
          KVQ_LAUNCH_CHECK();
          return KVQ_OK;
        });
    if (rc != KVQ_OK) return rc;
  }
  return KVQ_OK;
}

}  // namespace kvq
