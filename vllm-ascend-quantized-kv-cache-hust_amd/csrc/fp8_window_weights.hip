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
// group, joined in LDS: bound by the exponentials, one per (row, head, position).
#include <algorithm>

#include "fp8_window.h"

namespace {

using namespace kvq;

constexpr int kWaves = 4;
constexpr int kSplitCols = 64;  // columns from which a workgroup's waves share a run

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

// A unit is a workgroup's run(s) of one kv head: RUN positions if SPLIT, 4 RUN if not.
template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
win_weights_kernel(WinArg, int count, WinCache c, const T* __restrict__ query, int64_t q_stride,
                   int wide, float qscale, const float* __restrict__ lse, const float* w_in,
                   float* w_out, int64_t w_cols) {
  constexpr int NGRP = run_groups<D>(), RUN = 16 * NGRP, KS = D / 32, W = D / 64;
  __shared__ float s_scale[kWaves][RUN];
  __shared__ float s_sum[kWaves][RUN];
  const WinReq r = win_req(count, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh;
  const int wg0 = u / c.kvh * (SPLIT ? RUN : kWaves * RUN);
  const int j0 = wg0 + (SPLIT ? 0 : wave * RUN);  // the wave's first position
  const int rep = static_cast<int>(c.rep.d);
  const int cols = r.n * rep, base = r.len - r.n;
  const int j1 = min(j0 + RUN, r.len);  // past its last

  // rows that may see one of them
  int row_lo = max(j0 - base, 0), row_hi = r.n;
  if (c.window != kNoWindow && j0 >= c.sinks) {
    // the last position to see j1 - 1 is j1 - 2 + window
    const int64_t last = static_cast<int64_t>(j1) - 1 + c.window - base;
    row_hi = static_cast<int>(last < r.n ? (last < 0 ? 0 : last) : r.n);
  }
  const int t_lo = row_lo * rep / 16, t_hi = j0 < r.len ? (row_hi * rep + 15) / 16 : 0;
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
    } else {
      sum = s_sum[x / RUN][x % RUN];
    }
    w_out[dst + j] = (j < base ? w_in[dst + j] : 0.0f) + sum;
  }
}

}  // namespace

namespace kvq {

bool win_weights_takes(const WinCall& call, int64_t b) {
  const WinCache& c = call.cache;
  return win_matrix_geometry(call.dtype, c.hq, c.kvh, c.d, static_cast<int>(c.bs.d)) &&
         aligned16(c.kd, c.vd) && call.lens[b] > 0;
}

int win_weights(const WinCall& call) {
  const WinCache& c = call.cache;
  const int wide = call.q_wide() ? 1 : 0;
  for (int split = 0; split < 2; ++split) {
    const int64_t run = 16 * (c.d == 256 ? 4 : 8) * (split ? 1 : kWaves);
    const int rc = win_launches(
        call,
        [&](int64_t b, int64_t& units, int64_t&) {
          units = (call.lens[b] + run - 1) / run * c.kvh;
          return win_weights_takes(call, b) &&
                 (call.qlens[b] * c.rep.d >= kSplitCols) == (split != 0);
        },
        [&](const WinArg& arg, int count, int64_t units, int64_t) -> int {
#define KVQ_WIN_WGT(T, D, S)                                                                  \
  hipLaunchKernelGGL((win_weights_kernel<T, D, S>), dim3(static_cast<unsigned>(units)),       \
                     dim3(64 * kWaves), 0, call.stream, arg, count, c,                        \
                     static_cast<const T*>(call.query), call.q_stride, wide, call.qscale,     \
                     call.lse, call.w_in, call.w_out, call.w_cols)
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
          return KVQ_OK;
        });
    if (rc != KVQ_OK) return rc;
  }
  return KVQ_OK;
}

}  // namespace kvq
