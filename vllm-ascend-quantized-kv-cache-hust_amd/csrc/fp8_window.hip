// SPDX-License-Identifier: Apache-2.0
// Causal attention of each request's new rows straight over its paged E4M3
// rows, with an optional sliding window and sinks, and the running attention
// weights of the cached positions: the entry points, and the kernels that take
// any geometry (fp32 queries, any head size the cache has, any page size).
//
// K_j = code_k[j] * k_scale[j], V_j = code_v[j] * v_scale[j] per (token, kv head)
// (the values of pkg/methods/fp8_per_token_head/semantics.py:63-65, not rounded
// to the query's type), p_ij = softmax over the positions row i sees, out_i =
// sum_j p_ij V_j.  A row that sees nothing gives zeros.  The running weights:
// w_j = (j < len - n ? w_j : 0) + sum over the rows i and the heads of the kv
// head's group of p_ij.
//
// The general kernels: one wave per (row, head) and run of the row's positions, 64
// positions at a time, a lane a position for the scores; for the values as many
// positions at once as a row's words leave lanes for, four of each in flight; all in
// fp32 with the softmax's running maximum and sum.  Bound by the latency and the lanes
// of their loads, and by reading each code once per query head: one token at 31000
// positions, 32 heads on 8 of 96, 57 us (11050 with a wave to a row's whole history and
// one position in flight); 32 of 2048 - 16384 positions, 513 us (7881), 0.9 TB/s.
#include <algorithm>

#include "fp8_window.h"

namespace {

using namespace kvq;

__device__ __forceinline__ void codes4(uint32_t w, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  x[0] = lo[0];
  x[1] = lo[1];
  x[2] = hi[0];
  x[3] = hi[1];
}

constexpr int kGenWaves = 4;
constexpr int kGenMaxD = 512;

// fp32 dot product of the query row in LDS with a row of codes, 16 bytes at a time where
// rows are such (wide).
__device__ __forceinline__ float dot_codes(const float* q, const uint8_t* row, int d, bool wide) {
  float s = 0.0f;
  auto word = [&](uint32_t w, const float* at) {
    float x[4];
    codes4(w, x);
#pragma unroll
    for (int k = 0; k < 4; ++k) s = __builtin_fmaf(at[k], x[k], s);
  };
  if (wide) {
#pragma unroll 4
    for (int i = 0; i < d; i += 16) {
      const w_u4 w = *reinterpret_cast<const w_u4*>(row + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) word(w[k], q + i + 4 * k);
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < d; i += 4) word(*reinterpret_cast<const uint32_t*>(row + i), q + i);
  }
  return s;
}

// What a wave wrote to its own LDS is what it reads from here on.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A unit is one row, kGenWaves heads and an item: `split` 64-position groups of what the
// row sees.
template <typename T>
__global__ void __launch_bounds__(64 * kGenWaves)
win_attn_general_kernel(WinArg, int count, WinCache c, const T* __restrict__ query,
                        int64_t q_stride, int wide, float qscale, int split, T* __restrict__ out,
                        WinParts parts, float* __restrict__ lse) {
  __shared__ __align__(16) float s_q[kGenWaves][kGenMaxD];
  const WinReq r = win_req(count, blockIdx.x);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int groups = (c.hq + kGenWaves - 1) / kGenWaves;
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int i = u / groups / r.parts, item = u / groups - i * r.parts;
  const int head = u % groups * kGenWaves + wave;
  if (head >= c.hq) return;  // no barrier below: a wave reads its own part of s_q
  const int h = static_cast<int>(c.rep.div(static_cast<uint32_t>(head)));
  const int pos = r.len - r.n + i;
  const int64_t row = static_cast<int64_t>(r.q0) + i;
  const T* q = query + row * q_stride + static_cast<int64_t>(head) * c.d;
  for (int k = lane; k < c.d; k += 64) s_q[wave][k] = to_f32(q[k]);
  wave_lds_fence();
  // lane: word `word` (and 64 words on) of the positions `slice`, `slices` + `slice`, ..
  const int words = c.d / 4, width = min(words, 64), slices = 64 / width;
  const int slice = lane / width, word = lane - slice * width;
  const bool mine = slice < slices;
  float m = -INFINITY, l = 0.0f;
  w_f4 acc[2] = {w_f4{0.f, 0.f, 0.f, 0.f}, w_f4{0.f, 0.f, 0.f, 0.f}};
  const WinSpan span = pos >= 0 ? WinSpan::of(pos + 1, 1, c.window, c.sinks, 64) : WinSpan{0, 0, 0};
  const int g1 = min(span.groups, (item + 1) * split);
  for (int g = item * split; g < g1; ++g) {
    const int j = span.pos(g, 64) + lane;
    const bool on = c.sees(pos, j);
    const int64_t at = (on ? c.slot(r.table, j) : 0) * c.kvh + h;
    float s = -INFINITY, vs = 0.0f;
    if (on) {
      s = dot_codes(s_q[wave], c.kd + at * c.d, c.d, wide) * (c.ks[at] * qscale);
      vs = c.vs[at];
    }
    const uint64_t mask = __builtin_amdgcn_ballot_w64(on);
    if (!mask) continue;
    const float top = fmaxf(m, max_wave64(s));
    const float base = top == -INFINITY ? 0.0f : top;
    const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - base);
    const float p = on ? __builtin_amdgcn_exp2f(s - base) : 0.0f;
    m = top;
    l = l * alpha + sum_wave64(p);
    const float pv = on ? p * vs : 0.0f;
    acc[0] *= alpha;
    acc[1] *= alpha;
    constexpr int DEPTH = 4;  // positions in flight
    for (int t0 = 0; t0 < 64; t0 += DEPTH * slices) {
      if (!(mask >> t0)) break;
      uint32_t x[DEPTH][2];
      float pt[DEPTH];
#pragma unroll
      for (int e = 0; e < DEPTH; ++e) {
        const int t = t0 + e * slices + slice;
        const bool seen = mine && t < 64 && ((mask >> (t & 63)) & 1);
        pt[e] = __shfl(pv, t & 63, 64);
        const uint8_t* v = c.vd + __shfl(at, t & 63, 64) * c.d + 4 * word;
        x[e][0] = seen ? *reinterpret_cast<const uint32_t*>(v) : 0u;
        x[e][1] = seen && word + 64 < words ? *reinterpret_cast<const uint32_t*>(v + 256) : 0u;
        pt[e] = seen ? pt[e] : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < DEPTH; ++e)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float y[4];
          codes4(x[e][w], y);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[w][k] = __builtin_fmaf(pt[e], y[k], acc[w][k]);
        }
    }
  }
  if (slices > 1) {  // rows of at most 32 words
    float* sum = s_q[wave];
    wave_lds_fence();
    if (mine) *reinterpret_cast<w_f4*>(sum + slice * c.d + 4 * word) = acc[0];
    wave_lds_fence();
    if (slice == 0)
      for (int x = 1; x < slices; ++x)
        acc[0] += *reinterpret_cast<const w_f4*>(sum + x * c.d + 4 * word);
  }
  if (r.parts > 1) {
    const int64_t part = r.part0 + (static_cast<int64_t>(item) * r.n + i) * c.hq + head;
    if (slice == 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (word + 64 * w < words)
          *reinterpret_cast<w_f4*>(parts.o + part * c.d + 4 * (word + 64 * w)) = acc[w];
    }
    if (lane == 0)  // a NaN score leaves m without it, but not l
      *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{l != l ? INFINITY : m, l};
    return;
  }
  T* o = out + (row * c.hq + head) * c.d;
  if (slice == 0) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (word + 64 * w < words)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          // l is 0 only where nothing is seen; a NaN goes through
          o[4 * (word + 64 * w) + k] = from_f32<T>(l == 0.0f ? 0.0f : acc[w][k] / l);
  }
  // (max, sum) in one number: p = 2^(s - lse)
  if (lse && lane == 0) lse[row * c.hq + head] = l == 0.0f ? INFINITY : m + __log2f(l);
}

// Running weights, a thread a position, kGenCols columns (row, head) at a time, so that a
// key's codes are read and converted once for all of them (32 requests of 2048 - 16384
// positions, 32 heads on 8 of 96: 160 us beside the attention, 2170 a column at a time).
// A unit is 256 positions of one kv head.
constexpr int kGenCols = 8;

template <typename T>
__global__ void __launch_bounds__(256)
win_weights_general_kernel(WinArg, int count, WinCache c, const T* __restrict__ query,
                           int64_t q_stride, int wide, float qscale,
                           const float* __restrict__ lse, const float* w_in, float* w_out,
                           int64_t w_cols) {
  __shared__ __align__(16) float s_q[kGenCols][kGenMaxD];
  const WinReq r = win_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % c.kvh, j0 = u / c.kvh * 256;
  const int j = j0 + static_cast<int>(threadIdx.x);
  const int first = r.len - r.n;  // position of row 0
  const int rep = static_cast<int>(c.rep.d);
  const int64_t at = c.slot(r.table, min(j, r.len - 1)) * c.kvh + h;
  const uint8_t* key = c.kd + at * c.d;
  const float scale = c.ks[at] * qscale;
  float sum = 0.0f;
  // the rows that see some of these positions
  const int i0 = max(0, j0 - first);
  const int64_t past = j0 < c.sinks ? r.n : static_cast<int64_t>(j0) + 255 + c.window - first;
  const int i1 = static_cast<int>(past < 0 ? 0 : (past < r.n ? past : r.n));
  for (int x0 = i0 * rep; x0 < i1 * rep; x0 += kGenCols) {
    __syncthreads();  // the last columns are read
    for (int y = 0; y < kGenCols; ++y) {
      const int col = min(x0 + y, i1 * rep - 1);
      const int i = static_cast<int>(c.rep.div(static_cast<uint32_t>(col)));
      const T* q = query + (static_cast<int64_t>(r.q0) + i) * q_stride +
                   static_cast<int64_t>(h * rep + col - i * rep) * c.d;
      for (int e = static_cast<int>(threadIdx.x); e < c.d; e += 256) s_q[y][e] = to_f32(q[e]);
    }
    __syncthreads();
    float s[kGenCols] = {};
    auto word = [&](uint32_t w, int e) {
      float x[4];
      codes4(w, x);
#pragma unroll
      for (int y = 0; y < kGenCols; ++y) {
        const w_f4 q = *reinterpret_cast<const w_f4*>(&s_q[y][e]);
#pragma unroll
        for (int t = 0; t < 4; ++t) s[y] = __builtin_fmaf(q[t], x[t], s[y]);
      }
    };
    if (wide) {
      for (int e = 0; e < c.d; e += 16) {
        const w_u4 w = *reinterpret_cast<const w_u4*>(key + e);
#pragma unroll
        for (int t = 0; t < 4; ++t) word(w[t], e + 4 * t);
      }
    } else {
      for (int e = 0; e < c.d; e += 4) word(*reinterpret_cast<const uint32_t*>(key + e), e);
    }
#pragma unroll
    for (int y = 0; y < kGenCols; ++y) {
      if (x0 + y >= i1 * rep) break;
      const int i = static_cast<int>(c.rep.div(static_cast<uint32_t>(x0 + y)));
      if (!c.sees(first + i, j)) continue;
      const int64_t row = static_cast<int64_t>(r.q0) + i;
      sum += __builtin_amdgcn_exp2f(s[y] * scale -
                                    lse[row * c.hq + h * rep + x0 + y - i * rep]);
    }
  }
  if (j >= r.len) return;
  const int64_t dst = (static_cast<int64_t>(r.wrow) * c.kvh + h) * w_cols + j;
  w_out[dst] = (j < first ? w_in[dst] : 0.0f) + sum;
}

// The running weights of a request without rows, into the other array.  A unit is
// kIdleSpan positions of one kv head.
constexpr int kIdleSpan = 1024;

__global__ void __launch_bounds__(256)
win_weights_idle_kernel(WinArg, int count, int kvh, const float* __restrict__ w_in,
                        float* __restrict__ w_out, int64_t w_cols) {
  const WinReq r = win_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % kvh, j0 = u / kvh * kIdleSpan + static_cast<int>(threadIdx.x);
  const int64_t row = (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
#pragma unroll
  for (int k = 0; k < kIdleSpan; k += 256)
    if (j0 + k < r.len) w_out[row + j0 + k] = w_in[row + j0 + k];
}

// ---- joining partial results ---------------------------------------------------------

constexpr int kJoinThreads = 256;

// A unit is a row and head of a request that has parts: blockIdx.x of request blockIdx.y,
// or, where the grid has one row for several requests, of all of them.  d / 4 threads hold
// a part's row, the workgroup several parts at once, joined in LDS in a fixed order.
// D: d, or 0 for any.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
win_join_kernel(WinArg, int requests, int hq, int any_d, WinParts parts, T* __restrict__ out,
                float* __restrict__ lse) {
  const int d = D ? D : any_d, lanes = d / 4, slices = kJoinThreads / lanes;
  __shared__ w_f4 s_o[kJoinThreads];
  const bool flat = gridDim.y == 1 && requests > 1;
  const WinReq r = flat ? win_req(requests, blockIdx.x) : win_req_at(blockIdx.y);
  const int q0 = r.q0, count = r.parts, part0 = r.part0;
  const int64_t x = static_cast<int>(blockIdx.x) - (flat ? r.first : 0);
  const int64_t stride = static_cast<int64_t>(r.n) * hq;
  if (x >= stride) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const w_f2* ml = reinterpret_cast<const w_f2*>(parts.ml) + part0 + x;
  float m = -INFINITY;
  for (int s = lane; s < count; s += 64) m = fmaxf(m, ml[s * stride][0]);
  m = max_wave64(m);
  if (m >= 0x1.fffffep127f) m = INFINITY;  // the tiles' maxima stop at FLT_MAX
  float l = 0.0f;
  for (int s = lane; s < count; s += 64) {
    const w_f2 y = ml[s * stride];
    l += y[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y[0] - m) * y[1];
  }
  l = sum_wave64(l);
  const int slice = tid / lanes, k = tid - slice * lanes;
  w_f4 acc = w_f4{0.f, 0.f, 0.f, 0.f};
  constexpr int DEPTH = 4;  // loads in flight
  for (int s0 = slice < slices ? slice : count; s0 < count; s0 += DEPTH * slices) {
    float ms[DEPTH];
    w_f4 y[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      const int64_t s = min(s0 + i * slices, count - 1);
      ms[i] = s0 + i * slices < count ? ml[s * stride][0] : -INFINITY;
      y[i] = *reinterpret_cast<const w_f4*>(parts.o + (part0 + s * stride + x) * d + 4 * k);
    }
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      const float w = ms[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms[i] - m);
      // one that sees nothing may be unwritten
      acc += ms[i] == -INFINITY ? w_f4{0.f, 0.f, 0.f, 0.f} : w * y[i];
    }
  }
  s_o[tid] = acc;
  __syncthreads();
  if (slice) return;
#pragma unroll D ? 4 : 1
  for (int s = 1; s < slices; ++s) acc += s_o[s * lanes + k];
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = static_cast<int64_t>(q0) * hq + x;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[at * d + 4 * k + e] = from_f32<T>(acc[e] * inv);
  if (lse && k == 0) lse[at] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

}  // namespace

namespace kvq {

int launch_win_join(const WinCall& call, const WinArg& arg, int count, WinParts parts) {
  const int hq = call.cache.hq;
  WinArg cut;
  int n = 0;
  int64_t units = 0, most = 0;  // (at most the call's rows and heads, < 2^31)
  for (int i = 0; i < count; ++i) {
    if (arg.r[i].parts <= 1) continue;
    cut.r[n] = arg.r[i];
    cut.r[n++].first = static_cast<int32_t>(units);
    units += static_cast<int64_t>(arg.r[i].n) * hq;
    most = std::max(most, static_cast<int64_t>(arg.r[i].n) * hq);
  }
  if (n == 0) return KVQ_OK;
  // a grid of requests by the most rows, where half of it has rows (the request is at hand:
  // 64 of one row each, 104.0 us a call for 104.9), or of all rows in a line (100 requests of
  // 8 rows beside one of 2000: 204 us for 518, 347 of it in the empty rest of the grid)
  const dim3 grid = most * n <= 2 * units ? dim3(static_cast<unsigned>(most), static_cast<unsigned>(n))
                                          : dim3(static_cast<unsigned>(units));
#define KVQ_WIN_JOIN(T, D)                                                                    \
  hipLaunchKernelGGL((win_join_kernel<T, D>), grid, dim3(kJoinThreads), 0, call.stream, cut, n, \
                     hq, call.cache.d, parts, static_cast<T*>(call.out), call.lse)
#define KVQ_WIN_JOIN_D(T)                                                              \
  if (call.cache.d == 64) KVQ_WIN_JOIN(T, 64); else if (call.cache.d == 128)           \
  KVQ_WIN_JOIN(T, 128); else if (call.cache.d == 256) KVQ_WIN_JOIN(T, 256); else       \
  KVQ_WIN_JOIN(T, 0)
  if (call.dtype == KVQ_DTYPE_BF16) {
    KVQ_WIN_JOIN_D(bf16);
  } else if (call.dtype == KVQ_DTYPE_F16) {
    KVQ_WIN_JOIN_D(f16);
  } else {
    KVQ_WIN_JOIN(float, 0);
  }
#undef KVQ_WIN_JOIN_D
#undef KVQ_WIN_JOIN
  KVQ_LAUNCH_CHECK();
  return KVQ_OK;
}

}  // namespace kvq

namespace {

// ---- host -----------------------------------------------------------------------

// 64-position groups of an item of the general kernel: 16 waves a CU, or items of two
// groups.  From the lengths alone, whichever kernel takes them: the workspace's size,
// which does not know the addresses, goes by it.
int64_t gen_groups(const WinCall& call, int64_t b) {
  return call.qlens[b] > 0 && call.lens[b] > 0
             ? WinSpan::of(static_cast<int>(call.lens[b]), static_cast<int>(call.qlens[b]),
                           call.cache.window, call.cache.sinks, 64)
                   .groups
             : 0;
}
int64_t gen_split(const WinCall& call) {
  int cus = 0;
  if (device_cu_count(&cus) != KVQ_OK || cus <= 0) cus = 256;
  int64_t total = 0;
  for (int64_t b = 0; b < call.batch; ++b)
    total += gen_groups(call, b) * call.qlens[b] * call.cache.hq;
  return std::min<int64_t>(std::max<int64_t>(2, total / (16 * cus)), kMaxPositions / 64);
}
int64_t gen_parts(const WinCall& call, int64_t b, int64_t split) {
  return std::max<int64_t>(1, (gen_groups(call, b) + split - 1) / split);
}
int64_t general_bytes(const WinCall& call) {
  const int64_t split = gen_split(call);
  int64_t rows = 0;
  for (int64_t b = 0; b < call.batch; ++b)
    rows += win_part_rows(call, b, gen_parts(call, b, split));
  return win_parts_bytes(rows, call.cache.d);
}

// Requests that no matrix kernel takes.
template <typename T>
int attend_general(const WinCall& call, void* workspace) {
  const WinCache& c = call.cache;
  const int64_t groups = (c.hq + kGenWaves - 1) / kGenWaves, split = gen_split(call);
  const int wide = c.d % 16 == 0 && aligned16(c.kd, nullptr);
  return win_launches(
      call,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        if (win_decode_takes(call, b) || win_chunk_takes(call, b)) return false;
        parts = gen_parts(call, b, split);
        rows = win_part_rows(call, b, parts);
        units = call.qlens[b] * parts * groups;
        return true;
      },
      [&](const WinArg& arg, int count, int64_t blocks, int64_t rows) -> int {
        const WinParts parts{static_cast<float*>(workspace),
                             static_cast<float*>(workspace) + rows * c.d};
        hipLaunchKernelGGL((win_attn_general_kernel<T>), dim3(static_cast<unsigned>(blocks)),
                           dim3(64 * kGenWaves), 0, call.stream, arg, count, c,
                           static_cast<const T*>(call.query), call.q_stride, wide, call.qscale,
                           static_cast<int>(split), static_cast<T*>(call.out), parts, call.lse);
        KVQ_LAUNCH_CHECK();
        return rows > 0 ? launch_win_join(call, arg, count, parts) : KVQ_OK;
      });
}

template <typename T>
int weigh_general(const WinCall& call) {
  const int wide = call.cache.d % 16 == 0 && aligned16(call.cache.kd, nullptr);
  return win_launches(
      call,
      [&](int64_t b, int64_t& units, int64_t&, int64_t&) {
        units = (call.lens[b] + 255) / 256 * call.cache.kvh;
        return !win_weights_takes(call, b);
      },
      [&](const WinArg& arg, int count, int64_t blocks, int64_t) -> int {
        hipLaunchKernelGGL((win_weights_general_kernel<T>), dim3(static_cast<unsigned>(blocks)),
                           dim3(256), 0, call.stream, arg, count, call.cache,
                           static_cast<const T*>(call.query), call.q_stride, wide, call.qscale,
                           call.lse, call.w_in, call.w_out, call.w_cols);
        KVQ_LAUNCH_CHECK();
        return KVQ_OK;
      });
}

// What running weights that go to another array leave of requests without rows.
int copy_idle(const WinCall& call) {
  return win_launches(
      call,
      [&](int64_t b, int64_t& units, int64_t&, int64_t&) {
        units = (call.lens[b] + kIdleSpan - 1) / kIdleSpan * call.cache.kvh;
        return true;
      },
      [&](const WinArg& arg, int count, int64_t blocks, int64_t) -> int {
        hipLaunchKernelGGL(win_weights_idle_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256),
                           0, call.stream, arg, count, call.cache.kvh, call.w_in, call.w_out,
                           call.w_cols);
        KVQ_LAUNCH_CHECK();
        return KVQ_OK;
      },
      true);
}

// Lengths, window and geometry, checked alike by the sizing call and the call.
int check_shape(const int64_t* lens, const int64_t* qlens, int64_t batch, int dtype, int hq, int kvh,
                int d, int bs, int64_t window, int64_t sinks) {
  if (batch < 0 || (batch > 0 && (!lens || !qlens)) || window < 0 || sinks < 0)
    return KVQ_ERR_INVALID;
  if (dtype != KVQ_DTYPE_F32 && dtype != KVQ_DTYPE_F16 && dtype != KVQ_DTYPE_BF16)
    return KVQ_ERR_INVALID;
  if (kvh <= 0 || hq <= 0 || hq % kvh || d <= 0 || d % 4 || d > kGenMaxD || bs <= 0 || hq > 65536)
    return KVQ_ERR_GEOMETRY;
  int64_t rows = 0;
  for (int64_t b = 0; b < batch; ++b) {
    if (lens[b] < 0 || lens[b] > kMaxPositions || qlens[b] < 0 || qlens[b] > kMaxPositions)
      return KVQ_ERR_INVALID;
    rows += qlens[b];
    if (rows > kMaxPositions / hq) return KVQ_ERR_INVALID;
  }
  return KVQ_OK;
}

int64_t align16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Bytes of the log-sum-exps (kept for the running weights), before the partial results.
int64_t lse_bytes(const int64_t* qlens, int64_t batch, int hq, bool weigh) {
  if (!weigh) return 0;
  int64_t rows = 0;
  for (int64_t b = 0; b < batch; ++b) rows += qlens[b];
  return align16(4 * rows * hq);
}

WinCall make_call(const void* query, int dtype, int64_t query_stride, const int64_t* seq_lens,
                  const int64_t* query_lens, int64_t batch, int hq, int kvh, int d, float scale,
                  int64_t window, int64_t sinks, int block_size) {
  WinCall call{};
  call.query = query;
  call.dtype = dtype;
  call.q_stride = query_stride;
  call.lens = seq_lens;
  call.qlens = query_lens;
  call.batch = batch;
  call.cache.bs = FastDiv::make(static_cast<uint32_t>(block_size));
  call.cache.kvh = kvh;
  call.cache.hq = hq;
  call.cache.d = d;
  call.cache.rep = FastDiv::make(static_cast<uint32_t>(hq / kvh));
  call.cache.window = window > 0 && window < kNoWindow ? static_cast<int>(window) : kNoWindow;
  call.cache.sinks =
      static_cast<int>(window > 0 ? std::min<int64_t>(sinks, kMaxPositions) : 0);
  call.qscale = scale * 1.4426950408889634f;
  call.few_cols = win_few_cols(call);
  call.tiles_only = win_tiles_only(call);
  return call;
}

// A call's workspace: log-sum-exps, the decode's scores, partial results (the kernels run
// one after another and share these).
struct Layout {
  int64_t lse, scores, parts;
  WinScores scored;
  int64_t total() const { return lse + scores + parts; }
};
Layout layout_of(const WinCall& call, bool weigh, int* rc) {
  Layout x{};
  x.lse = lse_bytes(call.qlens, call.batch, call.cache.hq, weigh);
  if (weigh) x.scored = win_scores(call);
  x.scores = 64 * x.scored.units;
  const int64_t few = win_decode_bytes(call, rc);
  if (*rc != KVQ_OK) return x;
  const int64_t many = win_chunk_bytes(call, rc);
  if (*rc != KVQ_OK) return x;
  const int64_t sums = weigh ? win_weights_bytes(call, x.scored, rc) : 0;
  x.parts = align16(std::max(std::max(few, many), std::max(sums, general_bytes(call))));
  return x;
}

}  // namespace

extern "C" int64_t kvq_fp8_pth_window_attn_workspace_bytes(
    const int64_t* seq_lens, const int64_t* query_lens, int64_t batch, int dtype, int num_heads,
    int num_kv_heads, int head_size, int block_size, int64_t window, int64_t sinks,
    int with_weights) {
  int rc = check_shape(seq_lens, query_lens, batch, dtype, num_heads, num_kv_heads, head_size,
                       block_size, window, sinks);
  if (rc != KVQ_OK) return rc;
  // (caches off a 16-byte bound need less: the size does not know the addresses)
  const WinCall call = make_call(nullptr, dtype, 0, seq_lens, query_lens, batch, num_heads,
                                 num_kv_heads, head_size, 1.0f, window, sinks, block_size);
  const Layout layout = layout_of(call, with_weights != 0, &rc);
  return rc != KVQ_OK ? KVQ_ERR_INVALID : layout.total();
}

extern "C" int kvq_fp8_pth_window_attn(
    const void* query, int dtype, int64_t query_stride, const int64_t* seq_lens,
    const int64_t* query_lens, int64_t batch, int num_heads, int num_kv_heads, int head_size,
    float scale, int64_t window, int64_t sinks, const uint8_t* k_data, const float* k_scale,
    const uint8_t* v_data, const float* v_scale, int64_t num_blocks, int block_size,
    const void* block_table, int block_index_type, int64_t max_blocks, const float* weights_in,
    float* weights_out, const int64_t* weight_rows, int64_t weight_cols, void* workspace,
    int64_t workspace_bytes, void* out, void* stream) {
  int rc = check_shape(seq_lens, query_lens, batch, dtype, num_heads, num_kv_heads, head_size,
                       block_size, window, sinks);
  if (rc != KVQ_OK) return rc;
  int64_t rows = 0;
  for (int64_t b = 0; b < batch; ++b) rows += query_lens[b];
  // running weights that go to another array go there whole: of requests without rows too
  const bool weigh = weights_out != nullptr, apart = weigh && weights_in && weights_in != weights_out;
  if (rows == 0 && !apart) return KVQ_OK;
  if (rows > 0 &&
      (!query || !k_data || !k_scale || !v_data || !v_scale || !block_table || !out ||
       num_blocks <= 0 || max_blocks < 0 || !(scale > 0.0f && scale < INFINITY) ||
       query_stride < static_cast<int64_t>(num_heads) * head_size))
    return KVQ_ERR_INVALID;
  if (block_index_type != KVQ_INDEX_I32 && block_index_type != KVQ_INDEX_I64)
    return KVQ_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(k_data) | reinterpret_cast<uintptr_t>(v_data)) & 3)
    return KVQ_ERR_GEOMETRY;  // a row's words
  if (weigh != (weights_in != nullptr) || (weigh && !weight_rows)) return KVQ_ERR_INVALID;
  for (int64_t b = 0; b < batch; ++b) {
    if (query_lens[b] == 0 && !apart) continue;
    if (query_lens[b] > 0 && seq_lens[b] > max_blocks * block_size) return KVQ_ERR_INVALID;
    if (weigh && (seq_lens[b] > weight_cols || weight_rows[b] < 0 || weight_rows[b] > kMaxPositions))
      return KVQ_ERR_INVALID;
  }
  WinCall call = make_call(query, dtype, query_stride, seq_lens, query_lens, batch, num_heads,
                           num_kv_heads, head_size, scale, window, sinks, block_size);
  call.cache.kd = k_data;
  call.cache.ks = k_scale;
  call.cache.vd = v_data;
  call.cache.vs = v_scale;
  call.cache.table = block_table;
  call.cache.maxb = max_blocks;
  call.cache.nb = num_blocks;
  call.cache.bt64 = block_index_type == KVQ_INDEX_I64;
  call.w_in = weights_in;
  call.w_out = weights_out;
  call.w_rows = weight_rows;
  call.w_cols = weight_cols;
  call.out = out;
  call.stream = static_cast<hipStream_t>(stream);
  if (apart) rc = copy_idle(call);
  if (rc != KVQ_OK || rows == 0) return rc;
  const Layout layout = layout_of(call, weigh, &rc);
  if (rc != KVQ_OK) return rc;
  if (layout.total() > 0 &&
      (!workspace || !aligned16(workspace, nullptr) || workspace_bytes < layout.total()))
    return KVQ_ERR_INVALID;
  char* ws = static_cast<char*>(workspace);
  call.lse = weigh ? static_cast<float*>(workspace) : nullptr;
  call.scores = layout.scored.on ? reinterpret_cast<float*>(ws + layout.lse) : nullptr;
  void* parts = ws + layout.lse + layout.scores;
  rc = win_decode(call, parts);
  if (rc != KVQ_OK) return rc;
  rc = win_chunk(call, parts);
  if (rc != KVQ_OK) return rc;
  KVQ_DISPATCH_FLOAT(dtype, T, {
    rc = attend_general<T>(call, parts);
    if (rc != KVQ_OK) return rc;
    if (weigh) rc = weigh_general<T>(call);
    if (rc != KVQ_OK) return rc;
    if (weigh) rc = win_weights(call, layout.scored, parts);
  });
  return rc;
}

// ---- host checks ------------------------------------------------------------------

extern "C" int64_t kvq_fp8_pth_window_check(const void* block_table, int block_index_type,
                                            int64_t max_blocks, const int64_t* seq_lens,
                                            const int64_t* query_lens, int64_t batch,
                                            int64_t num_blocks, int block_size, int64_t window,
                                            int64_t sinks) {
  if (batch < 0 || block_size <= 0 || max_blocks < 0 || (batch > 0 && (!seq_lens || !query_lens)))
    return KVQ_ERR_INVALID;
  for (int64_t b = 0; b < batch; ++b) {
    const int64_t len = seq_lens[b], n = query_lens[b];
    if (len < 0 || n < 0) return KVQ_ERR_INVALID;
    if (n == 0 || len == 0) continue;
    if (len > max_blocks * block_size) return KVQ_ERR_CAPACITY;
    int64_t low = window > 0 ? len - n - window + 1 : 0;
    low = low < 0 ? 0 : low;
    const int64_t sink = window > 0 ? (sinks < low ? sinks : low) : 0;
    const int64_t sink_pages = (sink + block_size - 1) / block_size;
    for (int64_t i = 0; i < (len + block_size - 1) / block_size; ++i) {
      if (i >= sink_pages && (i + 1) * block_size <= low) continue;  // nobody sees it
      const int64_t at = b * max_blocks + i;
      const int64_t id = block_index_type == KVQ_INDEX_I64
                             ? static_cast<const int64_t*>(block_table)[at]
                             : static_cast<const int32_t*>(block_table)[at];
      if (id < 0 || id >= num_blocks) return b + 1;
    }
  }
  return KVQ_OK;
}
