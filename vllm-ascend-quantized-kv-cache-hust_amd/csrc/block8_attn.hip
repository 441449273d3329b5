// SPDX-License-Identifier: Apache-2.0
// Causal attention of each request's new rows straight over pages of 8-bit codes with a
// scale for each block of positions and kv head, with an optional sliding window and sinks:
// the entry points, and the kernel that takes any geometry.
//
// K_j = code_k[j] * k_scale[block of j], V_j likewise (E4M3 or INT8 codes, not rounded to the
// query's type), p_ij = softmax over the positions row i sees of scale * q_i . K_j,
// out_i = sum_j p_ij V_j.  A row that sees nothing gives zeros.
//
// The general kernel: one wave per (row, head) and run of the row's positions, 64 positions
// at a time, a lane a position for the scores, a lane four dims for the values, fp32 with
// the softmax's running maximum and sum.  Bound by the latency of its loads and by reading
// each code once per query head.
#include <algorithm>

#include "block8.h"

namespace {

using namespace kvq;

constexpr int kGenWaves = 4;
constexpr int kGenMaxD = 512;

template <bool INT8>
__device__ __forceinline__ void codes4(uint32_t w, float (&x)[4]) {
  if constexpr (INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo[0];
    x[1] = lo[1];
    x[2] = hi[0];
    x[3] = hi[1];
  }
}

// What a wave wrote to its own LDS is what it reads from here on.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A unit is one row, kGenWaves heads and an item: `split` 64-position groups of what the
// row sees.
template <typename T, bool INT8>
__global__ void __launch_bounds__(64 * kGenWaves)
b8_general_kernel(WinArg, int count, B8Cache c, const T* __restrict__ query, int64_t q_stride,
                  float qscale, int split, T* __restrict__ out, WinParts parts) {
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
  // lane: words `lane` and `lane` + 64 of a value row
  const int words = c.d / 4;
  float m = -INFINITY, l = 0.0f;
  w_f4 acc[2] = {w_f4{0.f, 0.f, 0.f, 0.f}, w_f4{0.f, 0.f, 0.f, 0.f}};
  const WinSpan span = pos >= 0 ? WinSpan::of(pos + 1, 1, c.window, c.sinks, 64) : WinSpan{0, 0, 0};
  const int g1 = min(span.groups, (item + 1) * split);
  for (int g = item * split; g < g1; ++g) {
    const int j = span.pos(g, 64) + lane;
    const bool on = c.sees(pos, j);
    const B8Cache::At at = on ? c.at(r.table, j) : B8Cache::At{0, 0};
    const int64_t slot = at.slot * c.kvh + h;
    float s = -INFINITY, vs = 0.0f;
    if (on) {
      const uint8_t* k = c.kd + slot * c.d;
      s = 0.0f;
#pragma unroll 4
      for (int e = 0; e < c.d; e += 4) {
        float x[4];
        codes4<INT8>(*reinterpret_cast<const uint32_t*>(k + e), x);
#pragma unroll
        for (int t = 0; t < 4; ++t) s = __builtin_fmaf(s_q[wave][e + t], x[t], s);
      }
      s *= c.ks[at.scale + h] * qscale;
      vs = c.vs[at.scale + h];
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
    for (int t0 = 0; t0 < 64; t0 += DEPTH) {
      if (!(mask >> t0)) break;
      uint32_t x[DEPTH][2];
      float pt[DEPTH];
#pragma unroll
      for (int e = 0; e < DEPTH; ++e) {
        const int t = t0 + e;
        const bool seen = (mask >> t) & 1;
        pt[e] = seen ? __shfl(pv, t, 64) : 0.0f;
        const uint8_t* v = c.vd + __shfl(slot, t, 64) * c.d + 4 * lane;
        x[e][0] = seen && lane < words ? *reinterpret_cast<const uint32_t*>(v) : 0u;
        x[e][1] = seen && lane + 64 < words ? *reinterpret_cast<const uint32_t*>(v + 256) : 0u;
      }
#pragma unroll
      for (int e = 0; e < DEPTH; ++e)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float y[4];
          codes4<INT8>(x[e][w], y);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[w][k] = __builtin_fmaf(pt[e], y[k], acc[w][k]);
        }
    }
  }
  if (r.parts > 1) {
    const int64_t part = r.part0 + (static_cast<int64_t>(item) * r.n + i) * c.hq + head;
#pragma unroll
    for (int w = 0; w < 2; ++w)
      if (lane + 64 * w < words)
        *reinterpret_cast<w_f4*>(parts.o + part * c.d + 4 * (lane + 64 * w)) = acc[w];
    if (lane == 0)  // a NaN score leaves m without it, but not l
      *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{l != l ? INFINITY : m, l};
    return;
  }
  T* o = out + (row * c.hq + head) * c.d;
#pragma unroll
  for (int w = 0; w < 2; ++w)
    if (lane + 64 * w < words)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        // l is 0 only where nothing is seen; a NaN goes through
        o[4 * (lane + 64 * w) + k] = from_f32<T>(l == 0.0f ? 0.0f : acc[w][k] / l);
}

// ---- host -----------------------------------------------------------------------

// 64-position groups of an item: 16 waves a CU, or items of two groups.  From the lengths
// alone, whichever kernel takes them: the workspace's size, which does not know the
// addresses, goes by it.
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
int attend_general(const B8Call& call, void* workspace) {
  const WinCall& win = call.win;
  const B8Cache& c = call.cache;
  const int64_t groups = (c.hq + kGenWaves - 1) / kGenWaves, split = gen_split(win);
  return win_launches(
      win,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        if (b8_decode_takes(call, b) || b8_chunk_takes(call, b)) return false;
        parts = gen_parts(win, b, split);
        rows = win_part_rows(win, b, parts);
        units = win.qlens[b] * parts * groups;
        return true;
      },
      [&](const WinArg& arg, int count, int64_t blocks, int64_t rows) -> int {
        const WinParts parts{static_cast<float*>(workspace),
                             static_cast<float*>(workspace) + rows * c.d};
        auto kernel = c.int8 ? b8_general_kernel<T, true> : b8_general_kernel<T, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * kGenWaves), 0,
                           win.stream, arg, count, c, static_cast<const T*>(win.query),
                           win.q_stride, win.qscale, static_cast<int>(split),
                           static_cast<T*>(win.out), parts);
        KVQ_LAUNCH_CHECK();
        return rows > 0 ? launch_win_join(win, arg, count, parts) : KVQ_OK;
      });
}

// Lengths, window and geometry, checked alike by the sizing call and the call.
int check_shape(const int64_t* lens, const int64_t* qlens, int64_t batch, int dtype, int hq, int kvh,
                int d, int bs, int group, int codes, int64_t window, int64_t sinks) {
  if (batch < 0 || (batch > 0 && (!lens || !qlens)) || window < 0 || sinks < 0)
    return KVQ_ERR_INVALID;
  if (dtype != KVQ_DTYPE_F32 && dtype != KVQ_DTYPE_F16 && dtype != KVQ_DTYPE_BF16)
    return KVQ_ERR_INVALID;
  if (codes != KVQ_CODES_E4M3 && codes != KVQ_CODES_INT8) return KVQ_ERR_INVALID;
  if (kvh <= 0 || hq <= 0 || hq % kvh || d <= 0 || d % 4 || d > kGenMaxD || bs <= 0 || hq > 65536 ||
      group <= 0 || bs % group)
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

B8Call make_call(const void* query, int dtype, int64_t query_stride, const int64_t* seq_lens,
                 const int64_t* query_lens, int64_t batch, int hq, int kvh, int d, float scale,
                 int64_t window, int64_t sinks, int block_size, int group, int codes) {
  B8Call call{};
  WinCall& win = call.win;
  win.query = query;
  win.dtype = dtype;
  win.q_stride = query_stride;
  win.lens = seq_lens;
  win.qlens = query_lens;
  win.batch = batch;
  B8Cache& c = call.cache;
  c.bs = FastDiv::make(static_cast<uint32_t>(block_size));
  c.group = FastDiv::make(static_cast<uint32_t>(group));
  c.int8 = codes == KVQ_CODES_INT8;
  c.kvh = kvh;
  c.hq = hq;
  c.d = d;
  c.rep = FastDiv::make(static_cast<uint32_t>(hq / kvh));
  c.window = window > 0 && window < kNoWindow ? static_cast<int>(window) : kNoWindow;
  c.sinks = static_cast<int>(window > 0 ? std::min<int64_t>(sinks, kMaxPositions) : 0);
  win.qscale = scale * 1.4426950408889634f;
  win.cache = c;
  win.few_cols = win_few_cols(win);
  win.tiles_only = b8_tiles_only(call);
  return call;
}

int64_t workspace_of(const B8Call& call, int* rc) {
  const int64_t few = b8_decode_bytes(call, rc);
  if (*rc != KVQ_OK) return 0;
  const int64_t many = b8_chunk_bytes(call, rc);
  if (*rc != KVQ_OK) return 0;
  // (the kernels run one after another and share it)
  return (std::max(std::max(few, many), general_bytes(call.win)) + 15) / 16 * 16;
}

}  // namespace

extern "C" int64_t kvq_block8_attn_workspace_bytes(const int64_t* seq_lens, const int64_t* query_lens,
                                                   int64_t batch, int dtype, int num_heads,
                                                   int num_kv_heads, int head_size, int block_size,
                                                   int group, int code_type, int64_t window,
                                                   int64_t sinks) {
  int rc = check_shape(seq_lens, query_lens, batch, dtype, num_heads, num_kv_heads, head_size,
                       block_size, group, code_type, window, sinks);
  if (rc != KVQ_OK) return rc;
  // (caches off a 16-byte bound need less: the size does not know the addresses)
  const B8Call call = make_call(nullptr, dtype, 0, seq_lens, query_lens, batch, num_heads,
                                num_kv_heads, head_size, 1.0f, window, sinks, block_size, group,
                                code_type);
  const int64_t bytes = workspace_of(call, &rc);
  return rc != KVQ_OK ? KVQ_ERR_INVALID : bytes;
}

extern "C" int kvq_block8_attn(const void* query, int dtype, int64_t query_stride,
                               const int64_t* seq_lens, const int64_t* query_lens, int64_t batch,
                               int num_heads, int num_kv_heads, int head_size, float scale,
                               int64_t window, int64_t sinks, int code_type, const void* k_data,
                               const float* k_scale, const void* v_data, const float* v_scale,
                               int64_t num_blocks, int block_size, int group,
                               const void* block_table, int block_index_type, int64_t max_blocks,
                               void* workspace, int64_t workspace_bytes, void* out, void* stream) {
  int rc = check_shape(seq_lens, query_lens, batch, dtype, num_heads, num_kv_heads, head_size,
                       block_size, group, code_type, window, sinks);
  if (rc != KVQ_OK) return rc;
  int64_t rows = 0;
  for (int64_t b = 0; b < batch; ++b) rows += query_lens[b];
  if (rows == 0) return KVQ_OK;
  if (!query || !k_data || !k_scale || !v_data || !v_scale || !block_table || !out ||
      num_blocks <= 0 || max_blocks < 0 || !(scale > 0.0f && scale < INFINITY) ||
      query_stride < static_cast<int64_t>(num_heads) * head_size)
    return KVQ_ERR_INVALID;
  if (block_index_type != KVQ_INDEX_I32 && block_index_type != KVQ_INDEX_I64)
    return KVQ_ERR_INVALID;
  if ((reinterpret_cast<uintptr_t>(k_data) | reinterpret_cast<uintptr_t>(v_data)) & 3)
    return KVQ_ERR_GEOMETRY;  // a row's words
  for (int64_t b = 0; b < batch; ++b)
    if (query_lens[b] > 0 && seq_lens[b] > max_blocks * block_size) return KVQ_ERR_INVALID;
  B8Call call = make_call(query, dtype, query_stride, seq_lens, query_lens, batch, num_heads,
                          num_kv_heads, head_size, scale, window, sinks, block_size, group,
                          code_type);
  call.cache.kd = static_cast<const uint8_t*>(k_data);
  call.cache.ks = k_scale;
  call.cache.vd = static_cast<const uint8_t*>(v_data);
  call.cache.vs = v_scale;
  call.cache.table = block_table;
  call.cache.maxb = max_blocks;
  call.cache.nb = num_blocks;
  call.cache.bt64 = block_index_type == KVQ_INDEX_I64;
  call.win.cache = call.cache;
  call.win.out = out;
  call.win.stream = static_cast<hipStream_t>(stream);
  const int64_t bytes = workspace_of(call, &rc);
  if (rc != KVQ_OK) return rc;
  if (bytes > 0 && (!workspace || !aligned16(workspace, nullptr) || workspace_bytes < bytes))
    return KVQ_ERR_INVALID;
  rc = b8_decode(call, workspace);
  if (rc != KVQ_OK) return rc;
  rc = b8_chunk(call, workspace);
  if (rc != KVQ_OK) return rc;
  KVQ_DISPATCH_FLOAT(dtype, T, { rc = attend_general<T>(call, workspace); });
  return rc;
}
