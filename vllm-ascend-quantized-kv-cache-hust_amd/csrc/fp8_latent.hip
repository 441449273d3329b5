// SPDX-License-Identifier: Apache-2.0
// Causal attention of each request's new rows over paged latent rows that all heads share,
// the up-projections absorbed into the queries and into what the caller does with the
// result: the entry points, and the kernel that takes any geometry.
//
// With c_j = code[j] * scale[j] (E4M3) and r_j the rotated position part of position j,
//   p_hj = softmax over j <= pos of s (q_h[:R] . c_j + q_h[R:] . r_j),  out_h = sum_j p_hj c_j,
// R dims a head.  Rows that see nothing give zeros.
//
// The general kernel: one wave per (row, head) and run of the row's positions, 64 positions
// at a time, a lane a position for the scores, a lane eight dims for the values, fp32 with
// the softmax's running maximum and sum.  Bound by the latency of its loads and by reading
// each code once per head.
#include <algorithm>

#include "fp8_latent.h"

namespace {

using namespace kvq;

constexpr int kGenWaves = 4;
constexpr int kGenMaxD = 512, kGenMaxPart = 256;

__device__ __forceinline__ void codes4(uint32_t w, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  x[0] = lo[0];
  x[1] = lo[1];
  x[2] = hi[0];
  x[3] = hi[1];
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
latent_general_kernel(WinArg, int count, LatentCache c, const T* __restrict__ query,
                      int64_t q_stride, float qscale, int split, T* __restrict__ out,
                      WinParts parts) {
  __shared__ __align__(16) float s_q[kGenWaves][kGenMaxD + kGenMaxPart];
  const WinReq r = win_req(count, blockIdx.x);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int groups = (c.hq + kGenWaves - 1) / kGenWaves;
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int i = u / groups / r.parts, item = u / groups - i * r.parts;
  const int head = u % groups * kGenWaves + wave;
  if (head >= c.hq) return;  // no barrier below: a wave reads its own part of s_q
  const int pos = r.len - r.n + i;
  const int64_t row = static_cast<int64_t>(r.q0) + i;
  const int wide = c.d + c.part;
  const T* q = query + row * q_stride + static_cast<int64_t>(head) * wide;
  for (int k = lane; k < wide; k += 64) s_q[wave][k] = to_f32(q[k]);
  wave_lds_fence();
  // lane: words `lane` and `lane` + 64 of a latent row
  const int words = c.d / 4;
  float m = -INFINITY, l = 0.0f;
  w_f4 acc[2] = {w_f4{0.f, 0.f, 0.f, 0.f}, w_f4{0.f, 0.f, 0.f, 0.f}};
  const WinSpan span = pos >= 0 ? WinSpan::of(pos + 1, 1, c.window, 0, 64) : WinSpan{0, 0, 0};
  const int g1 = min(span.groups, (item + 1) * split);
  for (int g = item * split; g < g1; ++g) {
    const int j = span.pos(g, 64) + lane;
    const bool on = j <= pos;
    const int64_t slot = on ? c.slot(r.table, j) : 0;
    float s = -INFINITY, vs = 0.0f;
    if (on) {
      const uint8_t* k = c.kd + slot * c.d;
      vs = c.ks[slot];
      s = 0.0f;
#pragma unroll 4
      for (int e = 0; e < c.d; e += 4) {
        float x[4];
        codes4(*reinterpret_cast<const uint32_t*>(k + e), x);
#pragma unroll
        for (int t = 0; t < 4; ++t) s = __builtin_fmaf(s_q[wave][e + t], x[t], s);
      }
      s *= vs;
      const T* rope = static_cast<const T*>(c.rope) + slot * c.part;
#pragma unroll 4
      for (int e = 0; e < c.part; ++e) s = __builtin_fmaf(s_q[wave][c.d + e], to_f32(rope[e]), s);
      s *= qscale;
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
        const uint8_t* v = c.kd + __shfl(slot, t, 64) * c.d + 4 * lane;
        x[e][0] = seen && lane < words ? *reinterpret_cast<const uint32_t*>(v) : 0u;
        x[e][1] = seen && lane + 64 < words ? *reinterpret_cast<const uint32_t*>(v + 256) : 0u;
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
  return call.qlens[b] > 0 ? (call.lens[b] + 63) / 64 : 0;
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

template <typename T>
int attend_general(const LatentCall& call, void* workspace) {
  const WinCall& win = call.win;
  const LatentCache& c = call.cache;
  const int64_t groups = (c.hq + kGenWaves - 1) / kGenWaves, split = gen_split(win);
  return win_launches(
      win,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        parts = gen_parts(win, b, split);
        rows = win_part_rows(win, b, parts);
        units = win.qlens[b] * parts * groups;
        return true;
      },
      [&](const WinArg& arg, int count, int64_t blocks, int64_t rows) -> int {
        const WinParts parts{static_cast<float*>(workspace),
                             static_cast<float*>(workspace) + rows * c.d};
        hipLaunchKernelGGL((latent_general_kernel<T>), dim3(static_cast<unsigned>(blocks)),
                           dim3(64 * kGenWaves), 0, win.stream, arg, count, c,
                           static_cast<const T*>(win.query), win.q_stride, win.qscale,
                           static_cast<int>(split), static_cast<T*>(win.out), parts);
        KVQ_LAUNCH_CHECK();
        return rows > 0 ? launch_win_join(win, arg, count, parts) : KVQ_OK;
      });
}

// Lengths and geometry, checked alike by the sizing call and the call.
int check_shape(const int64_t* lens, const int64_t* qlens, int64_t batch, int dtype, int heads,
                int rank, int part, int bs) {
  if (batch < 0 || (batch > 0 && (!lens || !qlens))) return KVQ_ERR_INVALID;
  if (dtype != KVQ_DTYPE_F32 && dtype != KVQ_DTYPE_F16 && dtype != KVQ_DTYPE_BF16)
    return KVQ_ERR_INVALID;
  if (heads <= 0 || heads > 65536 || rank <= 0 || rank % 4 || rank > kGenMaxD || part <= 0 ||
      part > kGenMaxPart || bs <= 0)
    return KVQ_ERR_GEOMETRY;
  int64_t rows = 0;
  for (int64_t b = 0; b < batch; ++b) {
    if (lens[b] < 0 || lens[b] > kMaxPositions || qlens[b] < 0 || qlens[b] > kMaxPositions)
      return KVQ_ERR_INVALID;
    rows += qlens[b];
    if (rows > kMaxPositions / heads) return KVQ_ERR_INVALID;
  }
  return KVQ_OK;
}

LatentCall make_call(const void* query, int dtype, int64_t query_stride, const int64_t* seq_lens,
                     const int64_t* query_lens, int64_t batch, int heads, int rank, int part,
                     float scale, int block_size) {
  LatentCall call{};
  WinCall& win = call.win;
  win.query = query;
  win.dtype = dtype;
  win.q_stride = query_stride;
  win.lens = seq_lens;
  win.qlens = query_lens;
  win.batch = batch;
  LatentCache& c = call.cache;
  c.bs = FastDiv::make(static_cast<uint32_t>(block_size));
  c.kvh = 1;
  c.hq = heads;
  c.d = rank;
  c.part = part;
  c.rep = FastDiv::make(static_cast<uint32_t>(heads));
  c.window = kNoWindow;
  win.qscale = scale * 1.4426950408889634f;
  win.cache = c;
  return call;
}

int64_t workspace_of(const LatentCall& call, int* rc) {
  int64_t most = general_bytes(call.win);
  *rc = KVQ_OK;
  if (latent_matrix(call)) {
    most = std::max(most, latent_few_bytes(call, rc));
    if (*rc == KVQ_OK) most = std::max(most, latent_tile_bytes(call, rc));
    if (*rc != KVQ_OK) return 0;
  }
  return (most + 15) / 16 * 16;
}

}  // namespace

extern "C" int64_t kvq_fp8_latent_attn_workspace_bytes(const int64_t* seq_lens,
                                                       const int64_t* query_lens, int64_t batch,
                                                       int dtype, int num_heads, int rank,
                                                       int part_size, int block_size) {
  int rc = check_shape(seq_lens, query_lens, batch, dtype, num_heads, rank, part_size, block_size);
  if (rc != KVQ_OK) return rc;
  // (caches off a 16-byte bound need less: the size does not know the addresses)
  const LatentCall call = make_call(nullptr, dtype, 0, seq_lens, query_lens, batch, num_heads, rank,
                                    part_size, 1.0f, block_size);
  const int64_t bytes = workspace_of(call, &rc);
  return rc != KVQ_OK ? KVQ_ERR_INVALID : bytes;
}

extern "C" int kvq_fp8_latent_attn(const void* query, int dtype, int64_t query_stride,
                                   const int64_t* seq_lens, const int64_t* query_lens, int64_t batch,
                                   int num_heads, int rank, int part_size, float scale,
                                   const uint8_t* data, const float* row_scale, const void* rope,
                                   int64_t num_blocks, int block_size, const void* block_table,
                                   int block_index_type, int64_t max_blocks, void* workspace,
                                   int64_t workspace_bytes, void* out, void* stream) {
  int rc = check_shape(seq_lens, query_lens, batch, dtype, num_heads, rank, part_size, block_size);
  if (rc != KVQ_OK) return rc;
  int64_t rows = 0;
  for (int64_t b = 0; b < batch; ++b) rows += query_lens[b];
  if (rows == 0) return KVQ_OK;
  if (!query || !data || !row_scale || !rope || !block_table || !out || num_blocks <= 0 ||
      max_blocks < 0 || !(scale > 0.0f && scale < INFINITY) ||
      query_stride < static_cast<int64_t>(num_heads) * (rank + part_size))
    return KVQ_ERR_INVALID;
  if (block_index_type != KVQ_INDEX_I32 && block_index_type != KVQ_INDEX_I64)
    return KVQ_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(data) & 3) return KVQ_ERR_GEOMETRY;  // a row's words
  for (int64_t b = 0; b < batch; ++b)
    if (query_lens[b] > 0 && seq_lens[b] > max_blocks * block_size) return KVQ_ERR_INVALID;
  LatentCall call = make_call(query, dtype, query_stride, seq_lens, query_lens, batch, num_heads,
                              rank, part_size, scale, block_size);
  call.cache.kd = data;
  call.cache.ks = row_scale;
  call.cache.rope = rope;
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
  if (latent_matrix(call)) {
    const int done = latent_few_attend(call, workspace);
    return done != KVQ_OK ? done : latent_tile_attend(call, workspace);
  }
  KVQ_DISPATCH_FLOAT(dtype, T, { rc = attend_general<T>(call, workspace); });
  return rc;
}
