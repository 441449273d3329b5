// SPDX-License-Identifier: Apache-2.0
// Attention over latent rows that all heads share, on the matrix units, where a request has
// few columns: decodes of few heads, where memory bounds it and the rows stream through once.
//
// One workgroup of eight waves per tile of 16 or 32 columns (row, head), request and part of
// its positions, 128 positions at a time.  The latent is key and value at once, so a stage's
// codes are read from memory once, by DMA into LDS (64 KB at R = 512, two stages, 16-byte
// chunk c of row t at c ^ t % 16), and converted to 16 bits on their way to the matrix units:
//   S^T = C * Q^T: wave w takes positions 16 w ..; A = codes in the query's type, exact: lane
//     (g, n) holds dims R/4 g .. of position n; B = the queries, all R dims of the tile's
//     columns in every wave's registers.  The position part beside it, from 16 KB of its own.
//   softmax: the waves put their positions' maxima into LDS; with t = (S s_j + S_r) scale
//     log2(e) + log2(s_j) and an offset m 14 below its running maximum, p' = 2^(t - m) = p s_j
//     fits fp16 whatever the scales are: rounded by 2^-11 of it, or, where fp16 is subnormal,
//     2^-38 of the row's largest; the sum takes p' / s_j in fp32 before that rounding.  Where
//     t has steps of 4 and more, m is what 14 below rounds to, or the maximum itself if that
//     is more than 15 away (2^-24 of the largest then).  Stages and parts are joined by m,
//     which is what their sums are relative to.  p' goes through LDS to all waves.  (In 16
//     bits it puts fp16 results up to 1.4 times as far off as their own rounding does, bf16
//     ones 1.01.)
//   O^T += C^T * p'^T: wave w takes dims R/8 w ..; A = codes in fp16, exact, by the transposing
//     reads of bytes (16 lanes read 8 rows of 16 bytes, lane s gets column s).
//
// 32 requests of 2048 - 16384 positions, 16 heads, R = 512, P = 64 (177 MB): 36 us, 5.0 TB/s, and
// 5 for the join, of a call that takes 46, for its host takes 41.
//
// Positions that a column does not see: weights by selection; in stages that some column
// does not wholly see, NaN codes become zeros in LDS between the two products (a row that
// sees one is NaN by its score).
#include <algorithm>

#include "fp8_latent.h"
#include "block8.h"

namespace {

using namespace kvq;

constexpr int kWaves = 8;
constexpr int kStage = 16 * kWaves;  // positions
constexpr float kRaise = 14.0f;      // log2 of the largest p'

typedef const __attribute__((address_space(4))) int32_t lat_ci32;
typedef const __attribute__((address_space(4))) int64_t lat_ci64;
typedef int lat_i2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) lat_i2* lat_lds2;
typedef const __attribute__((address_space(3))) w_u4* lat_cu4;

template <int R, int PART, int NG>
struct LatLds {
  static constexpr int STAGE = kStage * R;
  static constexpr int ROPE = 2 * STAGE;              // [kStage][PART] of 16 bits
  static constexpr int PROW = 2 * kStage + 16;        // bytes of a column's p', padded
  static constexpr int P = ROPE + 2 * kStage * PART;  // [16 NG][PROW]
  static constexpr int MAX = P + 16 * NG * PROW;      // [16 NG][kWaves] floats
  static constexpr int BYTES = MAX + 16 * NG * kWaves * 4;
};

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <typename T, int R, int PART, int NG>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
latent_few_kernel(WinArg, int count, LatentCache c, const T* __restrict__ query,
                     int64_t q_stride, int wide, float qscale, T* __restrict__ out, WinParts parts) {
  using L = LatLds<R, PART, NG>;
  constexpr int KS = R / 32;      // k-steps of a score
  constexpr int RS = PART / 32;   // and of its position part
  constexpr int DB = R / 128;     // 16-dim blocks of a wave's dims
  constexpr int CH = R / 16;      // 16-byte chunks of a row
  constexpr int RPI = 64 / CH;    // rows a DMA instruction brings
  constexpr int DMAS = 16 / RPI;  // of a wave's 16 rows
  extern __shared__ __align__(16) char lds[];
  const WinReq r = win_req(count, blockIdx.x);
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int heads = c.hq, cols = r.n * heads;
  const int tiles = (cols + 16 * NG - 1) / (16 * NG);
  // tiles of a part lie 8 workgroups apart, on one XCD, whose L2 then holds its codes once
  int u = static_cast<int>(blockIdx.x) - r.first;
  const int set = u / (8 * tiles);
  u -= set * 8 * tiles;
  const int across = min(8, r.parts - 8 * set);
  const int tile = tiles - 1 - u / across, seg = 8 * set + u % across;
  const int col0 = 16 * NG * tile;
  auto row_of = [&](int col) { return static_cast<int>(c.rep.div(static_cast<uint32_t>(col))); };
  const int base = r.len - r.n;  // position of the request's first row
  const int tile_first = base + row_of(col0);
  const int tile_last = base + row_of(min(col0 + 16 * NG, cols) - 1);
  // the lane's column of group x, found where it is needed (held, these would cost registers);
  // one past the last sees nothing
  struct Col {
    bool live;
    int row, head, pos;
  };
  auto col_at = [&](int x) {
    int col = col0 + 16 * x + n;
    asm volatile("" : "+v"(col));  // found anew
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
    for (int x = tid; x < 16 * NG * (R / 4); x += 64 * kWaves) {
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

  // ---- a stage on its way ----
  const uint32_t lds0 = win_lds(lds);
  // instruction j brings rows RPI j + lane / CH: off ^ 16 RPI j from its first one's start
  const uint32_t off = static_cast<uint32_t>(lane / CH) * R + 16 * ((lane % CH) ^ (lane / CH));
  // position parts: chunk c of row t at c ^ t % RC, a wave's own rows
  constexpr int RC = PART / 8;
  const uint32_t rope_off =
      static_cast<uint32_t>(lane / RC) * 2 * PART + 16 * ((lane % RC) ^ (lane / RC % RC));
  const uint32_t rope_lds = lds0 + L::ROPE + wave * 32 * PART;
  const int groups = (r.len + 15) / 16;  // 16-position groups, each in one page
  // slot of this wave's positions
  auto slot_of = [&](int stage) -> int64_t {
    const int p = 16 * min(stage * kWaves + wave, groups - 1);
    const uint32_t i = c.bs.div(static_cast<uint32_t>(p));
    const int64_t at = __builtin_amdgcn_readfirstlane(
        static_cast<int>(i) < c.maxb ? static_cast<int>(i) : static_cast<int>(c.maxb - 1));
    const int64_t e = static_cast<int64_t>(r.table) * c.maxb + at;
    const int64_t id = c.bt64 ? ((lat_ci64*)(const void*)c.table)[e]
                              : static_cast<int64_t>(((lat_ci32*)(const void*)c.table)[e]);
    const int64_t page = id < 0 ? 0 : (id >= c.nb ? c.nb - 1 : id);
    return page * c.bs.d + (static_cast<uint32_t>(p) - i * c.bs.d);
  };
  auto issue = [&](int stage, int64_t slot) {
    const uint32_t to = lds0 + stage % 2 * L::STAGE + wave * 16 * R;
#pragma unroll
    for (int j = 0; j < DMAS; ++j)
      win_dma16(c.kd + slot * R + j * 1024, off ^ (16 * RPI * j), to + j * 1024);
    return *reinterpret_cast<const w_f4*>(c.ks + slot + 4 * g);
  };
  auto issue_rope = [&](int64_t slot) {
#pragma unroll
    for (int s = 0; s < RS; ++s)
      win_dma16(static_cast<const T*>(c.rope) + slot * PART + 512 * s, rope_off, rope_lds + 1024 * s);
  };

  int64_t slot = slot_of(s0);
  w_f4 next = issue(s0, slot);
  issue_rope(slot);
  w_u4 q[NG][KS], qr[NG][RS];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const Col y = col_at(x);
    const T* qrow = query + (static_cast<int64_t>(r.q0) + y.row) * q_stride +
                    static_cast<int64_t>(y.head) * (R + PART);
#pragma unroll
    for (int s = 0; s < KS; ++s) q[x][s] = load_op8(qrow + (R / 4) * g + 8 * s, wide & 1);
#pragma unroll
    for (int s = 0; s < RS; ++s) qr[x][s] = load_op8(qrow + R + 32 * s + 8 * g, wide & 1);
    if (!y.live) {
#pragma unroll
      for (int s = 0; s < KS; ++s) q[x][s] = w_u4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < RS; ++s) qr[x][s] = w_u4{0, 0, 0, 0};
    }
  }
  float m[NG], l[NG];
  w_f4 o[DB][NG];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    m[x] = -INFINITY;
    l[x] = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d][x] = w_f4{0.f, 0.f, 0.f, 0.f};
  }
  float* const smax = reinterpret_cast<float*>(lds + L::MAX);

  for (int st = s0; st < s1; ++st) {
    wait_vmcnt<0>();  // this wave's part of the stage
    lds_barrier();    // everybody's; and the last stage's other buffer is read
    w_f4 scale = next;
    asm volatile("" : "+v"(scale));
    if (st + 1 < s1) {
      slot = slot_of(st + 1);
      next = issue(st + 1, slot);
    }
    char* const codes = lds + st % 2 * L::STAGE;
    const int p0 = st * kStage + 16 * wave;  // of this wave's positions
    const bool edge = st * kStage + kStage - 1 > tile_first;  // uniform

    // ---- scores ----
    w_f4 s[NG], sr[NG];
#pragma unroll
    for (int x = 0; x < NG; ++x) s[x] = sr[x] = w_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < RS; ++i) {
      const w_u4 k = *(lat_cu4)(rope_lds + n * 2 * PART + 16 * ((4 * i + g) ^ (n % RC)));
#pragma unroll
      for (int x = 0; x < NG; ++x) sr[x] = mfma_op(k, qr[x][i], sr[x], T{});
    }
    const uint32_t kr = win_lds(codes) + (16 * wave + n) * R + 16 * ((CH / 4 * g) ^ n);
#pragma unroll
    for (int w = 0; w < KS / 2; ++w) {
      const w_u4 k = *(lat_cu4)(kr ^ (16 * w));
      const w_u4 k0 = code_op8<T>(k[0], k[1]), k1 = code_op8<T>(k[2], k[3]);
#pragma unroll
      for (int x = 0; x < NG; ++x) s[x] = mfma_op(k0, q[x][2 * w], s[x], T{});
#pragma unroll
      for (int x = 0; x < NG; ++x) s[x] = mfma_op(k1, q[x][2 * w + 1], s[x], T{});
    }
    // b8_value's logarithms without a branch: behind one, the compiler has not always kept the
    // distance that a product's result needs (a scale that is not finite spoils its rows anyway)
    w_f4 lv;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      lv[e] = __builtin_amdgcn_logf(
          __builtin_amdgcn_fmed3f(fabsf(scale[e]), 0x1p-90f, 0x1.fffffep127f));
#pragma unroll
    for (int x = 0; x < NG; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[x][e] = __builtin_fmaf(s[x][e], scale[e] * qscale,
                                 __builtin_fmaf(sr[x][e], qscale, lv[e]));
    uint32_t seen[NG];
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      seen[x] = 0xf;
      if (edge) {
        seen[x] = 0;
        const int pos = col_at(x).pos;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool on = p0 + 4 * g + e <= pos;
          seen[x] |= on ? 1u << e : 0u;
          s[x][e] = on ? s[x][e] : -INFINITY;
        }
      }
      const float mx = max_rows4(fmaxf(fmaxf(s[x][0], s[x][1]), fmaxf(s[x][2], s[x][3])));
      if (g == 0) smax[(16 * x + n) * kWaves + wave] = mx;
    }
    lds_barrier();  // the maxima; and the codes are read as keys
    if (st + 1 < s1) issue_rope(slot);

    // ---- weights ----
    w_f4 iv;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      iv[e] = __builtin_amdgcn_rcpf(scale[e]);
      odd = odd || !(scale[e] >= 0x1p-90f && scale[e] < INFINITY);
    }
    const bool odds = __any(odd);  // (none that the store writes)
    if (odds) {
#pragma unroll
      for (int e = 0; e < 4; ++e) iv[e] = b8_value(scale[e]).iv;
    }
    float alpha[NG];
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      const w_f4* y = reinterpret_cast<const w_f4*>(smax + (16 * x + n) * kWaves);
      const w_f4 a = y[0], z = y[1];
      const float mx = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])),
                             fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
      const float raised = mx - kRaise;
      const float m_new = fmaxf(m[x], mx - raised > kRaise + 1.0f ? mx : raised);
      const float from = m_new == -INFINITY ? 0.0f : m_new;
      alpha[x] = m[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[x] - from);
      m[x] = m_new;
      float pv[4], sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pv[e] = __builtin_amdgcn_exp2f(s[x][e] - from);
        sum = __builtin_fmaf(pv[e], iv[e], sum);
      }
      if (odds) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pv[e] = (seen[x] >> e) & 1 ? pv[e] * b8_value(scale[e]).sign : 0.0f;
      }
      l[x] = l[x] * alpha[x] + sum;
      *reinterpret_cast<uint2*>(lds + L::P + (16 * x + n) * L::PROW + 2 * (16 * wave + 4 * g)) =
          make_uint2(pack_pair(pv[0], pv[1], f16{}), pack_pair(pv[2], pv[3], f16{}));
    }
    if (edge) {  // NaN codes of this wave's rows
#pragma unroll
      for (int j = 0; j < DMAS; ++j) {
        w_u4* p = reinterpret_cast<w_u4*>(codes + wave * 16 * R + j * 1024 + 16 * lane);
        w_u4 w = *p;
        const uint32_t odd = nan_codes(w[0]) | nan_codes(w[1]) | nan_codes(w[2]) | nan_codes(w[3]);
        if (odd) {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] &= ~((nan_codes(w[k]) >> 7) * 0xffu);
          *p = w;
        }
      }
    }
    lds_barrier();

    // ---- values ----
#pragma unroll
    for (int x = 0; x < NG; ++x)
      if (__any(alpha[x] != 1.0f)) {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d][x] *= alpha[x];
      }
#pragma unroll
    for (int k = 0; k < kStage / 32; ++k) {
      w_u4 p[NG];
#pragma unroll
      for (int x = 0; x < NG; ++x)
        p[x] = *reinterpret_cast<const w_u4*>(lds + L::P + (16 * x + n) * L::PROW +
                                              2 * (32 * k + 8 * g));
      const int t = 32 * k + 8 * g + n / 2;  // the row this lane addresses
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int chunk = (DB * wave + d) ^ (t % 16);
        const lat_i2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lat_lds2)(codes + t * R + 16 * chunk + 8 * (n % 2)));
        const w_u4 a = code_op8<f16>(static_cast<uint32_t>(v[0]), static_cast<uint32_t>(v[1]));
#pragma unroll
        for (int x = 0; x < NG; ++x) o[d][x] = mfma_op(a, p[x], o[d][x], f16{});
      }
    }
  }

  // ---- results: o[d][x][e] is dim R/8 wave + 16 d + 4 g + e of the column ----
  lds_barrier();  // the maxima's place is read
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const float sum = sum_rows4(l[x]);
    if (g == 0) smax[(16 * x + n) * kWaves + wave] = sum;
  }
  lds_barrier();
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += smax[(16 * x + n) * kWaves + w];
    const Col y = col_at(x);
    if (!y.live) continue;
    const int dim = R / 8 * wave + 4 * g;
    if (r.parts > 1) {
      const int64_t part =
          r.part0 + (static_cast<int64_t>(seg) * r.n + y.row) * heads + y.head;
#pragma unroll
      for (int d = 0; d < DB; ++d)
        *reinterpret_cast<w_f4*>(parts.o + part * R + dim + 16 * d) = o[d][x];
      if (g == 0 && wave == 0)  // a NaN score leaves m without it, but not l
        *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{sum != sum ? INFINITY : m[x], sum};
      continue;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* dst = out + ((static_cast<int64_t>(r.q0) + y.row) * heads + y.head) * R + dim;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint32_t lo = pack_pair(o[d][x][0] * inv, o[d][x][1] * inv, T{});
      const uint32_t hi = pack_pair(o[d][x][2] * inv, o[d][x][3] * inv, T{});
      if (wide & 2) {
        *reinterpret_cast<uint2*>(dst + 16 * d) = make_uint2(lo, hi);
      } else {
        uint16_t* d16 = reinterpret_cast<uint16_t*>(dst + 16 * d);
        d16[0] = static_cast<uint16_t>(lo);
        d16[1] = static_cast<uint16_t>(lo >> 16);
        d16[2] = static_cast<uint16_t>(hi);
        d16[3] = static_cast<uint16_t>(hi >> 16);
      }
    }
  }
}

// ---- host -----------------------------------------------------------------------

// Columns of a tile: 32, or 16 where no request has more.
LatentShape few_shape(const LatentCall& call) {
  int cols = 16;
  for (int64_t b = 0; b < call.win.batch; ++b)
    if (latent_few(call, b) && call.win.qlens[b] * call.cache.hq > 16) cols = 32;
  return LatentShape{true, cols, kStage, 2, 3, 6000000};
}

}  // namespace

namespace kvq {

bool latent_matrix(const LatentCall& call) {
  const LatentCache& c = call.cache;
  return (call.win.dtype == KVQ_DTYPE_BF16 || call.win.dtype == KVQ_DTYPE_F16) &&
         (c.d == 256 || c.d == 512) && (c.part == 32 || c.part == 64) && c.bs.d % 16 == 0 &&
         aligned16(c.kd, c.ks) && aligned16(c.rope, nullptr);
}

int64_t latent_few_bytes(const LatentCall& call, int* rc) {
  int64_t most = 0;
  *rc = latent_launches(call, few_shape(call),
                        [&](const WinArg&, int, int64_t, int64_t rows) -> int {
                          most = std::max(most, win_parts_bytes(rows, call.cache.d));
                          return KVQ_OK;
                        });
  return most;
}

int latent_few_attend(const LatentCall& call, void* workspace) {
  const WinCall& win = call.win;
  const LatentCache& c = call.cache;
  const int wide = (win.q_wide() ? 1 : 0) | (aligned16(win.out, nullptr) ? 2 : 0);
  const LatentShape shape = few_shape(call);
  const int cols = shape.cols;
  return latent_launches(call, shape, [&](const WinArg& arg, int count, int64_t units, int64_t rows) -> int {
    const WinParts parts{static_cast<float*>(workspace),
                         static_cast<float*>(workspace) + rows * c.d};
#define KVQ_LATENT(T, R, P, NG)                                                                \
  hipLaunchKernelGGL((latent_few_kernel<T, R, P, NG>), dim3(static_cast<unsigned>(units)),  \
                     dim3(64 * kWaves), (LatLds<R, P, NG>::BYTES), win.stream, arg, count, c,     \
                     static_cast<const T*>(win.query), win.q_stride, wide, win.qscale,         \
                     static_cast<T*>(win.out), parts)
#define KVQ_LATENT_N(T, R, P)   \
  if (cols == 32)               \
    KVQ_LATENT(T, R, P, 2);     \
  else                          \
    KVQ_LATENT(T, R, P, 1)
#define KVQ_LATENT_P(T, R)      \
  if (c.part == 64) {           \
    KVQ_LATENT_N(T, R, 64);     \
  } else {                      \
    KVQ_LATENT_N(T, R, 32);     \
  }
#define KVQ_LATENT_R(T)         \
  if (c.d == 512) {             \
    KVQ_LATENT_P(T, 512)        \
  } else {                      \
    KVQ_LATENT_P(T, 256)        \
  }
    if (win.dtype == KVQ_DTYPE_BF16) {
      KVQ_LATENT_R(bf16)
    } else {
      KVQ_LATENT_R(f16)
    }
#undef KVQ_LATENT_R
#undef KVQ_LATENT_P
#undef KVQ_LATENT_N
#undef KVQ_LATENT
    KVQ_LAUNCH_CHECK();
    return rows > 0 ? launch_win_join(win, arg, count, parts) : KVQ_OK;
  });
}

}  // namespace kvq
