// SPDX-License-Identifier: Apache-2.0
// Attention over pages with block scales for requests of few rows (decode): the codes
// stream through once, bound by HBM.  32 requests of 2048 - 16384 positions, 40 heads on 8 of
// 128 (536 MB): E4M3 102 us and 5 for the join, 5.2 TB/s; INT8 109 and 5.
//
// As fp8_window_decode.hip: a unit is an item (a run of a request's visible 16-position
// groups) and some kv heads, one wave per kv head, which takes all of the request's columns
// (row, head), 16 or 32 at most; a wave's tile is two groups, double-buffered in its own LDS
// by DMA, 16-byte chunk c of row t at c ^ t % (D/16).
//   S^T = K * Q^T: A = key codes, exact in the query's type; INT8 in fp16 times 2^-9, with
//     bf16 queries raised by a power of two for each row into fp16's range (exact too).
//   softmax: a group of 16 positions has one key scale and one value scale, so the scales
//     are one fma a score, t = S ks' + log2(vs), and an offset m 14 below the running maximum
//     of t leaves p' = 2^(t - m) = p vs within fp16's range whatever the scales are: rounded
//     by 2^-11 of it, or, where fp16 is subnormal, 2^-38 of the row's largest.  Where t has
//     steps of 4 and more, m is what 14 below rounds to, or the maximum itself if that is
//     more than 15 away (2^-24 of the largest then).  Tiles and parts are joined by m, which
//     is what their sums are relative to.  (p' in 16 bits puts fp16 results up to 1.4 times as
//     far off as their own rounding does, 1.07 at 2 positions, 1.28 at 128; bf16 ones 1.01.
//     Two parts of 16 bits would double the value products.)  The sum takes p' / vs in fp32,
//     before that rounding.
//   O^T += V^T * p'^T: A = value codes, exact in fp16; one product where the scales of
//     single positions need p' in two parts.
//
// Tiles at the edges of what the columns see take the masked path: weights by selection,
// and NaN codes apart (an indicator product says which columns see one), so that what a
// row does not see cannot reach it.
#include <algorithm>

#include "block8.h"

namespace {

using namespace kvq;

constexpr int kGroup = 16;
constexpr int kTileGroups = 2;
constexpr float kRaise = 14.0f;  // log2 of the largest p'

template <int D>
constexpr int dec_tile_bytes() { return 2 * 32 * D + 256; }
// waves whose tiles a CU's LDS holds, and the most of a workgroup
template <int D>
constexpr int dec_waves() { return D == 256 ? 4 : 8; }
template <int D>
constexpr int dec_dmas() { return D / 16 + 1; }

typedef const __attribute__((address_space(4))) int32_t dec_ci32;
typedef const __attribute__((address_space(4))) int64_t dec_ci64;

// NG: groups of 16 columns, sharing the loads and conversions.
template <typename T, int D, int NG, bool INT8>
__global__ void __launch_bounds__(64 * dec_waves<D>())
__attribute__((amdgpu_waves_per_eu(dec_waves<D>() / 4, dec_waves<D>() / 4)))
b8_decode_kernel(WinArg, int count, B8Cache c, const T* __restrict__ query, int64_t q_stride,
                 int wide, float qscale, int split, int hpw, T* __restrict__ out, WinParts parts) {
  constexpr int CH = D / 16;    // 16-byte chunks of a row
  constexpr int RPI = 64 / CH;  // rows a DMA instruction brings
  constexpr int KS = D / 32;    // k-steps of a score
  constexpr int DB = D / 16;    // dims of a lane in o, and value tiles
  constexpr int W = D / 64;     // value words of a lane and row
  constexpr bool RAISE = INT8 && !std::is_same<T, f16>::value;
  using K = typename std::conditional<INT8, f16, T>::type;
  constexpr float kUnit = INT8 ? 1.0f / kInt8Unit : 1.0f;
  extern __shared__ __align__(16) char dec_lds[];
  const WinReq r = win_req(count, blockIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const int rep = static_cast<int>(c.rep.d);
  const int cols = r.n * rep;
  const int hgs = c.kvh / hpw;
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int hg = u % hgs, item = u / hgs;
  const int h = hg * hpw + wave;
  const WinSpan span = WinSpan::of(r.len, r.n, c.window, c.sinks, kGroup);
  const int g0 = item * split, g1 = min(span.groups, g0 + split);
  // the columns' rows, heads and positions; -1 sees nothing
  bool live[NG];
  int row[NG], head[NG], pos[NG];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const int col = 16 * x + n;
    live[x] = col < cols;
    row[x] = static_cast<int>(c.rep.div(static_cast<uint32_t>(live[x] ? col : 0)));
    head[x] = h * rep + (live[x] ? col : 0) - row[x] * rep;
    pos[x] = live[x] ? r.len - r.n + row[x] : -1;
  }
  const int pos_lo = r.len - r.n, pos_hi = r.len - 1;

  // ---- tiles ----
  char* const buf = dec_lds + wave * 2 * dec_tile_bytes<D>();
  const uint32_t lds0 = win_lds(buf);
  const uint32_t row_bytes = static_cast<uint32_t>(c.kvh) * D;
  // DMA instruction `part` of a group: rows RPI * part + lane / CH
  uint32_t off[16 / RPI];
#pragma unroll
  for (int part = 0; part < 16 / RPI; ++part) {
    const int t = RPI * part + lane / CH;
    off[part] = static_cast<uint32_t>(t) * row_bytes + 16 * ((lane % CH) ^ (t % CH));
  }
  const int64_t per_page = c.bs.d / c.group.d;
  // where a group's rows and its scale are, from the table by scalar loads
  struct At {
    int64_t slot, scale;
  };
  auto place = [&](int gr) -> At {
    const int p = span.pos(min(gr, g1 - 1), kGroup);
    const uint32_t i = c.bs.div(static_cast<uint32_t>(p));
    const int64_t at = __builtin_amdgcn_readfirstlane(
        static_cast<int>(i) < c.maxb ? static_cast<int>(i) : static_cast<int>(c.maxb - 1));
    const int64_t e = static_cast<int64_t>(r.table) * c.maxb + at;
    const int64_t id = c.bt64 ? ((dec_ci64*)(const void*)c.table)[e]
                              : static_cast<int64_t>(((dec_ci32*)(const void*)c.table)[e]);
    const int64_t page = id < 0 ? 0 : (id >= c.nb ? c.nb - 1 : id);
    const uint32_t in = static_cast<uint32_t>(p) - i * c.bs.d;
    return At{page * c.bs.d + in, (page * per_page + c.group.div(in)) * c.kvh + h};
  };
  auto issue = [&](int which, const At& s0, const At& s1) {
    const uint32_t lds = lds0 + which * dec_tile_bytes<D>();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t base = ((j ? s1.slot : s0.slot) * c.kvh + h) * D;
#pragma unroll
      for (int part = 0; part < 16 / RPI; ++part) {
        win_dma16(c.kd + base, off[part], lds + (16 * j + RPI * part) * D);
        win_dma16(c.vd + base, off[part], lds + 32 * D + (16 * j + RPI * part) * D);
      }
    }
    // the groups' scales, one address a lane: words 0, 1 the keys', 2, 3 the values' (the
    // other lanes bring them again)
    const float* p = (lane & 2 ? c.vs : c.ks) + (lane & 1 ? s1.scale : s0.scale);
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds + 64 * D);
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off"
                 :
                 : "v"(p), "{m0}"(m0)
                 : "memory");
  };

  At s0 = place(g0), s1 = place(g0 + 1);
  issue(0, s0, s1);
  w_u4 q[NG][KS];
  float col_scale[NG];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const T* qrow = query + (static_cast<int64_t>(r.q0) + row[x]) * q_stride +
                    static_cast<int64_t>(head[x]) * D + (D / 4) * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[x][s] = load_op8(qrow + 8 * s, wide & 1);
    col_scale[x] = qscale * kUnit;
    if constexpr (RAISE) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) top = pair_bits_max(top, q[x][s][k]);
      // (the bits of NaN and infinity too: not finite raises nothing)
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
      const float raise = query_raise(top);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) q[x][s][k] = raised_pair(q[x][s][k], raise);
      col_scale[x] *= 1.0f / raise;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
      if (!live[x]) q[x][s] = w_u4{0, 0, 0, 0};
    // landed before the loop: a wait for them inside it would be one for the DMA too
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[x][s]));
  }
  s0 = place(g0 + 2);
  s1 = place(g0 + 3);
  float m[NG], l[NG];
  w_f4 o[DB][NG];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    m[x] = -INFINITY;
    l[x] = 0.0f;
#pragma unroll
    for (int t = 0; t < DB; ++t) o[t][x] = w_f4{0.f, 0.f, 0.f, 0.f};
  }

  int which = 0;
  for (int gr = g0; gr < g1; gr += kTileGroups, which ^= 1) {
    if (gr + kTileGroups < g1) {
      issue(which ^ 1, s0, s1);
      s0 = place(gr + 4);
      s1 = place(gr + 5);
      wait_vmcnt<dec_dmas<D>()>();  // the next tile's may stay in flight
    } else {
      wait_vmcnt<0>();
    }
    const char* b = buf + which * dec_tile_bytes<D>();
    const int p0 = span.pos(gr, kGroup);
    // an item's odd last group has no second: a position nobody sees
    const int p1 = gr + 1 < g1 ? span.pos(gr + 1, kGroup) : 0x7ffffff0;
    auto all_see = [&](int p) {
      return p + 15 <= pos_lo && (p > pos_hi - c.window || p + 15 < c.sinks);
    };
    const bool whole = p1 != 0x7ffffff0 && all_see(p0) && all_see(p1);  // uniform

    // ---- scores ----
    const w_f4 sc = *reinterpret_cast<const w_f4*>(b + 64 * D);
    const B8Value val[2] = {b8_value(sc[2]), b8_value(sc[3])};
    w_f4 s[2][NG];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* kr = b + (16 * j + n) * D;
#pragma unroll
      for (int x = 0; x < NG; ++x) s[j][x] = w_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const w_u4 k = *reinterpret_cast<const w_u4*>(kr + 16 * ((W * g + w) ^ (n % CH)));
        const w_u4 k0 = b8_op8<K, INT8>(k[0], k[1]), k1 = b8_op8<K, INT8>(k[2], k[3]);
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          s[j][x] = mfma_op(k0, q[x][2 * w], s[j][x], K{});
          s[j][x] = mfma_op(k1, q[x][2 * w + 1], s[j][x], K{});
        }
      }
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const float a = sc[j] * col_scale[x];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][x][e] = __builtin_fmaf(s[j][x][e], a, val[j].lv);
      }
    }
    uint32_t seen[NG];
#pragma unroll
    for (int x = 0; x < NG; ++x) seen[x] = 0xff;
    if (!whole) {
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        seen[x] = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int p = (j ? p1 : p0) + 4 * g + e;
            const bool on = c.sees(pos[x], p);
            seen[x] |= on ? 1u << (4 * j + e) : 0u;
            s[j][x][e] = on ? s[j][x][e] : -INFINITY;
          }
      }
    }
    w_u4 bp[NG];  // p' in fp16
    const bool signs = val[0].sign != 1.0f || val[1].sign != 1.0f;  // the same in every lane
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[j][x][e]);
      mx = max_rows4(mx);
      const float raised = mx - kRaise;
      const float m_new = fmaxf(m[x], mx - raised > kRaise + 1.0f ? mx : raised);
      const float low = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = m[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[x] - low);
      m[x] = m_new;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float part = 0.0f, pv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv[e] = __builtin_amdgcn_exp2f(s[j][x][e] - low);
          part += pv[e];
        }
        sum = __builtin_fmaf(part, val[j].iv, sum);
        if (__any(signs)) {  // (none that the store writes)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            pv[e] = (seen[x] >> (4 * j + e)) & 1 ? pv[e] * val[j].sign : 0.0f;
        }
        bp[x][2 * j] = pack_pair(pv[0], pv[1], f16{});
        bp[x][2 * j + 1] = pack_pair(pv[2], pv[3], f16{});
      }
      l[x] = l[x] * alpha + sum;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int t = 0; t < DB; ++t) o[t][x] *= alpha;
      }
    }

    // ---- values ----
    uint32_t v[2][4][W];  // [group][position 4 g + e][word]
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 16 * j + 4 * g + e;
        const char* vr = b + (32 + t) * D + 16 * ((n * W / 4) ^ (t % CH)) + 4 * W * (n % (4 / W));
        if constexpr (W == 1) {
          v[j][e][0] = *reinterpret_cast<const uint32_t*>(vr);
        } else if constexpr (W == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(vr);
          v[j][e][0] = x.x;
          v[j][e][1] = x.y;
        } else {
          const w_u4 x = *reinterpret_cast<const w_u4*>(vr);
#pragma unroll
          for (int w = 0; w < 4; ++w) v[j][e][w] = x[w];
        }
      }
    // the four words x[e] of a group's positions as bytes of dim 4 w + k: tr[k]
    auto transpose = [](const uint32_t (&x)[4], uint32_t (&tr)[4]) {
      const uint32_t l01 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);
      const uint32_t h01 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
      const uint32_t l23 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
      const uint32_t h23 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
      tr[0] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
      tr[1] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
      tr[2] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
      tr[3] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
    };
    if constexpr (!INT8) {
      uint32_t odd = 0;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int w = 0; w < W; ++w) odd |= nan_codes(v[j][e][w]);
      }
      if (__any(odd != 0)) {  // an edge tile with NaN codes
        w_u4 ones[NG];        // the columns' masks as operands
#pragma unroll
        for (int x = 0; x < NG; ++x)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            ones[x][k] = ((seen[x] >> (2 * k)) & 1 ? 0x3f80u : 0u) |
                         ((seen[x] >> (2 * k + 1)) & 1 ? 0x3f800000u : 0u);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t tr[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = nan_codes(v[j][e][w]) >> 7;
              v[j][e][w] &= ~(x[e] * 0xffu);
              x[e] *= 0x38u;  // the code of 1
            }
            transpose(x, tr[j]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int x = 0; x < NG; ++x) {
              const w_f4 hit = mfma_op(code_op8<bf16>(tr[0][k], tr[1][k]), ones[x],
                                       w_f4{0.f, 0.f, 0.f, 0.f}, bf16{});
              w_f4& acc = o[4 * w + k][x];
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[e] = hit[e] > 0.0f ? NAN : acc[e];
            }
        }
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      uint32_t tr[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x[4] = {v[j][0][w], v[j][1][w], v[j][2][w], v[j][3][w]};
        transpose(x, tr[j]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const w_u4 a = b8_op8<f16, INT8>(tr[0][k], tr[1][k]);
#pragma unroll
        for (int x = 0; x < NG; ++x) o[4 * w + k][x] = mfma_op(a, bp[x], o[4 * w + k][x], f16{});
      }
    }
    // this buffer's reads are consumed before the DMA two tiles on overwrites it
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (hpw > 1) __builtin_amdgcn_s_barrier();  // the workgroup's heads share the item
  }

  // ---- results: o[t][x][e] is dim DB * (4 g + e) + t of the column ----
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const float sum = sum_rows4(l[x]);
    if (!live[x]) continue;
    const int64_t at = (static_cast<int64_t>(r.q0) + row[x]) * c.hq + head[x];
    if (r.parts == 1) {
      const float inv = sum == 0.0f ? 0.0f : kUnit / sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        T* dst = out + at * D + DB * (4 * g + e);
        uint32_t w[DB / 2];
#pragma unroll
        for (int t = 0; t < DB; t += 2)
          w[t / 2] = pack_pair(o[t][x][e] * inv, o[t + 1][x][e] * inv, T{});
        if (wide & 2) {
          if constexpr (DB == 4)
            *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
          else
#pragma unroll
            for (int t = 0; t < DB / 8; ++t)
              reinterpret_cast<uint4*>(dst)[t] =
                  make_uint4(w[4 * t], w[4 * t + 1], w[4 * t + 2], w[4 * t + 3]);
        } else {
          uint16_t* d16 = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
          for (int t = 0; t < DB / 2; ++t) {
            d16[2 * t] = static_cast<uint16_t>(w[t]);
            d16[2 * t + 1] = static_cast<uint16_t>(w[t] >> 16);
          }
        }
      }
      continue;
    }
    const int64_t part = r.part0 + (static_cast<int64_t>(item) * r.n + row[x]) * c.hq + head[x];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float* dst = parts.o + part * D + DB * (4 * g + e);
#pragma unroll
      for (int t = 0; t < DB; t += 4)
        *reinterpret_cast<w_f4*>(dst + t) =
            kUnit * w_f4{o[t][x][e], o[t + 1][x][e], o[t + 2][x][e], o[t + 3][x][e]};
    }
    if (g == 0)  // a NaN score leaves m without it, but not l
      *reinterpret_cast<w_f2*>(parts.ml + 2 * part) = w_f2{sum != sum ? INFINITY : m[x], sum};
  }
}

// ---- host -----------------------------------------------------------------------

int dec_hpw(int kvh, int d) {
  const int most = d == 256 ? 4 : 8;
  int hpw = std::min(kvh, most);
  while (kvh % hpw) --hpw;
  return hpw;
}

// Groups per item: one workgroup of heads per slot of the chip (two waves a SIMD, or
// as many as the LDS holds) while items stay long enough to be worth their partial
// results.
template <typename F>
int64_t dec_split(const WinCall& call, int cus, F&& groups) {
  const WinCache& c = call.cache;
  const int64_t waves = c.d == 256 ? 4 : 8;
  int64_t total = 0, requests = 0, cells = 0;  // (group, row, head)s
  for (int64_t b = 0; b < call.batch; ++b) {
    const int64_t n = groups(b);
    total += n;
    cells += n * call.qlens[b] * c.hq;
    requests += n > 0;
  }
  const int64_t target = std::max<int64_t>(1, cus * waves / c.kvh);
  // items of 4 groups, or of 8 where those of 4 leave 8 MB of partial results
  const int64_t least = cells / 4 * c.d * 4 > 8 << 20 ? 8 : 4;
  int64_t split = std::max<int64_t>(least, ((total + target - 1) / target + 1) / 2 * 2);
  auto items = [&](int64_t s) {
    int64_t n = 0;
    for (int64_t b = 0; b < call.batch; ++b) n += (groups(b) + s - 1) / s;
    return n;
  };
  while (split < 4096 && items(split) > std::max(target, requests)) split += (split / 16 + 1) * 2;
  return split;
}

bool dec_few(const WinCall& call, int64_t b) {
  return call.lens[b] > 0 && call.qlens[b] > 0 && call.qlens[b] * call.cache.rep.d <= call.few_cols;
}

int64_t dec_groups(const B8Call& call, int64_t b) {
  const WinCall& win = call.win;
  if (win.qlens[b] <= 0 || !b8_decode_takes(call, b)) return 0;
  return WinSpan::of(static_cast<int>(win.lens[b]), static_cast<int>(win.qlens[b]),
                     win.cache.window, win.cache.sinks, kGroup)
      .groups;
}

template <typename G>
int dec_launches(const B8Call& call, int64_t* split_out, G&& go) {
  int cus = 0;
  const int rc = device_cu_count(&cus);
  if (rc != KVQ_OK) return rc;
  if (cus <= 0) cus = 256;
  const WinCall& win = call.win;
  const int64_t split = dec_split(win, cus, [&](int64_t b) { return dec_groups(call, b); });
  if (split_out) *split_out = split;
  const int hgs = win.cache.kvh / dec_hpw(win.cache.kvh, win.cache.d);
  return win_launches(
      win,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        const int64_t groups = dec_groups(call, b);
        parts = (groups + split - 1) / split;
        rows = win_part_rows(win, b, parts);
        units = parts * hgs;
        return groups > 0;
      },
      go);
}

}  // namespace

namespace kvq {

bool b8_decode_takes(const B8Call& call, int64_t b) {
  return !call.win.tiles_only && dec_few(call.win, b) && b8_matrix(call);
}

// In a batch with chunks, requests of few rows ride with their tiles where they see no
// more than the chunks do and all tiles run at once: a launch less.
bool b8_tiles_only(const B8Call& call) {
  if (!b8_matrix(call)) return false;
  const WinCall& win = call.win;
  const WinCache& c = win.cache;
  int64_t few = 0, many = 0, tiles = 0;  // most positions seen by either kind
  for (int64_t b = 0; b < win.batch; ++b) {
    if (win.lens[b] <= 0 || win.qlens[b] <= 0) continue;
    const int64_t seen = WinSpan::of(static_cast<int>(win.lens[b]), static_cast<int>(win.qlens[b]),
                                     c.window, c.sinks, kGroup).groups;
    int64_t& most = dec_few(win, b) ? few : many;
    most = std::max(most, seen);
    tiles += (win.qlens[b] * c.rep.d + 127) / 128;
  }
  int cus = 0;
  if (device_cu_count(&cus) != KVQ_OK || cus <= 0) cus = 256;
  return few > 0 && few <= many && tiles * c.kvh <= cus;
}

int64_t b8_decode_bytes(const B8Call& call, int* rc) {
  int64_t most = 0;
  *rc = dec_launches(call, nullptr,
                     [&](const WinArg&, int, int64_t, int64_t rows) -> int {
                       most = std::max(most, win_parts_bytes(rows, call.cache.d));
                       return KVQ_OK;
                     });
  return most;
}

int b8_decode(const B8Call& call, void* workspace) {
  const WinCall& win = call.win;
  const B8Cache& c = call.cache;
  const int hpw = dec_hpw(c.kvh, c.d);
  const int wide = (win.q_wide() ? 1 : 0) | (aligned16(win.out, nullptr) ? 2 : 0);
  int64_t split = 0;
  return dec_launches(call, &split, [&](const WinArg& arg, int count, int64_t units, int64_t rows) -> int {
    const WinParts parts{static_cast<float*>(workspace),
                         static_cast<float*>(workspace) + rows * c.d};
#define KVQ_B8_DECODE(T, D, NG, I)                                                             \
  hipLaunchKernelGGL((b8_decode_kernel<T, D, NG, I>), dim3(static_cast<unsigned>(units)),      \
                     dim3(64 * hpw), hpw * 2 * dec_tile_bytes<D>(), win.stream, arg, count, c, \
                     static_cast<const T*>(win.query), win.q_stride, wide, win.qscale,         \
                     static_cast<int>(split), hpw, static_cast<T*>(win.out), parts)
#define KVQ_B8_DECODE_I(T, D, NG) \
  if (c.int8)                     \
    KVQ_B8_DECODE(T, D, NG, true); \
  else                            \
    KVQ_B8_DECODE(T, D, NG, false)
#define KVQ_B8_DECODE_N(T, D)    \
  if (win.few_cols > 16) {       \
    KVQ_B8_DECODE_I(T, D, 2);    \
  } else {                       \
    KVQ_B8_DECODE_I(T, D, 1);    \
  }
#define KVQ_B8_DECODE_D(T)       \
  if (c.d == 256) {              \
    KVQ_B8_DECODE_N(T, 256)      \
  } else if (c.d == 128) {       \
    KVQ_B8_DECODE_N(T, 128)      \
  } else {                       \
    KVQ_B8_DECODE_N(T, 64)       \
  }
    if (win.dtype == KVQ_DTYPE_BF16) {
      KVQ_B8_DECODE_D(bf16)
    } else {
      KVQ_B8_DECODE_D(f16)
    }
#undef KVQ_B8_DECODE_D
#undef KVQ_B8_DECODE_N
#undef KVQ_B8_DECODE_I
#undef KVQ_B8_DECODE
    KVQ_LAUNCH_CHECK();
    return rows > 0 ? launch_win_join(win, arg, count, parts) : KVQ_OK;
  });
}

}  // namespace kvq
