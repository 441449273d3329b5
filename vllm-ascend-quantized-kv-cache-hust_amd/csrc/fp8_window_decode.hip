// SPDX-License-Identifier: Apache-2.0
// Windowed attention over paged E4M3 rows for requests of few rows (decode): the
// codes stream through once, bound by HBM.
//
// A unit is an item (a run of a request's visible 16-position groups) and some kv heads,
// one wave per kv head, which takes all of the request's columns (row, head): at most 16
// or 32.  The waves of a workgroup step through the item together, so that the rows of
// one token, which its heads' codes share DRAM pages for, are requested together.
//
// A wave's tile is two groups of 16 positions, double-buffered in its own LDS by
// DMA (16 bytes a lane, whole rows; 16-byte chunk c of row t sits at c ^ t % (D/16),
// which spreads the operand reads over the banks):
//   S^T = K * Q^T: A = key codes converted to the query's type, exact; lane (g, n)
//     of the wave holds bytes D/4 g .. of position n of the group, so k-step s takes
//     dims D/4 g + 8 s ..; B = the query as it is.  The key's scale multiplies the
//     fp32 score, with the softmax scale and log2(e).
//   softmax: a lane holds 8 positions of its column; online maximum and sum in fp32.
//   O^T += V^T * P^T: B = p * value scale as bf16 hi + lo parts (16 bits of it, any
//     range) straight from the score registers; A = value codes, exact in bf16: the
//     lane's 8 positions' bytes D/16 n .., transposed 4 x 4 by v_perm.
// Neither rounds a key or a value, and both leave the column in the same lanes, so
// the rescale needs no lane exchange.
//
// 32 requests of 2048 - 16384 positions, 40 heads on 8 of 128: 120 us, 5.4 TB/s, where a
// large copy reaches 5.2; 64 of 4096 - 16384 with a window of 4096: 103 us, 5.4 TB/s.  One
// request of 600: 7 us and 4 to join, the rest of its 22 the host's.
//
// Tiles at the edges of what the columns see take the masked path: weights by
// selection, and NaN codes apart (an indicator product says which columns see one),
// so that what a row does not see cannot reach it.
#include <algorithm>

#include "fp8_window.h"

namespace {

using namespace kvq;

constexpr int kGroup = 16;
constexpr int kTileGroups = 2;

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
template <typename T, int D, int NG>
__global__ void __launch_bounds__(64 * dec_waves<D>())
__attribute__((amdgpu_waves_per_eu(dec_waves<D>() / 4, dec_waves<D>() / 4)))
win_decode_kernel(WinArg, int count, WinCache c, const T* __restrict__ query, int64_t q_stride,
                  int wide, float qscale, int split, int hpw, T* __restrict__ out,
                  WinParts parts, float* __restrict__ lse, float* __restrict__ scores) {
  constexpr int CH = D / 16;    // 16-byte chunks of a row
  constexpr int RPI = 64 / CH;  // rows a DMA instruction brings
  constexpr int KS = D / 32;    // k-steps of a score
  constexpr int DB = D / 16;    // dims of a lane in o, and value tiles
  constexpr int W = D / 64;     // value words of a lane and row
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
  const uint32_t soff = 4u * static_cast<uint32_t>(lane & 15) * static_cast<uint32_t>(c.kvh);
  // slots of the tile's two groups, from the table by scalar loads
  auto slot = [&](int gr) -> int64_t {
    const int p = span.pos(min(gr, g1 - 1), kGroup);
    const uint32_t i = c.bs.div(static_cast<uint32_t>(p));
    const int64_t at = __builtin_amdgcn_readfirstlane(
        static_cast<int>(i) < c.maxb ? static_cast<int>(i) : static_cast<int>(c.maxb - 1));
    const int64_t e = static_cast<int64_t>(r.table) * c.maxb + at;
    const int64_t id = c.bt64 ? ((dec_ci64*)(const void*)c.table)[e]
                              : static_cast<int64_t>(((dec_ci32*)(const void*)c.table)[e]);
    const int64_t page = id < 0 ? 0 : (id >= c.nb ? c.nb - 1 : id);
    return page * c.bs.d + (static_cast<uint32_t>(p) - i * c.bs.d);
  };
  auto issue = [&](int which, int64_t s0, int64_t s1) {
    const uint32_t lds = lds0 + which * dec_tile_bytes<D>();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t base = ((j ? s1 : s0) * c.kvh + h) * D;
#pragma unroll
      for (int part = 0; part < 16 / RPI; ++part) {
        win_dma16(c.kd + base, off[part], lds + (16 * j + RPI * part) * D);
        win_dma16(c.vd + base, off[part], lds + 32 * D + (16 * j + RPI * part) * D);
      }
    }
    // scales of the 32 positions: lanes 0-15 and 16-31 the keys' of the two groups,
    // 32-63 the values'
    const int64_t f0 = 4 * (s0 * c.kvh + h), f1 = 4 * (s1 * c.kvh + h);
    const char* k = reinterpret_cast<const char*>(c.ks);
    const char* v = reinterpret_cast<const char*>(c.vs);
    // one address per lane: the four runs lie anywhere
    const char* p = (lane & 32 ? v : k) + (lane & 16 ? f1 : f0) + soff;
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds + 64 * D);
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off"
                 :
                 : "v"(p), "{m0}"(m0)
                 : "memory");
  };

  int64_t s0 = slot(g0), s1 = slot(g0 + 1);
  issue(0, s0, s1);
  w_u4 q[NG][KS];
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const T* qrow = query + (static_cast<int64_t>(r.q0) + row[x]) * q_stride +
                    static_cast<int64_t>(head[x]) * D + (D / 4) * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[x][s] = load_op8(qrow + 8 * s, wide & 1);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      if (!live[x]) q[x][s] = w_u4{0, 0, 0, 0};
    // landed before the loop: a wait for them inside it would be one for the DMA too
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[x][s]));
  }
  s0 = slot(g0 + 2);
  s1 = slot(g0 + 3);
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
      s0 = slot(gr + 4);
      s1 = slot(gr + 5);
      wait_vmcnt<dec_dmas<D>()>();  // the next tile's may stay in flight
    } else {
      wait_vmcnt<0>();
    }
    const char* b = buf + which * dec_tile_bytes<D>();
    const float* sc = reinterpret_cast<const float*>(b + 64 * D);
    const int p0 = span.pos(gr, kGroup);
    // an item's odd last group has no second: a position nobody sees
    const int p1 = gr + 1 < g1 ? span.pos(gr + 1, kGroup) : 0x7ffffff0;
    auto all_see = [&](int p) {
      return p + 15 <= pos_lo && (p > pos_hi - c.window || p + 15 < c.sinks);
    };
    const bool whole = p1 != 0x7ffffff0 && all_see(p0) && all_see(p1);  // uniform

    // ---- scores ----
    w_f4 s[2][NG];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* kr = b + (16 * j + n) * D;
#pragma unroll
      for (int x = 0; x < NG; ++x) s[j][x] = w_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const w_u4 k = *reinterpret_cast<const w_u4*>(kr + 16 * ((W * g + w) ^ (n % CH)));
        const w_u4 k0 = code_op8<T>(k[0], k[1]), k1 = code_op8<T>(k[2], k[3]);
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          s[j][x] = mfma_op(k0, q[x][2 * w], s[j][x], T{});
          s[j][x] = mfma_op(k1, q[x][2 * w + 1], s[j][x], T{});
        }
      }
      const w_f4 ks = *reinterpret_cast<const w_f4*>(sc + 16 * j + 4 * g);
#pragma unroll
      for (int x = 0; x < NG; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][x][e] *= ks[e] * qscale;
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
    if (scores && live[0] && cols < kScoreCols) {
      // (one group of columns; the positions past the end have their places)
      float* dst = scores + 16 * static_cast<int64_t>(r.wrow) +
                   (static_cast<int64_t>(h) * cols + n) * ((r.len + 15) & ~15) + 4 * g;
      *reinterpret_cast<w_f4*>(dst + p0) = s[0][0];
      if (p1 != 0x7ffffff0) *reinterpret_cast<w_f4*>(dst + p1) = s[1][0];
    }
    const w_f4 vs[2] = {*reinterpret_cast<const w_f4*>(sc + 32 + 4 * g),
                        *reinterpret_cast<const w_f4*>(sc + 48 + 4 * g)};
    w_u4 bh[NG], bl[NG];  // p * value scale, hi and lo parts
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[j][x][e]);
      mx = max_rows4(mx);
      const float m_new = fmaxf(m[x], mx);
      const float base = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = m[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[x] - base);
      m[x] = m_new;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float pv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(s[j][x][e] - base);
          sum += p;
          pv[e] = whole || (seen[x] >> (4 * j + e)) & 1 ? p * vs[j][e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t hi = pack_pair(pv[e], pv[e + 1], bf16{});
          bh[x][2 * j + e / 2] = hi;
          bl[x][2 * j + e / 2] = pack_pair(pv[e] - __uint_as_float(hi << 16),
                                           pv[e + 1] - __uint_as_float(hi & 0xffff0000u), bf16{});
        }
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
        const w_u4 a = code_op8<bf16>(tr[0][k], tr[1][k]);
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          w_f4& acc = o[4 * w + k][x];
          acc = mfma_op(a, bh[x], acc, bf16{});
          acc = mfma_op(a, bl[x], acc, bf16{});
        }
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
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
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
      if (lse && g == 0) lse[at] = sum == 0.0f ? INFINITY : m[x] + __builtin_amdgcn_logf(sum);
      continue;
    }
    const int64_t part = r.part0 + (static_cast<int64_t>(item) * r.n + row[x]) * c.hq + head[x];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float* dst = parts.o + part * D + DB * (4 * g + e);
#pragma unroll
      for (int t = 0; t < DB; t += 4)
        *reinterpret_cast<w_f4*>(dst + t) =
            w_f4{o[t][x][e], o[t + 1][x][e], o[t + 2][x][e], o[t + 3][x][e]};
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
  // items of 4 groups, or of 8 where those of 4 leave 8 MB of partial results (4 requests
  // of up to 16000 positions, 2 kv heads of 128, 16 columns: 20.5 for 23.1 us; 8 of up to
  // 1000, 8 kv heads, 4 columns, which leave less: 17.2 for 13.3)
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

}  // namespace

namespace kvq {

namespace {

bool dec_few(const WinCall& call, int64_t b) {
  return call.lens[b] > 0 && call.qlens[b] > 0 && call.qlens[b] * call.cache.rep.d <= call.few_cols;
}

bool dec_geometry(const WinCall& call) {
  const WinCache& c = call.cache;
  return win_matrix_geometry(call.dtype, c.hq, c.kvh, c.d, static_cast<int>(c.bs.d)) &&
         aligned16(c.kd, c.vd);
}

}  // namespace

bool win_decode_takes(const WinCall& call, int64_t b) {
  return !call.tiles_only && dec_few(call, b) && dec_geometry(call);
}

// Columns up to which a request comes here instead of to the tiles of
// fp8_window_chunk.hip, both sides in us a call.  16: one request of 4000 positions, 8 kv
// heads of 128, 4 and 16 columns, 14 and 17 here, 20 and 20 there; 8 of 1000, 13 and 19,
// 22 and 23.  Past that the partial results cost more than the codes that a tile reads
// again (4 of up to 16000, 2 kv heads, 16, 32 and 64 columns: 21, 30 and 40, 21, 22 and
// 25), but where the requests of 17 - 32 columns have 100 MB of codes to stream (32 of up
// to 2000: 55 and 56; of up to 16384: 171 and 391) and the others, whom the second group
// of columns costs a fifth (122 and 147), are not most of the work.
int win_few_cols(const WinCall& call) {
  const WinCache& c = call.cache;
  int64_t wide = 0, narrow = 0;  // positions seen
  for (int64_t b = 0; b < call.batch; ++b) {
    const int64_t cols = call.qlens[b] * c.rep.d;
    if (call.lens[b] <= 0 || cols <= 0 || cols > 32) continue;
    (cols > 16 ? wide : narrow) +=
        WinSpan::of(static_cast<int>(call.lens[b]), static_cast<int>(call.qlens[b]), c.window,
                    c.sinks, kGroup).groups * int64_t{kGroup};
  }
  return 2 * wide * c.kvh * c.d >= 100 << 20 && wide >= narrow / 8 ? 32 : 16;
}

// In a batch with chunks, requests of few rows ride with their tiles where they see no
// more than the chunks do and all tiles run at once: a launch less (19 requests of up to
// 26 positions with 3 - 11 rows each, head size 256, with weights: 43 and 39 us a call).
bool win_tiles_only(const WinCall& call) {
  if (!dec_geometry(call)) return false;
  const WinCache& c = call.cache;
  int64_t few = 0, many = 0, tiles = 0;  // most positions seen by either kind
  for (int64_t b = 0; b < call.batch; ++b) {
    if (call.lens[b] <= 0 || call.qlens[b] <= 0) continue;
    const int64_t seen = WinSpan::of(static_cast<int>(call.lens[b]), static_cast<int>(call.qlens[b]),
                                     c.window, c.sinks, kGroup).groups;
    int64_t& most = dec_few(call, b) ? few : many;
    most = std::max(most, seen);
    tiles += (call.qlens[b] * c.rep.d + 127) / 128;
  }
  int cus = 0;
  if (device_cu_count(&cus) != KVQ_OK || cus <= 0) cus = 256;
  return few > 0 && few <= many && tiles * c.kvh <= cus;
}

bool win_decode_scores(const WinCall& call, int64_t b) {
  return call.qlens[b] > 0 && call.qlens[b] * call.cache.rep.d < kScoreCols &&
         win_decode_takes(call, b);
}

WinScores win_scores(const WinCall& call) {
  WinScores s{false, 0};
  int64_t keys = 0;  // (position, kv head)s that the scores spare
  bool rest = false;
  for (int64_t b = 0; b < call.batch; ++b) {
    if (win_decode_scores(call, b)) {
      s.units += win_score_units(call, b);
      keys += call.lens[b] * call.cache.kvh;
    } else {
      rest = rest || (call.qlens[b] > 0 && call.lens[b] > 0);
    }
  }
  // beside other requests, whose launch these could share, only where it is worth one
  // (16 requests of 1000 - 2000 positions beside a chunk of 64 rows, 24 MB of keys: 65 us
  // with the scores, 60 without; of 3000 - 6000, 74 MB: 87 and 91)
  s.on = s.units > 0 && 64 * s.units <= kScoreBytes &&
         (!rest || keys * call.cache.d >= (40 << 20));
  if (!s.on) s.units = 0;
  return s;
}

namespace {

int64_t dec_groups(const WinCall& call, int64_t b) {
  if (call.qlens[b] <= 0 || !win_decode_takes(call, b)) return 0;
  return WinSpan::of(static_cast<int>(call.lens[b]), static_cast<int>(call.qlens[b]),
                     call.cache.window, call.cache.sinks, kGroup)
      .groups;
}

template <typename G>
int dec_launches(const WinCall& call, int64_t* split_out, G&& go) {
  int cus = 0;
  const int rc = device_cu_count(&cus);
  if (rc != KVQ_OK) return rc;
  if (cus <= 0) cus = 256;
  const int64_t split = dec_split(call, cus, [&](int64_t b) { return dec_groups(call, b); });
  if (split_out) *split_out = split;
  const int hgs = call.cache.kvh / dec_hpw(call.cache.kvh, call.cache.d);
  return win_launches(
      call,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        const int64_t groups = dec_groups(call, b);
        parts = (groups + split - 1) / split;
        rows = win_part_rows(call, b, parts);
        units = parts * hgs;
        return groups > 0;
      },
      go);
}

}  // namespace

int64_t win_decode_bytes(const WinCall& call, int* rc) {
  int64_t most = 0;
  *rc = dec_launches(call, nullptr,
                     [&](const WinArg&, int, int64_t, int64_t rows) -> int {
                       most = std::max(most, win_parts_bytes(rows, call.cache.d));
                       return KVQ_OK;
                     });
  return most;
}

int win_decode(const WinCall& call, void* workspace) {
  const WinCache& c = call.cache;
  const int hpw = dec_hpw(c.kvh, c.d);
  const int wide = (call.q_wide() ? 1 : 0) | (aligned16(call.out, nullptr) ? 2 : 0);
  int64_t split = 0, scored = 0;
  return dec_launches(call, &split, [&](const WinArg& plan, int count, int64_t units, int64_t rows) -> int {
    WinArg arg = plan;
    if (call.scores)
      for (int i = 0; i < count; ++i)
        if (win_decode_scores(call, arg.r[i].table)) {
          arg.r[i].wrow = static_cast<int32_t>(scored);
          scored += win_score_units(call, arg.r[i].table);
        }
    const WinParts parts{static_cast<float*>(workspace),
                         static_cast<float*>(workspace) + rows * c.d};
#define KVQ_WIN_DECODE(T, D, NG)                                                              \
  hipLaunchKernelGGL((win_decode_kernel<T, D, NG>), dim3(static_cast<unsigned>(units)),       \
                     dim3(64 * hpw), hpw * 2 * dec_tile_bytes<D>(), call.stream, arg, count, c, \
                     static_cast<const T*>(call.query), call.q_stride, wide, call.qscale,     \
                     static_cast<int>(split), hpw, static_cast<T*>(call.out), parts, call.lse, \
                     call.scores)
#define KVQ_WIN_DECODE_N(T, D)  \
  if (call.few_cols > 16)       \
    KVQ_WIN_DECODE(T, D, 2);    \
  else                          \
    KVQ_WIN_DECODE(T, D, 1)
#define KVQ_WIN_DECODE_D(T)     \
  if (c.d == 256) {             \
    KVQ_WIN_DECODE_N(T, 256);   \
  } else if (c.d == 128) {      \
    KVQ_WIN_DECODE_N(T, 128);   \
  } else {                      \
    KVQ_WIN_DECODE_N(T, 64);    \
  }
    if (call.dtype == KVQ_DTYPE_BF16) {
      KVQ_WIN_DECODE_D(bf16)
    } else {
      KVQ_WIN_DECODE_D(f16)
    }
#undef KVQ_WIN_DECODE_D
#undef KVQ_WIN_DECODE_N
#undef KVQ_WIN_DECODE
    KVQ_LAUNCH_CHECK();
    return rows > 0 ? launch_win_join(call, arg, count, parts) : KVQ_OK;
  });
}

}  // namespace kvq
