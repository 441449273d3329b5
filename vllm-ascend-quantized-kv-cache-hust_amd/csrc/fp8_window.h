// SPDX-License-Identifier: Apache-2.0
// Shared by the translation units of the windowed attention over paged E4M3
// rows (fp8_window*.hip): the requests of a launch, which cached positions a
// query row sees, and the layout of partial results.
//
// Request b holds L = len cached rows, the last n of which are its query rows:
// row i sits at position L - n + i and sees position j when
//   0 <= j <= pos_i  and  (no window, or j > pos_i - window, or j < sinks).
// The kernels take the rows of one kv head's group of rep = hq / kvh query heads
// together: column c is row c / rep, head h * rep + c % rep.
#pragma once

#include "kvq_common.h"

namespace kvq {

constexpr int kNoWindow = 0x7fffffff;  // a window that hides nothing (positions stay below)
constexpr int64_t kMaxPositions = 0x7fff0000;

// One request of a launch.  They travel as the kernel's first argument.
struct WinReq {
  int32_t q0;     // its first row in query / out
  int32_t n;      // rows
  int32_t len;    // cached positions
  int32_t table;  // its row of the block table
  int32_t first;  // units (workgroups, items) of the requests before it
  int32_t parts;  // partial results per row
  int32_t part0;  // its first partial row
  int32_t wrow;   // its row of the running weights; where the decode leaves scores, theirs
};
constexpr int kWinReqs = 112;
struct WinArg {
  WinReq r[kWinReqs];
};
static_assert(sizeof(WinArg) <= 3584, "kernel arguments end at 4 KB");

// Request `at` (uniform) of the launch, read in place: the argument is the kernel's
// first (indexed by value it would be copied to scratch).
typedef const __attribute__((address_space(4))) int32_t win_cint;
__device__ __forceinline__ WinReq win_req_at(int at) {
  win_cint* r = (win_cint*)__builtin_amdgcn_kernarg_segment_ptr() + 8 * at;
  return WinReq{r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]};
}

// The request whose units [first, first + its own) hold `unit`.  All lanes of the wave
// ask for the same unit.
__device__ __forceinline__ WinReq win_req(int count, int unit) {
  win_cint* a = (win_cint*)__builtin_amdgcn_kernarg_segment_ptr();
  const int lane = threadIdx.x & 63;
  int at = 0;  // requests that start at or before `unit`
  for (int c = 0; c < count; c += 64) {
    const bool on = c + lane < count && a[8 * (c + lane) + 4] <= unit;
    at += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on));
  }
  // requests without units share their first with the next one that has some
  return win_req_at(__builtin_amdgcn_readfirstlane(at - 1));
}

// Everything else a kernel needs of the cache.
struct WinCache {
  const uint8_t* kd;
  const float* ks;
  const uint8_t* vd;
  const float* vs;
  const void* table;
  int64_t maxb, nb;
  FastDiv bs;
  int bt64;  // table entries are int64
  int kvh, hq, d;
  FastDiv rep;
  int window, sinks;
  // Slot of position p of the request with table row t.  A page id outside the
  // cache (a page nobody sees any more) reads a page inside it: such positions
  // are masked.
  __device__ __forceinline__ int64_t page(int t, int i) const {
    const int64_t at = static_cast<int64_t>(t) * maxb + (i < maxb ? i : maxb - 1);
    const int64_t b = bt64 ? static_cast<const int64_t*>(table)[at]
                           : static_cast<int64_t>(static_cast<const int32_t*>(table)[at]);
    return b < 0 ? 0 : (b >= nb ? nb - 1 : b);
  }
  __device__ __forceinline__ int64_t slot(int t, int p) const {
    const uint32_t i = bs.div(static_cast<uint32_t>(p));
    return page(t, static_cast<int>(i)) * bs.d + (static_cast<uint32_t>(p) - i * bs.d);
  }
  __device__ __forceinline__ bool sees(int pos, int j) const {
    return j <= pos && (j > pos - window || j < sinks);
  }
};

// The positions a request's rows see at all: [0, sink) and [low, len), as one
// list of 16-position groups.  The sinks' groups come first; where they reach
// the window's the two are one range (sink 0, low 0).
struct WinSpan {
  int sink_groups, low, groups;
  __host__ __device__ static WinSpan of(int len, int n, int window, int sinks, int align) {
    int64_t lo = static_cast<int64_t>(len) - n - window + 1;  // of the first row
    lo = lo < 0 ? 0 : lo;
    lo = lo > len ? len : lo;
    int low = static_cast<int>(lo) / align * align;
    int sg = (sinks + align - 1) / align;
    if (sg * static_cast<int64_t>(align) >= low) {
      low = 0;
      sg = 0;
    }
    return WinSpan{sg, low, sg + (len - low + align - 1) / align};
  }
  __host__ __device__ int pos(int g, int align) const {
    return g < sink_groups ? g * align : low + (g - sink_groups) * align;
  }
};

// ---- operands of the matrix kernels ------------------------------------------------
typedef float w_f4 __attribute__((ext_vector_type(4)));
typedef float w_f2 __attribute__((ext_vector_type(2)));
typedef uint32_t w_u4 __attribute__((ext_vector_type(4)));
typedef _Float16 w_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 w_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 w_b8 __attribute__((ext_vector_type(8)));

// Codes (bytes 0, 1 or 2, 3 of x) as a pair of T, exact (NaN codes give NaN).
template <bool HI>
__device__ __forceinline__ uint32_t code_pair(uint32_t x, bf16) {
  return __builtin_bit_cast(
      uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(x), 1.0f, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t code_pair(uint32_t x, f16) {
  return __builtin_bit_cast(
      uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(x), 1.0f, HI));
}
template <typename T>
__device__ __forceinline__ w_u4 code_op8(uint32_t w0, uint32_t w1) {
  return w_u4{code_pair<false>(w0, T{}), code_pair<true>(w0, T{}), code_pair<false>(w1, T{}),
              code_pair<true>(w1, T{})};
}
// 0x80 in every byte of x that is a NaN code.
__device__ __forceinline__ uint32_t nan_codes(uint32_t x) {
  return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// Two fp32 values as a pair of T (round to nearest even).
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, bf16) { return bf16x2_bits(lo, hi); }
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, f16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((w_f2{lo, hi}), w_h2));
}

__device__ __forceinline__ w_f4 mfma_op(w_u4 a, w_u4 b, w_f4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w_b8, a),
                                                 __builtin_bit_cast(w_b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ w_f4 mfma_op(w_u4 a, w_u4 b, w_f4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(w_h8, a),
                                                __builtin_bit_cast(w_h8, b), c, 0, 0, 0);
}

// Eight consecutive 16-bit elements; `wide` (uniform): on a 16-byte bound.
template <typename T>
__device__ __forceinline__ w_u4 load_op8(const T* p, bool wide) {
  if (wide) return *reinterpret_cast<const w_u4*>(p);
  w_u4 r;
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = static_cast<uint32_t>(e[2 * i]) | (static_cast<uint32_t>(e[2 * i + 1]) << 16);
  return r;
}

// LDS DMA of 16 (4) bytes a lane from base + off (base uniform) to LDS bytes m0 + 16
// (4) * lane.  Outside the compiler's wait counting: waits are explicit.
__device__ __forceinline__ void win_dma16(const void* base, uint32_t off, uint32_t m0) {
  m0 = __builtin_amdgcn_readfirstlane(m0);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "{m0}"(m0)
               : "memory");
}
__device__ __forceinline__ void win_dma4(const void* base, uint32_t off, uint32_t m0) {
  m0 = __builtin_amdgcn_readfirstlane(m0);
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1"
               :
               : "v"(off), "s"(base), "{m0}"(m0)
               : "memory");
}
__device__ __forceinline__ uint32_t win_lds(const void* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)(p)));
}

// ---- partial results -----------------------------------------------------------------
// Row (i, head) of part s of a request: partial row part0 + (s * n + i) * hq + head,
// o fp32 [D] and (m, l), m in the log2 domain.  A part that sees nothing of the row
// has m = -inf and its o may be unwritten; m = +inf makes the joined row NaN.
struct WinParts {
  float* o;
  float* ml;
};

// A call's launches share these.
struct WinCall {
  const void* query;
  int dtype;
  int64_t q_stride;
  const int64_t *lens, *qlens;
  int64_t batch;
  WinCache cache;
  float qscale;
  const float* w_in;
  float* w_out;
  const int64_t* w_rows;
  int64_t w_cols;
  void* out;
  float* lse;  // per (row, head), where running weights are kept
  int few_cols;     // columns (row, head) up to which a request is one of few rows (win_few_cols)
  bool tiles_only;  // requests of few rows go with the chunks' tiles (win_tiles_only)
  float* scores;  // of the requests whose weights are summed from them (win_scores_at)
  hipStream_t stream;
  bool q_wide() const {
    return (reinterpret_cast<uintptr_t>(query) & 15) == 0 && q_stride % 8 == 0;
  }
};

// Launches over some requests of a call, kWinReqs at a time.  shape(b, units, parts,
// rows): whether request b takes part, its workgroups, its parts and its partial rows
// (of whatever the kernel leaves in the workspace); go(arg, requests, workgroups,
// partial rows).  Partial rows count from 0 in every launch: launches of one stream
// share the workspace.  Of the requests with rows, or those without (idle).
template <typename U, typename G>
int win_launches(const WinCall& call, U&& shape, G&& go, bool idle = false) {
  WinArg arg;
  int count = 0;
  int64_t total = 0, q0 = 0, part0 = 0;
  for (int64_t b = 0; b <= call.batch; ++b) {
    if (count == kWinReqs || (b == call.batch && count)) {
      const int rc = go(arg, count, total, part0);
      if (rc != KVQ_OK) return rc;
      count = 0;
      total = part0 = 0;
    }
    if (b == call.batch) break;
    int64_t units = 0, parts = 1, rows = 0;
    if ((call.qlens[b] == 0) == idle && shape(b, units, parts, rows) && units > 0) {
      if (total + units > 0x7fffffff) return KVQ_ERR_INVALID;
      arg.r[count++] = WinReq{static_cast<int32_t>(q0), static_cast<int32_t>(call.qlens[b]),
                              static_cast<int32_t>(call.lens[b]), static_cast<int32_t>(b),
                              static_cast<int32_t>(total), static_cast<int32_t>(parts),
                              static_cast<int32_t>(part0),
                              static_cast<int32_t>(call.w_rows ? call.w_rows[b] : 0)};
      total += units;
      part0 += rows;
      if (part0 > 0x7fffffff) return KVQ_ERR_INVALID;
    }
    q0 += call.qlens[b];
  }
  return KVQ_OK;
}

// Partial rows of an attention's request.
inline int64_t win_part_rows(const WinCall& call, int64_t b, int64_t parts) {
  return parts > 1 ? parts * call.qlens[b] * call.cache.hq : 0;
}
// Requests whose decode leaves its scores in the workspace, [kv head][column][positions,
// a multiple of 16] in the log2 domain, for the weights to be summed from: below this
// many columns that takes less than the keys once more and their products, while all of
// them stay a small workspace.  Written and read, a column's 4 bytes a position are less
// than the keys' D + 4 up to 15 columns at D = 128 and up to 8 at 64, where the products
// they spare decide.  32 requests of 2048 - 16384 positions, us a call with the scores
// and without, 9, 12 and 15 columns: 8 kv heads of 64, 124, 134 and 147 to 146, 147 and
// 149; 8 of 128, 196, 210 and 227 to 216, 219 and 222; 2 of 256, 89, 94 and 99 to 101, 102
// and 104.  16 columns, 8 kv heads of 128: 227 to 215.
constexpr int kScoreCols = 16;
constexpr int64_t kScoreBytes = 256ll << 20;
struct WinScores {
  bool on;
  int64_t units;  // of 16 floats
};
inline int64_t win_score_units(const WinCall& call, int64_t b) {
  return call.qlens[b] * call.cache.hq * ((call.lens[b] + 15) / 16);
}

inline int64_t win_parts_bytes(int64_t rows, int d) {
  return rows * (static_cast<int64_t>(d) + 2) * static_cast<int64_t>(sizeof(float));
}

// Joins the parts of the requests of `arg` that have several (fp8_window.hip).
int launch_win_join(const WinCall& call, const WinArg& arg, int count, WinParts parts);

// fp8_window_decode.hip: requests of few rows.  _takes: request b is one of them
// (the geometry is one of the matrix kernels'); _bytes: the partial results.
bool win_decode_takes(const WinCall& call, int64_t b);
int win_few_cols(const WinCall& call);
bool win_tiles_only(const WinCall& call);
bool win_decode_scores(const WinCall& call, int64_t b);
WinScores win_scores(const WinCall& call);
int64_t win_decode_bytes(const WinCall& call, int* rc);
int win_decode(const WinCall& call, void* workspace);

// fp8_window_chunk.hip: the other requests of that geometry, likewise.
bool win_chunk_takes(const WinCall& call, int64_t b);
int64_t win_chunk_bytes(const WinCall& call, int* rc);
int win_chunk(const WinCall& call, void* workspace);

// fp8_window_weights.hip: the running weights of the requests of that geometry; `scores`:
// those of win_decode_scores from their scores.
bool win_weights_takes(const WinCall& call, int64_t b);
int64_t win_weights_bytes(const WinCall& call, const WinScores& scores, int* rc);
int win_weights(const WinCall& call, const WinScores& scores, void* workspace);

// 16-bit queries, head sizes 64, 128 and 256, whole groups of 16 positions a page, at
// most 16 query heads per kv head, codes on 16-byte bounds.
inline bool win_matrix_geometry(int dtype, int hq, int kvh, int d, int bs) {
  return (dtype == KVQ_DTYPE_BF16 || dtype == KVQ_DTYPE_F16) && (d == 64 || d == 128 || d == 256) &&
         bs % 16 == 0 && hq / kvh <= 16;
}

}  // namespace kvq
