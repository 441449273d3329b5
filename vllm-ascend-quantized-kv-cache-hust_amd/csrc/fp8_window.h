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
  int32_t wrow;   // its row of the running weights
};
constexpr int kWinReqs = 112;
struct WinArg {
  WinReq r[kWinReqs];
};
static_assert(sizeof(WinArg) <= 3584, "kernel arguments end at 4 KB");

// The request whose units [first, first + its own) hold `unit`, read in place:
// the argument is the kernel's first (indexed by value it would be copied to
// scratch).  All lanes of the wave ask for the same unit.
typedef const __attribute__((address_space(4))) int32_t win_cint;
__device__ __forceinline__ WinReq win_req(int count, int unit) {
  win_cint* a = (win_cint*)__builtin_amdgcn_kernarg_segment_ptr();
  const int lane = threadIdx.x & 63;
  int at = 0;  // requests that start at or before `unit`
  for (int c = 0; c < count; c += 64) {
    const bool on = c + lane < count && a[8 * (c + lane) + 4] <= unit;
    at += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on));
  }
  // requests without units share their first with the next one that has some
  win_cint* r = a + 8 * __builtin_amdgcn_readfirstlane(at - 1);
  return WinReq{r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]};
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

}  // namespace kvq
