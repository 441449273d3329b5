// SPDX-License-Identifier: Apache-2.0
// Eviction from the paged E4M3 cache by running attention weight.
//
// A request of L cached rows with a budget of `keep` < L keeps, per kv head, its
// first `sinks` rows, its last `recent` and the keep - sinks - recent heaviest of
// the rest (of equal weights the earliest), in the order of their positions: row
// kept[r] becomes row r, in codes, scales and weights.  The cached row of a
// (token, head) stands by itself (its scale is its own), so heads keep rows of
// their own.  A request within its budget keeps all.
//
// evict_select_kernel: one workgroup per (request, kv head).  The weights' bits
//   become integers in their order (NaN above all, -0 as 0); three rounds of
//   histograms over 11, 11 and 10 bits find the threshold (the top 11 bits of a
//   float, its sign, exponent and two bits of fraction, spread weights of similar
//   size over many more counters than its top byte would), then each wave counts,
//   and after one barrier writes, the survivors of a run of positions of its own.
// Rows past kHeldRow positions are cut into chunks, a workgroup each, and the same
//   rounds run as launches (evict_count_kernel, evict_emit_kernel), the counts passing
//   through the workspace: integers, so their order changes nothing.
// evict_move_kernel: a workgroup copies some ranks of a request, all kv heads: their
//   rows lie side by side in the destination pages.
// evict_compact_kernel: in place.  kept[r] >= r and kept is increasing, so what a
//   chunk of ranks reads is nothing that an earlier chunk has written; one
//   workgroup per (request, kv head, side) walks its chunks in order, and within
//   a chunk every load has returned before the first store.
//
// Bound by HBM where much moves, by the rounds' latencies where little does: 32 requests
// of 4096 - 16384 rows, 8 kv heads of 128, 2048 kept, 83 us a call, of which 19 to select
// and 52 to move (5.3 TB/s); one of 100001, 50000 kept, 80, of which 31 in the selection's
// launches; one of 1100, 2 kv heads, 600 kept, 27, most of it the host's launches.
#include <algorithm>
#include <memory>
#include <new>

#include "fp8_window.h"

namespace {

using namespace kvq;

struct EvictReq {
  int32_t len, keep;
  int32_t table;  // row of both block tables and of kept
  int32_t wrow;   // row of the running weights
  int32_t first;  // units of the requests before it
  int32_t row0;   // rows (kv heads) of the requests before it, in the workspace
  int32_t chunk0; // their chunks
  int32_t unused;
};
constexpr int kEvictReqs = 112;
struct EvictArg {
  EvictReq r[kEvictReqs];
};

__device__ __forceinline__ EvictReq evict_req(int count, int unit) {
  win_cint* a = (win_cint*)__builtin_amdgcn_kernarg_segment_ptr();
  const int lane = threadIdx.x & 63;
  int at = 0;
  for (int c = 0; c < count; c += 64) {
    const bool on = c + lane < count && a[8 * (c + lane) + 4] <= unit;
    at += __builtin_popcountll(__builtin_amdgcn_ballot_w64(on));
  }
  win_cint* r = a + 8 * __builtin_amdgcn_readfirstlane(at - 1);
  return EvictReq{r[0], r[1], r[2], r[3], r[4], r[5], r[6], 0};
}

// ---- selection ------------------------------------------------------------------

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;

// Unsigned integers in the order of the weights: 0 for a place past the row's end, above
// it -inf .. inf, NaN, and on top the rows that stay whatever they weigh.
constexpr uint32_t kStays = 0xffffffffu;
__device__ __forceinline__ uint32_t weight_key(uint32_t bits) {
  if ((bits & 0x7fffffffu) > 0x7f800000u) return kStays - 1;  // NaN
  if (bits == 0x80000000u) bits = 0;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

constexpr uint32_t kZeroKey = 0x80000000u;

// x[0] + .. + x[wave - 1], in every lane.
__device__ __forceinline__ uint32_t sum_before(const uint32_t* x, int wave, int lane) {
  static_assert(kSelWaves == 16, "one row of lanes");
  int v = (lane & 15) < wave ? static_cast<int>(x[lane & 15]) : 0;
  v += __builtin_amdgcn_update_dpp(0, v, kDppQuadXor1, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, kDppQuadXor2, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, kDppHalfMirror, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, kDppRowMirror, 0xf, 0xf, false);
  return static_cast<uint32_t>(v);
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t x, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t y = __shfl_up(x, d, 64);
    x += lane >= d ? y : 0;
  }
  return x;
}

// The weights of a row, or of a chunk of it, in registers: wave w holds a run of
// positions, lane l of it its positions 64 i + l, NK of them; every pass then runs
// without a load.
template <int NK>
struct WeightRow {
  const float* in;
  int begin, stop, lane;  // of this wave (none: begin = stop)
  int len, sinks, end;    // [sinks, end) is up for choice
  uint32_t held[NK], keys[NK];
  __device__ __forceinline__ uint32_t key_at(int k, uint32_t bits) const {
    const uint32_t key = k < sinks || k >= end ? kStays : weight_key(bits);
    return k < stop ? key : 0u;
  }
  // of the row's positions, those from `from` to `to` (the whole row: 0, n)
  __device__ __forceinline__ WeightRow(const float* row, int n, int first, int last, int from, int to,
                                       int wave, int l)
      : in(row), lane(l), len(n), sinks(first), end(n - last) {
    const int per = ((to - from + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
    begin = from + wave * per < to ? from + wave * per : to;
    stop = begin + per < to ? begin + per : to;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int k = begin + 64 * i + lane;
      held[i] = __float_as_uint(in[k < stop ? k : len - 1]);
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) keys[i] = key_at(begin + 64 * i + lane, held[i]);
  }
  // f(position, key, bits) over the wave's run in order, 64 positions at a time
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    constexpr int G = NK < 4 ? NK : 4;  // places past the end come as key 0
#pragma unroll
    for (int i = 0; i < NK; i += G) {
      if (begin + 64 * i >= stop) break;  // uniform
#pragma unroll
      for (int j = i; j < i + G; ++j) f(begin + 64 * j + lane, keys[j], held[j]);
    }
  }
};

// The rounds' fields of a key.
__device__ __forceinline__ int round_shift(int round) { return round == 0 ? 21 : (round == 1 ? 10 : 0); }
__device__ __forceinline__ uint32_t round_field(int round) { return round == 2 ? 0x3ffu : 0x7ffu; }

// Adds this workgroup's keys that agree with prefix on mask to the counters in LDS
// (zeroed here).  Weights of exactly 0, of positions that nothing looked at, are many:
// counted by ballots, where they would queue at one counter.  The rows that stay are
// known: `stay` of them among this workgroup's.
template <int NK>
__device__ __forceinline__ void count_keys(const WeightRow<NK>& row, uint32_t* hist, int round,
                                           uint32_t prefix, uint32_t mask, uint32_t stay) {
  const int tid = threadIdx.x, shift = round_shift(round);
  const uint32_t field = round_field(round);
  for (int k = tid; k < kBins; k += kSelThreads) hist[k] = 0;
  __syncthreads();
  uint32_t zeros = 0;
  row.each([&](int, uint32_t key, uint32_t) {
    const bool match = (key & mask) == prefix;
    zeros += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key == kZeroKey));
    if (match & (key != kZeroKey) & (key - 1 < kStays - 1))
      atomicAdd(&hist[(key >> shift) & field], 1u);
  });
  if ((tid & 63) == 0 && zeros && (kZeroKey & mask) == prefix)
    atomicAdd(&hist[(kZeroKey >> shift) & field], zeros);
  if (tid == 0 && stay && (kStays & mask) == prefix) atomicAdd(&hist[field], stay);
  __syncthreads();
}

// The bin in which the `want`th key from the top lies, and which of the bin's it is;
// c0 and c1: thread t's counts of bins 2 N - 1 - 2 t and 2 N - 2 - 2 t, N threads.
// Returns whether it is the bin's last.
__device__ __forceinline__ bool find_bin(uint32_t c0, uint32_t c1, uint32_t& bin, uint32_t& want,
                                         uint32_t* s_wave, uint32_t* s_found) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t upto = wave_scan(c0 + c1, lane);
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  const uint32_t above = upto - (c0 + c1) + sum_before(s_wave, wave, lane);
  if (above < want && want <= above + c0 + c1) {  // one thread
    const bool upper = want <= above + c0;
    s_found[0] = static_cast<uint32_t>(2 * kSelThreads - 1 - 2 * tid) - (upper ? 0u : 1u);
    const uint32_t nth = want - above - (upper ? 0u : c0);
    s_found[1] = nth;
    s_found[2] = nth == (upper ? c0 : c1);
  }
  __syncthreads();
  bin = s_found[0];
  want = s_found[1];
  const bool last = s_found[2] != 0;
  __syncthreads();  // read before the next call writes them
  return last;
}

// Writes the survivors of this workgroup's run: the keys above `prefix`, and those equal
// to it that are among the first `want` of the row.  more0 / same0: such keys in the
// chunks before this one.
template <int NK>
__device__ __forceinline__ void emit_rows(const WeightRow<NK>& row, uint32_t prefix, uint32_t want,
                                          uint32_t more0, uint32_t same0, uint32_t (*s_wave)[kSelWaves],
                                          int32_t* ids, float* out) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t more = 0, same = 0;  // of this wave's run
  row.each([&](int, uint32_t key, uint32_t) {
    more += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key > prefix));
    same += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key == prefix));
  });
  if (lane == 0) {
    s_wave[0][wave] = more;
    s_wave[1][wave] = same;
  }
  __syncthreads();  // (and every weight held has been read)
  more0 += sum_before(s_wave[0], wave, lane);
  same0 += sum_before(s_wave[1], wave, lane);
  uint32_t at = more0 + (same0 < want ? same0 : want);
  const uint64_t below = (1ull << lane) - 1;
  row.each([&](int k, uint32_t key, uint32_t bits) {
    const uint64_t ties = __builtin_amdgcn_ballot_w64(key == prefix);
    const uint32_t tie_rank = same0 + __builtin_popcountll(ties & below);
    const bool take = (key > prefix) | ((key == prefix) & (tie_rank < want));
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    if (take) {
      const uint32_t rank = at + __builtin_popcountll(taken & below);
      ids[rank] = k;
      out[rank] = __uint_as_float(bits);
    }
    at += __builtin_popcountll(taken);
    same0 += __builtin_popcountll(ties);
  });
}

// A unit is one kv head of a request.  NK: weights a lane holds (16 NK waves cover the
// longest row that is cut).
template <int NK>
__global__ void __launch_bounds__(kSelThreads)
evict_select_kernel(EvictArg, int count, int kvh, int sinks, int recent, const float* w_in,
                    float* w_out, int64_t w_cols, int32_t* __restrict__ kept, int64_t kept_cols) {
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_wave[2][kSelWaves];
  __shared__ uint32_t s_found[3];
  const EvictReq r = evict_req(count, blockIdx.x);
  const int h = static_cast<int>(blockIdx.x) - r.first;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* in = w_in + (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
  float* out = w_out + (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
  int32_t* ids = kept + (static_cast<int64_t>(r.table) * kvh + h) * kept_cols;
  const int stay = r.len < r.keep ? r.len : r.keep;
  for (int64_t k = stay + tid; k < kept_cols; k += kSelThreads) ids[k] = -1;
  if (r.len <= r.keep) {  // uniform
    for (int k = tid; k < r.len; k += kSelThreads) {
      ids[k] = k;
      if (in != out) out[k] = in[k];
    }
    return;
  }
  if (stay == 0) return;
  const WeightRow<NK> row(in, r.len, sinks, recent, 0, r.len, wave, lane);
  uint32_t want = static_cast<uint32_t>(r.keep), prefix = 0, mask = 0;
  // three rounds: `want` survivors among the keys that agree with prefix on mask
#pragma unroll
  for (int round = 0; round < 3; ++round) {
    count_keys(row, s_hist, round, prefix, mask, static_cast<uint32_t>(sinks + recent));
    uint32_t bin;
    const bool all = find_bin(s_hist[kBins - 1 - 2 * tid], s_hist[kBins - 2 - 2 * tid], bin, want,
                              s_wave[0], s_found);
    prefix |= bin << round_shift(round);
    mask |= round_field(round) << round_shift(round);
    if (all && round < 2) {  // uniform: every key of the bin stays, whatever its other bits
      prefix = prefix ? prefix - 1 : 0;  // (0 is no weight's key)
      want = 0;
      break;
    }
  }
  emit_rows(row, prefix, want, 0, 0, s_wave, ids, out);
}

// ---- rows of many chunks ---------------------------------------------------------------

// (4, 8 and 16 a lane: 1 request of 100001 rows, 8 kv heads, 73, 77 and 84 us a call; 4 of
// 60000, 70, 62 and 69; 1 of 10^6, 2 kv heads, 89, 52 and 61.)
constexpr int kChunkNk = 8, kChunk = kSelThreads * kChunkNk;  // positions of a chunk
// The longest row of one workgroup: what its registers hold.  Up to there it is the
// faster way (8 rows of 32000: 35 us a call, 50 in chunks; 256 of 16000: 125, 148).
constexpr int kHeldRow = 32 * kSelThreads;
constexpr int kLowBins = 1024;              // of the last round

// counts: [row][2][kBins] of the first two rounds; low: [chunk of a row][kLowBins] of the
// last; above: per such chunk, its keys past what the first two rounds found; tmp: the
// weights kept, [row][tmp_cols].
struct EvictWs {
  uint32_t *counts, *low, *above;
  float* tmp;
  int64_t tmp_cols;
};

__global__ void __launch_bounds__(256) evict_zero_kernel(uint4* p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = make_uint4(0, 0, 0, 0);
}

// What the first ROUNDS rounds found: the prefix and which of its keys is wanted.
template <int ROUNDS>
__device__ __forceinline__ void found_so_far(const uint32_t* counts, uint32_t& prefix,
                                             uint32_t& mask, uint32_t& want, uint32_t* s_wave,
                                             uint32_t* s_found) {
#pragma unroll
  for (int round = 0; round < ROUNDS; ++round) {
    const uint32_t* c = counts + round * kBins + kBins - 2 - 2 * threadIdx.x;
    uint32_t bin;
    find_bin(c[1], c[0], bin, want, s_wave, s_found);
    prefix |= bin << round_shift(round);
    mask |= round_field(round) << round_shift(round);
  }
}

// Round ROUND over a chunk.  A unit is a chunk of one kv head.
template <int ROUND>
__global__ void __launch_bounds__(kSelThreads)
evict_count_kernel(EvictArg, int count, int kvh, int sinks, int recent, const float* w_in,
                   int64_t w_cols, EvictWs ws) {
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_wave[2][kSelWaves];
  __shared__ uint32_t s_found[3];
  const EvictReq r = evict_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % kvh, chunk = u / kvh, chunks = (r.len + kChunk - 1) / kChunk;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* in = w_in + (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
  const int from = chunk * kChunk, to = r.len - from < kChunk ? r.len : from + kChunk;
  const WeightRow<kChunkNk> row(in, r.len, sinks, recent, from, to, wave, lane);
  uint32_t* counts = ws.counts + static_cast<int64_t>(r.row0 + h) * 2 * kBins;
  uint32_t want = static_cast<uint32_t>(r.keep), prefix = 0, mask = 0;
  found_so_far<ROUND>(counts, prefix, mask, want, s_wave[0], s_found);
  // of the rows that stay, those of this chunk
  const int stay = max(0, min(to, sinks) - from) + max(0, to - max(from, r.len - recent));
  count_keys(row, s_hist, ROUND, prefix, mask, static_cast<uint32_t>(stay));
  if constexpr (ROUND < 2) {
    for (int k = tid; k < kBins; k += kSelThreads)
      if (s_hist[k]) atomicAdd(&counts[ROUND * kBins + k], s_hist[k]);
  } else {
    const int64_t at = r.chunk0 + static_cast<int64_t>(h) * chunks + chunk;
    for (int k = tid; k < kLowBins; k += kSelThreads) ws.low[at * kLowBins + k] = s_hist[k];
    uint32_t more = 0;
    row.each([&](int, uint32_t key, uint32_t) {
      more += __builtin_popcountll(__builtin_amdgcn_ballot_w64((key & mask) > prefix));
    });
    if (lane == 0) s_wave[0][wave] = more;
    __syncthreads();
    if (tid == 0) {
      uint32_t sum = 0;
      for (int w = 0; w < kSelWaves; ++w) sum += s_wave[0][w];
      ws.above[at] = sum;
    }
  }
}

// The survivors of a chunk.  Where the weights move in place they go by ws.tmp.
__global__ void __launch_bounds__(kSelThreads)
evict_emit_kernel(EvictArg, int count, int kvh, int sinks, int recent, const float* w_in,
                  float* w_out, int64_t w_cols, int32_t* __restrict__ kept, int64_t kept_cols,
                  EvictWs ws) {
  __shared__ uint32_t s_wave[2][kSelWaves];
  __shared__ uint32_t s_found[3];
  const EvictReq r = evict_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % kvh, chunk = u / kvh, chunks = (r.len + kChunk - 1) / kChunk;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* in = w_in + (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
  const int from = chunk * kChunk, to = r.len - from < kChunk ? r.len : from + kChunk;
  const WeightRow<kChunkNk> row(in, r.len, sinks, recent, from, to, wave, lane);
  uint32_t want = static_cast<uint32_t>(r.keep), prefix = 0, mask = 0;
  found_so_far<2>(ws.counts + static_cast<int64_t>(r.row0 + h) * 2 * kBins, prefix, mask, want,
                  s_wave[0], s_found);
  // thread t: the last round's bin t, in the whole row and in the chunks before this one
  const int64_t at = r.chunk0 + static_cast<int64_t>(h) * chunks;
  uint32_t all = 0, before = 0, more0 = 0;
#pragma unroll 8
  for (int x = 0; x < chunks; ++x) {
    const uint32_t n = ws.low[(at + x) * kLowBins + tid];
    all += n;
    before += x < chunk ? n : 0;
    more0 += x < chunk ? ws.above[at + x] : 0;
  }
  static_assert(kLowBins == kSelThreads, "a thread a bin");
  // as bins of find_bin: thread t's are 2047 - 2 t and 2046 - 2 t, of which those under
  // 1024 belong to threads 512 .. 1023
  __shared__ uint32_t s_all[kLowBins], s_before[kLowBins];
  s_all[tid] = all;
  s_before[tid] = before;
  __syncthreads();
  const int top = kBins - 1 - 2 * tid;
  uint32_t bin;
  find_bin(top < kLowBins ? s_all[top] : 0, top < kLowBins ? s_all[top - 1] : 0, bin, want,
           s_wave[0], s_found);
  prefix |= bin;
  // keys of the chunks before this one past `bin`, and in it
  uint32_t past = tid > static_cast<int>(bin) ? before : 0;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) past += __shfl_xor(past, d, 64);
  if (lane == 0) s_wave[0][wave] = past;
  __syncthreads();
  more0 += sum_before(s_wave[0], kSelWaves, lane);
  const uint32_t same0 = s_before[bin];
  __syncthreads();  // s_wave is read before emit_rows writes it
  int32_t* ids = kept + (static_cast<int64_t>(r.table) * kvh + h) * kept_cols;
  if (chunk == 0)
    for (int64_t k = r.keep + tid; k < kept_cols; k += kSelThreads) ids[k] = -1;
  float* out = w_in == w_out ? ws.tmp + (static_cast<int64_t>(r.row0) + h) * ws.tmp_cols
                             : w_out + (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
  emit_rows(row, prefix, want, more0, same0, s_wave, ids, out);
}

// ws.tmp into the weights.  A unit is a chunk of one kv head.
__global__ void __launch_bounds__(kSelThreads)
evict_weights_kernel(EvictArg, int count, int kvh, float* w_out, int64_t w_cols, EvictWs ws) {
  const EvictReq r = evict_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int h = u % kvh, from = u / kvh * kChunk;
  const float* src = ws.tmp + (static_cast<int64_t>(r.row0) + h) * ws.tmp_cols;
  float* dst = w_out + (static_cast<int64_t>(r.wrow) * kvh + h) * w_cols;
  for (int k = from + threadIdx.x; k < from + kChunk && k < r.keep; k += kSelThreads) dst[k] = src[k];
}

// ---- moving the rows ----------------------------------------------------------------

struct EvictCache {
  uint8_t *kd, *vd;
  float *ks, *vs;
  const void *src, *dst;  // block tables
  int64_t src_cols, dst_cols, nb;
  FastDiv bs, kvh;
  int bt64, d;
  __device__ __forceinline__ int64_t slot(const void* table, int64_t cols, int row, int p) const {
    const uint32_t i = bs.div(static_cast<uint32_t>(p));
    const int64_t at = static_cast<int64_t>(row) * cols + i;
    const int64_t b = bt64 ? static_cast<const int64_t*>(table)[at]
                           : static_cast<int64_t>(static_cast<const int32_t*>(table)[at]);
    const int64_t page = b < 0 ? 0 : (b >= nb ? nb - 1 : b);  // live ids are checked on the host
    return page * bs.d + (static_cast<uint32_t>(p) - i * bs.d);
  }
};

constexpr int kMoveThreads = 256;

// Ranks of a workgroup: a thread finds one row's places, then all copy.
__host__ __device__ __forceinline__ int move_ranks(int kvh) {
  return kvh < kMoveThreads ? kMoveThreads / kvh : 1;
}

// W: the words a row moves in.  A unit is move_ranks ranks.
template <typename W>
__global__ void __launch_bounds__(kMoveThreads)
evict_move_kernel(EvictArg, int count, EvictCache c, const int32_t* __restrict__ kept,
                  int64_t kept_cols, FastDiv pieces) {
  constexpr int DEPTH = 4;  // words of each side in flight per thread
  __shared__ int64_t s_from[kMoveThreads], s_to[kMoveThreads];
  const EvictReq r = evict_req(count, blockIdx.x);
  const int kvh = static_cast<int>(c.kvh.d), most = move_ranks(kvh), tid = threadIdx.x;
  const int rank0 = (static_cast<int>(blockIdx.x) - r.first) * most;
  const int stay = r.len < r.keep ? r.len : r.keep;
  const int rows = (stay - rank0 < most ? stay - rank0 : most) * kvh;
  for (int x0 = 0; x0 < rows; x0 += kMoveThreads) {  // once, up to kMoveThreads kv heads
    const int n = rows - x0 < kMoveThreads ? rows - x0 : kMoveThreads;
    __syncthreads();  // the last round's places are read
    if (tid < n) {
      // row x: rank rank0 + x / kvh, head x % kvh (rows side by side in the new pages)
      const int x = x0 + tid, k = static_cast<int>(c.kvh.div(static_cast<uint32_t>(x)));
      const int h = x - k * kvh, rank = rank0 + k;
      const int p = kept[(static_cast<int64_t>(r.table) * kvh + h) * kept_cols + rank];
      const int64_t from = c.slot(c.src, c.src_cols, r.table, p) * kvh + h;
      const int64_t to = c.slot(c.dst, c.dst_cols, r.table, rank) * kvh + h;
      s_from[tid] = from * c.d;
      s_to[tid] = to * c.d;
      const float s = c.ks[from], t = c.vs[from];
      c.ks[to] = s;
      c.vs[to] = t;
    }
    __syncthreads();
    const int total = n * static_cast<int>(pieces.d);
    for (int e0 = tid; e0 < total; e0 += DEPTH * kMoveThreads) {
      W a[DEPTH], b[DEPTH];
      int64_t to[DEPTH];
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        const int e = e0 + i * kMoveThreads < total ? e0 + i * kMoveThreads : total - 1;
        const int x = static_cast<int>(pieces.div(static_cast<uint32_t>(e)));
        const int64_t off = static_cast<int64_t>(e - x * static_cast<int>(pieces.d)) * sizeof(W);
        a[i] = *reinterpret_cast<const W*>(c.kd + s_from[x] + off);
        b[i] = *reinterpret_cast<const W*>(c.vd + s_from[x] + off);
        to[i] = s_to[x] + off;
      }
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        if (e0 + i * kMoveThreads < total) {
          *reinterpret_cast<W*>(c.kd + to[i]) = a[i];
          *reinterpret_cast<W*>(c.vd + to[i]) = b[i];
        }
      }
    }
  }
}

constexpr int kCompactThreads = 1024;
constexpr int kCompactDepth = 4;  // words in flight per thread

// In place.  A unit is one side of one kv head, and a slice of its rows' bytes: slices
// move by themselves.
template <typename W>
__global__ void __launch_bounds__(kCompactThreads)
evict_compact_kernel(EvictArg, int count, EvictCache c, const int32_t* __restrict__ kept,
                     int64_t kept_cols, FastDiv pieces, int sinks) {
  const EvictReq r = evict_req(count, blockIdx.x);
  const int u = static_cast<int>(blockIdx.x) - r.first;
  const int kvh = static_cast<int>(c.kvh.d);
  const int slice = u / (2 * kvh), h = (u - slice * 2 * kvh) >> 1;
  const bool scales = slice == 0;
  uint8_t* data = (u & 1 ? c.vd : c.kd) + static_cast<int64_t>(slice) * pieces.d * sizeof(W);
  float* scale = u & 1 ? c.vs : c.ks;
  const int32_t* ids = kept + (static_cast<int64_t>(r.table) * kvh + h) * kept_cols;
  const int64_t total = static_cast<int64_t>(r.keep) * pieces.d;  // words, < 2^31 (host)
  for (int64_t e0 = static_cast<int64_t>(sinks) * pieces.d; e0 < total;
       e0 += kCompactThreads * kCompactDepth) {
    W word[kCompactDepth];
    float s[kCompactDepth];
    int64_t to[kCompactDepth];
    int part[kCompactDepth];
#pragma unroll
    for (int k = 0; k < kCompactDepth; ++k) {
      const int64_t e = e0 + k * kCompactThreads + threadIdx.x;
      to[k] = -1;
      if (e < total) {
        const int rank = static_cast<int>(pieces.div(static_cast<uint32_t>(e)));
        part[k] = static_cast<int>(e) - rank * static_cast<int>(pieces.d);
        const int p = ids[rank];
        if (p != rank) {
          const int64_t from = c.slot(c.src, c.src_cols, r.table, p) * kvh + h;
          to[k] = c.slot(c.src, c.src_cols, r.table, rank) * kvh + h;
          word[k] = reinterpret_cast<const W*>(data + from * c.d)[part[k]];
          if (scales && part[k] == 0) s[k] = scale[from];
        }
      }
    }
    // every load of the chunk has returned before any of its rows is overwritten
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCompactDepth; ++k) {
      if (to[k] >= 0) {
        reinterpret_cast<W*>(data + to[k] * c.d)[part[k]] = word[k];
        if (scales && part[k] == 0) scale[to[k]] = s[k];
      }
    }
  }
}

// ---- host -----------------------------------------------------------------------

template <typename U, typename G>
int for_requests(const int64_t* lens, const int64_t* keeps, const int64_t* rows, int64_t batch,
                 int kvh, U&& units, G&& go) {
  EvictArg arg;
  int count = 0;
  int64_t total = 0, longest = 0, row0 = 0, chunk0 = 0;
  for (int64_t b = 0; b <= batch; ++b) {
    if (count == kEvictReqs || (b == batch && count)) {
      const int rc = go(arg, count, static_cast<unsigned>(total), longest, row0, chunk0);
      if (rc != KVQ_OK) return rc;
      count = 0;
      total = longest = row0 = chunk0 = 0;
    }
    if (b == batch) break;
    const int64_t u = units(b);
    if (u <= 0) continue;
    if (total + u > 0x7fffffff) return KVQ_ERR_INVALID;
    arg.r[count++] = EvictReq{static_cast<int32_t>(lens[b]), static_cast<int32_t>(keeps[b]),
                              static_cast<int32_t>(b), static_cast<int32_t>(rows ? rows[b] : 0),
                              static_cast<int32_t>(total), static_cast<int32_t>(row0),
                              static_cast<int32_t>(chunk0), 0};
    total += u;
    row0 += kvh;
    chunk0 += (lens[b] + kChunk - 1) / kChunk * kvh;
    if (chunk0 > 0x7fffffff) return KVQ_ERR_INVALID;
    longest = lens[b] > keeps[b] && lens[b] > longest ? lens[b] : longest;
  }
  return KVQ_OK;
}

// Rows cut into chunks, and their workgroups.
int64_t chunk_units(const int64_t* lens, const int64_t* keeps, int64_t b, int kvh) {
  return keeps[b] > 0 && lens[b] > keeps[b] && lens[b] > kHeldRow
             ? (lens[b] + kChunk - 1) / kChunk * kvh
             : 0;
}

// Bytes of a launch's EvictWs, whose arrays lie one behind the other.
int64_t evict_ws_bytes(int64_t rows, int64_t chunks, int64_t tmp_cols) {
  return 4 * (rows * 2 * kBins + chunks * kLowBins + (chunks + 3) / 4 * 4 + rows * tmp_cols);
}

// The most rows that a request cut into chunks keeps.
int64_t evict_tmp_cols(const int64_t* lens, const int64_t* keeps, int64_t batch) {
  int64_t cols = 0;
  for (int64_t b = 0; b < batch; ++b)
    if (chunk_units(lens, keeps, b, 1) > 0) cols = std::max(cols, keeps[b]);
  return (cols + 3) / 4 * 4;
}

int64_t evict_bytes(const int64_t* lens, const int64_t* keeps, int64_t batch, int kvh, int* rc) {
  const int64_t cols = evict_tmp_cols(lens, keeps, batch);
  int64_t most = 0;
  *rc = cols == 0 ? KVQ_OK
                  : for_requests(
                        lens, keeps, nullptr, batch, kvh,
                        [&](int64_t b) { return chunk_units(lens, keeps, b, kvh); },
                        [&](const EvictArg&, int, unsigned, int64_t, int64_t rows, int64_t chunks) -> int {
                          most = std::max(most, evict_ws_bytes(rows, chunks, cols));
                          return KVQ_OK;
                        });
  return most;
}

int64_t table_id(const void* table, int type, int64_t at) {
  return type == KVQ_INDEX_I64 ? static_cast<const int64_t*>(table)[at]
                               : static_cast<const int32_t*>(table)[at];
}

}  // namespace

extern "C" int64_t kvq_fp8_pth_evict_check(const void* block_table, const void* out_block_table,
                                           int block_index_type, int64_t max_blocks,
                                           int64_t out_max_blocks, const int64_t* seq_lens,
                                           const int64_t* keep, int64_t batch, int64_t num_blocks,
                                           int block_size) {
  if (batch < 0 || block_size <= 0 || num_blocks <= 0 || max_blocks < 0 || out_max_blocks < 0 ||
      (batch > 0 && (!block_table || !seq_lens || !keep)) ||
      (block_index_type != KVQ_INDEX_I32 && block_index_type != KVQ_INDEX_I64))
    return KVQ_ERR_INVALID;
  // 1: a page of some request's rows, 2: of one whose rows move within it (or a
  // page that rows move to)
  const std::unique_ptr<uint8_t[]> seen(new (std::nothrow) uint8_t[num_blocks]());
  if (!seen) return KVQ_ERR_INVALID;
  for (int64_t b = 0; b < batch; ++b) {
    if (seq_lens[b] < 0 || keep[b] < 0) return KVQ_ERR_INVALID;
    if (seq_lens[b] > max_blocks * block_size) return KVQ_ERR_CAPACITY;
    const bool moves = !out_block_table && seq_lens[b] > keep[b];
    for (int64_t i = 0; i < (seq_lens[b] + block_size - 1) / block_size; ++i) {
      const int64_t id = table_id(block_table, block_index_type, b * max_blocks + i);
      if (id < 0 || id >= num_blocks) return 2 * b + 1;
      if (seen[id] == 2 || (moves && seen[id])) return 2 * b + 2;
      seen[id] = moves ? 2 : 1;
    }
  }
  if (!out_block_table) return KVQ_OK;
  for (int64_t b = 0; b < batch; ++b) {
    const int64_t stay = seq_lens[b] < keep[b] ? seq_lens[b] : keep[b];
    if (stay > out_max_blocks * block_size) return KVQ_ERR_CAPACITY;
    for (int64_t i = 0; i < (stay + block_size - 1) / block_size; ++i) {
      const int64_t id = table_id(out_block_table, block_index_type, b * out_max_blocks + i);
      if (id < 0 || id >= num_blocks) return 2 * b + 1;
      if (seen[id]) return 2 * b + 2;
      seen[id] = 2;
    }
  }
  return KVQ_OK;
}

extern "C" int64_t kvq_fp8_pth_evict_workspace_bytes(const int64_t* seq_lens, const int64_t* keep,
                                                     int64_t batch, int num_kv_heads) {
  if (batch < 0 || (batch > 0 && (!seq_lens || !keep)) || num_kv_heads <= 0)
    return KVQ_ERR_INVALID;
  for (int64_t b = 0; b < batch; ++b)
    if (seq_lens[b] < 0 || seq_lens[b] > kMaxPositions || keep[b] < 0 || keep[b] > kMaxPositions)
      return KVQ_ERR_INVALID;
  int rc = KVQ_OK;
  const int64_t bytes = evict_bytes(seq_lens, keep, batch, num_kv_heads, &rc);
  return rc != KVQ_OK ? KVQ_ERR_INVALID : bytes;
}

extern "C" int kvq_fp8_pth_evict(uint8_t* k_data, float* k_scale, uint8_t* v_data, float* v_scale,
                                 int64_t num_blocks, int block_size, int num_kv_heads,
                                 int head_size, const void* block_table,
                                 const void* out_block_table, int block_index_type,
                                 int64_t max_blocks, int64_t out_max_blocks,
                                 const int64_t* seq_lens, const int64_t* keep, int64_t batch,
                                 int64_t sinks, int64_t recent, const float* weights_in,
                                 float* weights_out, const int64_t* weight_rows,
                                 int64_t weight_cols, int32_t* kept, int64_t kept_cols,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  if (batch == 0) return KVQ_OK;
  if (!k_data || !k_scale || !v_data || !v_scale || !block_table || !seq_lens || !keep ||
      !weights_in || !weights_out || !weight_rows || !kept || batch < 0 || num_blocks <= 0 ||
      block_size <= 0 || sinks < 0 || recent < 0 || max_blocks < 0 || out_max_blocks < 0 ||
      (block_index_type != KVQ_INDEX_I32 && block_index_type != KVQ_INDEX_I64))
    return KVQ_ERR_INVALID;
  if (num_kv_heads <= 0 || head_size <= 0 || head_size % 4 || head_size > 512)
    return KVQ_ERR_GEOMETRY;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k_data) | reinterpret_cast<uintptr_t>(v_data);
  if (bits & 3) return KVQ_ERR_GEOMETRY;
  const bool wide = head_size % 16 == 0 && (bits & 15) == 0;
  const int pieces = head_size / (wide ? 16 : 4);
  for (int64_t b = 0; b < batch; ++b) {
    const int64_t len = seq_lens[b], stay = len < keep[b] ? len : keep[b];
    if (len < 0 || len > kMaxPositions || keep[b] < 0 || keep[b] > kMaxPositions ||
        len > max_blocks * block_size || len > weight_cols || stay > kept_cols ||
        weight_rows[b] < 0 || weight_rows[b] > kMaxPositions ||
        (out_block_table && stay > out_max_blocks * block_size))
      return KVQ_ERR_INVALID;
    if (len > keep[b] && (sinks + recent > keep[b] || keep[b] * pieces > 0x7fffffff))
      return KVQ_ERR_INVALID;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const EvictCache c{k_data, v_data, k_scale, v_scale, block_table,
                     out_block_table ? out_block_table : block_table, max_blocks,
                     out_block_table ? out_max_blocks : max_blocks, num_blocks,
                     FastDiv::make(static_cast<uint32_t>(block_size)),
                     FastDiv::make(static_cast<uint32_t>(num_kv_heads)),
                     block_index_type == KVQ_INDEX_I64, head_size};
  const FastDiv piece_div = FastDiv::make(static_cast<uint32_t>(pieces));
  const int kvh = num_kv_heads, snk = static_cast<int>(sinks), rec = static_cast<int>(recent);
  int rc = KVQ_OK;
  const int64_t need = evict_bytes(seq_lens, keep, batch, kvh, &rc);
  if (rc != KVQ_OK) return rc;
  if (need > 0 && (!workspace || !aligned16(workspace, nullptr) || workspace_bytes < need))
    return KVQ_ERR_INVALID;
  rc = for_requests(
      seq_lens, keep, weight_rows, batch, kvh,
      [&](int64_t b) { return chunk_units(seq_lens, keep, b, kvh) > 0 ? 0 : kvh; },
      [&](const EvictArg& arg, int count, unsigned blocks, int64_t longest, int64_t, int64_t) -> int {
#define KVQ_EVICT_SELECT(NK)                                                                  \
  hipLaunchKernelGGL((evict_select_kernel<NK>), dim3(blocks), dim3(kSelThreads), 0, s, arg,   \
                     count, kvh, snk, rec, weights_in, weights_out, weight_cols, kept, kept_cols)
        // what a lane has to hold of the longest row that is cut
        const int64_t held = ((longest + kSelWaves - 1) / kSelWaves + 63) / 64;
        if (held <= 2)
          KVQ_EVICT_SELECT(2);
        else if (held <= 8)
          KVQ_EVICT_SELECT(8);
        else
          KVQ_EVICT_SELECT(32);
#undef KVQ_EVICT_SELECT
        KVQ_LAUNCH_CHECK();
        return KVQ_OK;
      });
  if (rc != KVQ_OK) return rc;
  const int64_t tmp_cols = need > 0 ? evict_tmp_cols(seq_lens, keep, batch) : 0;
  if (need > 0)
    rc = for_requests(
        seq_lens, keep, weight_rows, batch, kvh,
        [&](int64_t b) { return chunk_units(seq_lens, keep, b, kvh); },
        [&](const EvictArg& arg, int count, unsigned blocks, int64_t, int64_t rows,
            int64_t chunks) -> int {
          EvictWs ws;
          ws.counts = static_cast<uint32_t*>(workspace);
          ws.low = ws.counts + rows * 2 * kBins;
          ws.above = ws.low + chunks * kLowBins;
          ws.tmp = reinterpret_cast<float*>(ws.above + (chunks + 3) / 4 * 4);
          ws.tmp_cols = tmp_cols;
          const int64_t words = rows * 2 * kBins / 4;
          hipLaunchKernelGGL(evict_zero_kernel, dim3(static_cast<unsigned>((words + 255) / 256)),
                             dim3(256), 0, s, reinterpret_cast<uint4*>(ws.counts), words);
          KVQ_LAUNCH_CHECK();
          const dim3 grid(blocks), block(kSelThreads);
          hipLaunchKernelGGL((evict_count_kernel<0>), grid, block, 0, s, arg, count, kvh, snk, rec,
                             weights_in, weight_cols, ws);
          hipLaunchKernelGGL((evict_count_kernel<1>), grid, block, 0, s, arg, count, kvh, snk, rec,
                             weights_in, weight_cols, ws);
          hipLaunchKernelGGL((evict_count_kernel<2>), grid, block, 0, s, arg, count, kvh, snk, rec,
                             weights_in, weight_cols, ws);
          KVQ_LAUNCH_CHECK();
          hipLaunchKernelGGL(evict_emit_kernel, grid, block, 0, s, arg, count, kvh, snk, rec,
                             weights_in, weights_out, weight_cols, kept, kept_cols, ws);
          KVQ_LAUNCH_CHECK();
          if (weights_in == weights_out) {
            hipLaunchKernelGGL(evict_weights_kernel, grid, block, 0, s, arg, count, kvh,
                               weights_out, weight_cols, ws);
            KVQ_LAUNCH_CHECK();
          }
          return KVQ_OK;
        });
  if (rc != KVQ_OK) return rc;
  if (out_block_table) {
    const int ranks = move_ranks(kvh);
    return for_requests(
        seq_lens, keep, weight_rows, batch, kvh,
        [&](int64_t b) {
          return ((seq_lens[b] < keep[b] ? seq_lens[b] : keep[b]) + ranks - 1) / ranks;
        },
        [&](const EvictArg& arg, int count, unsigned blocks, int64_t, int64_t, int64_t) -> int {
          if (wide)
            hipLaunchKernelGGL((evict_move_kernel<w_u4>), dim3(blocks), dim3(kMoveThreads), 0, s, arg,
                               count, c, kept, kept_cols, piece_div);
          else
            hipLaunchKernelGGL((evict_move_kernel<uint32_t>), dim3(blocks), dim3(kMoveThreads), 0, s, arg,
                               count, c, kept, kept_cols, piece_div);
          KVQ_LAUNCH_CHECK();
          return KVQ_OK;
        });
  }
  // slices of the rows while CUs are free (1 request, 8 kv heads of 128, 32768 of 100001
  // rows kept: 406, 222, 166 and 144 us in 1, 2, 4 and 8; 1000 of 1100: 26 - 28)
  int cus = 0;
  if (device_cu_count(&cus) != KVQ_OK || cus <= 0) cus = 256;
  int64_t moved = 0, slices = 1;
  for (int64_t b = 0; b < batch; ++b) moved += seq_lens[b] > keep[b];
  while (moved * 2 * num_kv_heads * slices * 2 <= cus && piece_div.d % (2 * slices) == 0) slices *= 2;
  const FastDiv slice_div = FastDiv::make(static_cast<uint32_t>(piece_div.d / slices));
  return for_requests(
      seq_lens, keep, weight_rows, batch, kvh,
      [&](int64_t b) { return seq_lens[b] > keep[b] ? 2 * slices * num_kv_heads : 0; },
      [&](const EvictArg& arg, int count, unsigned blocks, int64_t, int64_t, int64_t) -> int {
        if (wide)
          hipLaunchKernelGGL((evict_compact_kernel<w_u4>), dim3(blocks), dim3(kCompactThreads), 0,
                             s, arg, count, c, kept, kept_cols, slice_div,
                             static_cast<int>(sinks));
        else
          hipLaunchKernelGGL((evict_compact_kernel<uint32_t>), dim3(blocks), dim3(kCompactThreads),
                             0, s, arg, count, c, kept, kept_cols, slice_div,
                             static_cast<int>(sinks));
        KVQ_LAUNCH_CHECK();
        return KVQ_OK;
      });
}
