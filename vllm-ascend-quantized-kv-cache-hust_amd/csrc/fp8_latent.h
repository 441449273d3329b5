// SPDX-License-Identifier: Apache-2.0
// Shared by the attention over latent rows that all heads share (fp8_latent*.hip).
// Requests, positions and partial results are those of the windowed attention
// (fp8_window.h), with one kv head: column c of a request is row c / H, head c % H.
#pragma once

#include <algorithm>

#include "fp8_window.h"

namespace kvq {

// kd: codes [pages, positions, d], ks: a scale a position, rope: the position parts
// [pages, positions, part] of the queries' type.
struct LatentCache : WinCache {
  const void* rope;
  int part;
};

// A call: `win.cache` is `cache`'s part of it.
struct LatentCall {
  WinCall win;
  LatentCache cache;
};

// fp8_latent_mfma.hip: requests of at most kLatentFew columns; fp8_latent_tile.hip: the
// others; both where latent_matrix applies.  _bytes: their partial results.
//
// A decode of 32 requests of 2048 - 16384 positions, R = 512, us a call by the first and by
// the second: 16 columns 47 and 57, 32 columns 57 and 60, 48 columns 83 and 66, 64 columns 87
// and 68; R = 256: 41 and 45, 41 and 45, 64 columns 58 and 46.
constexpr int kLatentFew = 32;
bool latent_matrix(const LatentCall& call);
int64_t latent_few_bytes(const LatentCall& call, int* rc);
int latent_few_attend(const LatentCall& call, void* workspace);
int64_t latent_tile_bytes(const LatentCall& call, int* rc);
int latent_tile_attend(const LatentCall& call, void* workspace);

// ---- their launches --------------------------------------------------------------

inline bool latent_few(const LatentCall& call, int64_t b) {
  return call.win.qlens[b] * call.cache.hq <= kLatentFew;
}

// How a kernel cuts its requests: columns of a tile, positions of a stage; in stages of one
// workgroup, a workgroup's own work (queries in, results out) and the joining launch; bytes
// of partial results that go through memory and back within a stage.
struct LatentShape {
  bool few;
  int cols, stage, own, join, bytes;
};

inline int64_t latent_tiles(const LatentCall& call, const LatentShape& s, int64_t b) {
  return (call.win.qlens[b] * call.cache.hq + s.cols - 1) / s.cols;
}
inline int64_t latent_stages(const LatentCall& call, const LatentShape& s, int64_t b) {
  return std::max<int64_t>(1, (call.win.lens[b] + s.stage - 1) / s.stage);
}

// Stages of a part: what ends soonest when the CUs take one workgroup each at a time.  Host
// work, some dozens of cuts times every request: 1 us for one request, 6 for 32, 12 for 64, 24
// for 128, 48 for 256; a call does it three times (its sizing, the check of that, the launch).
inline int64_t latent_split(const LatentCall& call, const LatentShape& s, int cus) {
  int64_t longest = 1;
  for (int64_t b = 0; b < call.win.batch; ++b)
    if (call.win.qlens[b] > 0 && latent_few(call, b) == s.few)
      longest = std::max(longest, latent_stages(call, s, b));
  int64_t best = longest, cost = INT64_MAX;
  for (int64_t split = longest; split >= 1;
       split = split > 64 ? split - split / 8 : (split > 16 ? split - 4 : split - 1)) {
    int64_t work = 0, groups = 0, rows = 0;
    for (int64_t b = 0; b < call.win.batch; ++b) {
      if (call.win.qlens[b] <= 0 || latent_few(call, b) != s.few) continue;
      const int64_t tiles = latent_tiles(call, s, b), n = latent_stages(call, s, b);
      const int64_t parts = (n + split - 1) / split;
      work += tiles * (n + s.own * parts);
      groups += tiles * parts;
      rows += win_part_rows(call.win, b, parts);
    }
    // (what is left over when the CUs come out unevenly: half of a workgroup's time)
    const int64_t each = split + s.own;
    int64_t time = groups <= cus ? each : std::max(each, work / cus + each / 2);
    if (rows > 0) time += s.join + rows * call.cache.d * 4 / s.bytes;
    if (time < cost) {
      best = split;
      cost = time;
    }
  }
  return best;
}

// go(arg, count, units, partial rows) for each launch, whose requests of the longest parts
// come first: what the CUs come to last is short.  64 requests of 1000 - 8192 positions and
// 256 columns: 220 us, in the batch's order 242.
template <typename G>
int latent_launches(const LatentCall& call, const LatentShape& s, G&& go) {
  int cus = 0;
  const int rc = device_cu_count(&cus);
  if (rc != KVQ_OK) return rc;
  if (cus <= 0) cus = 256;
  const int64_t split = latent_split(call, s, cus);
  return win_launches(
      call.win,
      [&](int64_t b, int64_t& units, int64_t& parts, int64_t& rows) {
        if (latent_few(call, b) != s.few) return false;
        parts = (latent_stages(call, s, b) + split - 1) / split;
        rows = win_part_rows(call.win, b, parts);
        units = latent_tiles(call, s, b) * parts;
        return true;
      },
      [&](const WinArg& in, int count, int64_t total, int64_t rows) -> int {
        WinArg arg = in;
        int32_t units[kWinReqs];
        for (int i = 0; i < count; ++i)
          units[i] = (i + 1 < count ? in.r[i + 1].first : static_cast<int32_t>(total)) - in.r[i].first;
        auto each = [](const WinReq& r) { return r.len / r.parts; };
        for (int i = 1; i < count; ++i) {
          const WinReq r = arg.r[i];
          const int32_t u = units[i];
          int j = i;
          for (; j > 0 && each(arg.r[j - 1]) < each(r); --j) {
            arg.r[j] = arg.r[j - 1];
            units[j] = units[j - 1];
          }
          arg.r[j] = r;
          units[j] = u;
        }
        int32_t first = 0;
        for (int i = 0; i < count; ++i) {
          arg.r[i].first = first;
          first += units[i];
        }
        return go(arg, count, total, rows);
      });
}

}  // namespace kvq
