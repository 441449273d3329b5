// SPDX-License-Identifier: Apache-2.0
// Shared by the attention over latent rows that all heads share (fp8_latent*.hip).
// Requests, positions and partial results are those of the windowed attention
// (fp8_window.h), with one kv head: column c of a request is row c / H, head c % H.
#pragma once

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

// fp8_latent_mfma.hip: every request with history, where latent_matrix applies.
bool latent_matrix(const LatentCall& call);
int64_t latent_matrix_bytes(const LatentCall& call, int* rc);
int latent_matrix_attend(const LatentCall& call, void* workspace);

}  // namespace kvq
