# SPDX-License-Identifier: Apache-2.0
"""Windowed attention and eviction over the paged E4M3 cache, without a GPU: calls
and arguments at the edges of what is allowed."""

from __future__ import annotations

import pytest
import torch

from tests import _fp8_window as ref
from vllm_ascend_quantized_kv_cache.ops import _native, fp8_window

attend = fp8_window.fp8_per_token_head_window_attention
evict = fp8_window.fp8_per_token_head_evict


@pytest.fixture(scope="module", autouse=True)
def _built():
    if not _native.library_path().exists():
        pytest.skip("libkvq_hip.so not built (run __graft_entry__.build())")


def test_idle_requests_weights_are_work():
    """A call without rows has running weights to move where they go elsewhere."""
    c = ref.Cache([5], 1, 16, 16)
    q = torch.ones(0, 1, 16, dtype=torch.bfloat16)
    w = torch.ones(1, 1, 5)
    assert attend(q, *c.args(), [5], [0], 0.1, weights=w).shape == (0, 1, 16)
    assert attend(q, *c.args(), [0], [0], 0.1, weights=w, out_weights=w.clone()).shape[0] == 0
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attend(q, *c.args(), [5], [0], 0.1, weights=w, out_weights=w.clone())


@pytest.mark.parametrize("past", [2 ** 31, 2 ** 63, 2 ** 64 + 5])
def test_lengths_past_the_library_are_refused(past):
    """Not taken for what is left of them in 64 bits."""
    c = ref.Cache([40, 17], 2, 64, 16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="seq_lens past"):
        attend(q, *c.args(), [past, 17], [1, 1], 0.1)
    with pytest.raises(RuntimeError, match="query_lens past"):
        attend(q, *c.args(), [40, 17], [1, past], 0.1)
    with pytest.raises(RuntimeError, match="seq_lens past"):
        evict(*c.args(), [40, past], torch.zeros(2, 2, 40), 8)
    with pytest.raises(RuntimeError, match="weight_rows past"):
        evict(*c.args(), [40, 17], torch.zeros(2, 2, 40), 8, weight_rows=[0, past])
