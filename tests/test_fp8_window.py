# SPDX-License-Identifier: Apache-2.0
"""Windowed attention and eviction over the paged E4M3 cache, without a GPU: what is
refused, and the host's page checks."""

from __future__ import annotations

import numpy as np
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


def _attend(lens=(40, 17), news=(1, 3), hq=4, kvh=2, d=64, edit=None, **kw):
    c = ref.Cache(lens, kvh, d, 16)
    a = dict(query=torch.zeros(sum(news), hq, d, dtype=torch.bfloat16), k_data=c.k, k_scale=c.ks,
             v_data=c.v, v_scale=c.vs, block_table=c.table, seq_lens=list(lens),
             query_lens=list(news), scale=0.1)
    a.update(kw)
    if edit:
        edit(a)
    return attend(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(query=torch.zeros(4, 4, 32, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(4, 64, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(4, 3, 64, dtype=torch.bfloat16)), "3 query heads over 2"),
    (dict(query=torch.zeros(4, 4, 64, dtype=torch.float64)), "unsupported floating dtype"),
    (dict(query=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "sum to 4"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(scale=float("inf")), "scale must be positive"),
    (dict(window=0), "window must be at least 1"),
    (dict(sinks=-1), "sinks must not be negative"),
    (dict(seq_lens=[40, -1]), "negative seq_lens"),
    (dict(query_lens=[5, -1]), "negative query_lens"),
    (dict(query_lens=[4]), "1 query_lens for 2"),
    (dict(seq_lens=[40, 49]), "does not cover the longest"),
    (dict(out=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), "does not match query"),
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int32)), "2D with a row per request"),
    (dict(block_table=torch.zeros(2, 3)), "int32/int64"),
    (dict(block_table_host=np.zeros((1, 3))), "the host's copy is \\(1, 3\\)"),
    (dict(weight_rows=[0, 1]), "need weights"),
    (dict(out_weights=torch.zeros(2, 2, 40)), "need weights"),
    (dict(weights=torch.zeros(2, 3, 40)), "weights must be float32"),
    (dict(weights=torch.zeros(2, 2, 40, dtype=torch.float16)), "weights must be float32"),
    (dict(weights=torch.zeros(2, 2, 39)), "hold 39 positions"),
    (dict(weights=torch.zeros(2, 40, 2).transpose(1, 2)), "contiguous"),
    (dict(weights=torch.zeros(2, 2, 40), out_weights=torch.zeros(3, 2, 40)), "does not match"),
    (dict(weights=torch.zeros(2, 2, 40), weight_rows=[1, 1]), "distinct rows"),
    (dict(weights=torch.zeros(2, 2, 40), weight_rows=[0, 2]), "distinct rows"),
    (dict(weights=torch.zeros(2, 2, 40), weight_rows=[-1, 0]), "negative weight_rows"),
    (dict(weights=torch.zeros(2, 2, 40), weight_rows=[0]), "1 weight_rows for 2"),
    (dict(weights=torch.zeros(1, 2, 40)), "distinct rows"),
    ({}, "no CPU fallback"),
])
def test_attention_refuses(kw, match):
    with pytest.raises(RuntimeError, match=match):
        _attend(**kw)


def test_attention_refuses_overlapping_weights():
    buf = torch.zeros(2 * 2 * 40 + 7)
    w, o = buf[:160].view(2, 2, 40), buf[7:].view(2, 2, 40)
    with pytest.raises(RuntimeError, match="overlaps"):
        _attend(weights=w, out_weights=o)


@pytest.mark.parametrize("edit,match", [
    (lambda a: a.update(k_data=a["k_data"].view(torch.int8)), "must be uint8"),
    (lambda a: a.update(v_scale=a["v_scale"][:-1]), "views disagree"),
    (lambda a: a.update(v_data=a["v_data"][:, :8]), "views disagree"),
    (lambda a: a.update(k_scale=a["k_scale"].half()), "must be float32"),
    (lambda a: a.update(k_data=a["k_data"].transpose(1, 2).contiguous().transpose(1, 2)),
     "contiguous"),
])
def test_attention_refuses_caches(edit, match):
    with pytest.raises(RuntimeError, match=match):
        _attend(edit=edit)


def test_a_call_without_rows_needs_no_gpu():
    c = ref.Cache([5], 1, 16, 16)
    q = torch.ones(2, 1, 16, dtype=torch.bfloat16)
    assert not attend(q, *c.args(), [5], [0], 0.1).any()
    assert attend(q[:0], *c.args(), [], [], 0.1).shape == (0, 1, 16)


def test_numpy_lengths_and_tensors_are_lengths():
    c = ref.Cache([5, 7], 1, 16, 16)
    q = torch.ones(0, 1, 16, dtype=torch.bfloat16)
    for lens in (np.array([5, 7]), torch.tensor([5, 7]), (5, 7), [np.int32(5), 7]):
        assert attend(q, *c.args(), lens, [0, 0], 0.1).shape == (0, 1, 16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        evict(*c.args(), np.array([5, 7]), torch.zeros(2, 1, 7), np.int64(5))


@pytest.mark.parametrize("window,sinks,bad,ok", [
    (None, 0, [0, 3, 6], []),
    (20, 0, [4, 5, 6], [0, 1, 2, 3]),
    (20, 1, [0, 4, 5, 6], [1, 2, 3]),
    (20, 17, [0, 1, 5], [2, 3]),
    (20, 500, [0, 1, 2, 3, 4, 5, 6], []),
    (1, 0, [5, 6], [0, 1, 2, 3, 4]),
    (200, 0, [0, 6], []),
])
def test_pages_that_are_seen_are_checked(window, sinks, bad, ok):
    """100 positions, the last 5 the request's rows, pages of 16: the first row sits
    at 95."""
    host = np.arange(8, dtype=np.int64)[None]
    lens, news = np.array([100], dtype=np.int64), np.array([5], dtype=np.int64)
    fn = _native.lib().kvq_fp8_pth_window_check

    def check(table, index=np.int64):
        t = np.ascontiguousarray(table, dtype=index)
        return fn(t.ctypes.data, int(index is np.int64), 8, lens.ctypes.data, news.ctypes.data, 1,
                  8, 16, window or 0, sinks)

    assert check(host) == 0 and check(host, np.int32) == 0
    for i in [*bad, *ok, 7]:
        for value in (-1, 8):
            t = host.copy()
            t[0, i] = value
            assert check(t) == (1 if i in bad else 0), (i, value)
            assert check(t, np.int32) == (1 if i in bad else 0)


def test_a_page_outside_the_cache_is_refused():
    c = ref.Cache([40, 17], 2, 64, 16)
    host = c.host.copy()
    host[1, 1] = c.nb
    with pytest.raises(RuntimeError, match="request 1 sees"):
        attend(torch.zeros(2, 4, 64, dtype=torch.bfloat16), *c.args(), [40, 17], [1, 1], 0.1,
               block_table_host=host)
    # behind the last position, or behind the window: nobody sees it
    host = c.host.copy()
    host[1, 2] = -1
    host[0, 0] = -1
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        attend(torch.zeros(2, 4, 64, dtype=torch.bfloat16), *c.args(), [40, 17], [1, 1], 0.1,
               window=17, block_table_host=host)


def _evict(lens=(40, 17), keep=8, kvh=2, edit=None, **kw):
    c = ref.Cache(lens, kvh, 64, 16, spare=4)
    a = dict(k_data=c.k, k_scale=c.ks, v_data=c.v, v_scale=c.vs, block_table=c.table,
             seq_lens=list(lens), weights=torch.zeros(len(lens), kvh, max(lens)), keep=keep)
    a.update(kw)
    if edit:
        edit(a, c)
    return evict(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(sinks=-1), "not be negative"),
    (dict(recent=-1), "not be negative"),
    (dict(keep=-1), "negative keep"),
    (dict(keep=[8]), "1 budgets for 2"),
    (dict(sinks=5, recent=4), "under sinks"),
    (dict(seq_lens=[40, -17]), "negative seq_lens"),
    (dict(seq_lens=[400, 17], weights=torch.zeros(2, 2, 400)), "does not cover"),
    (dict(weights=torch.zeros(2, 2, 39)), "hold 39 positions"),
    (dict(weight_rows=[0, 0]), "distinct rows"),
    (dict(out_block_table=torch.zeros(2, 1, dtype=torch.int64)), "out_block_table is"),
    (dict(out_block_table=torch.zeros(1, 1, dtype=torch.int32)), "row per request"),
    ({}, "no CPU fallback"),
])
def test_eviction_refuses(kw, match):
    with pytest.raises(RuntimeError, match=match):
        _evict(**kw)


def test_eviction_refuses_pages_in_use_twice():
    def shared(a, c):
        a["block_table_host"] = c.host.copy()
        a["block_table_host"][1, 0] = c.host[0, 1]

    with pytest.raises(RuntimeError, match="request 1 has a page in use twice"):
        _evict(edit=shared)
    with pytest.raises(RuntimeError, match="in use twice"):  # whichever of the two moves
        _evict(edit=shared, keep=[40, 8])
    with pytest.raises(RuntimeError, match="in use twice"):
        _evict(edit=shared, keep=[8, 17])
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # neither does
        _evict(edit=shared, keep=40)

    def outside(a, c):
        a["block_table_host"] = c.host.copy()
        a["block_table_host"][0, 2] = c.nb

    with pytest.raises(RuntimeError, match="request 0 has a page outside"):
        _evict(edit=outside)

    def into(ids):
        def edit(a, c):
            free = [i for i in range(c.nb) if i not in set(c.host.reshape(-1).tolist())]
            t = [[free[0]], [free[1]]]
            for b, i in ids(c, free).items():
                t[b][0] = i
            a["out_block_table"] = torch.tensor(t, dtype=torch.int32)
        return edit

    with pytest.raises(RuntimeError, match="request 1 has a page in use twice"):
        _evict(edit=into(lambda c, free: {1: free[0]}))
    with pytest.raises(RuntimeError, match="request 0 has a page in use twice"):
        _evict(edit=into(lambda c, free: {0: int(c.host[1, 1])}))
    with pytest.raises(RuntimeError, match="request 1 has a page outside"):
        _evict(edit=into(lambda c, free: {1: -1}))
    with pytest.raises(RuntimeError, match="does not cover"):
        _evict(edit=into(lambda c, free: {}), keep=17)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _evict(edit=into(lambda c, free: {}))


def test_the_oracle_of_kept_rows():
    w = np.array([5, 1, 9, np.nan, 1, 0, -0.0, 0, 7, 7], dtype=np.float32)
    assert ref.kept_rows(w, 10, 10, 0, 0).tolist() == list(range(10))
    assert ref.kept_rows(w, 10, 3, 0, 0).tolist() == [2, 3, 8]
    assert ref.kept_rows(w, 10, 4, 1, 1).tolist() == [0, 2, 3, 9]
    assert ref.kept_rows(w, 10, 8, 0, 0).tolist() == [0, 1, 2, 3, 4, 5, 8, 9]
    assert ref.kept_rows(w, 10, 9, 0, 0).tolist() == [0, 1, 2, 3, 4, 5, 6, 8, 9]
