# SPDX-License-Identifier: Apache-2.0
"""Windowed attention, running weights and eviction over the paged E4M3 cache, on
the GPU against 64-bit restatements (``tests/_fp8_window.py`` derives the bounds).
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests import _fp8_window as ref
from vllm_ascend_quantized_kv_cache.ops import fp8_ops, fp8_window

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
attend = fp8_window.fp8_per_token_head_window_attention
evict = fp8_window.fp8_per_token_head_evict


def _attend_and_check(device, lens, news, hq, kvh, d, bs, dtype, window, sinks, *, weigh=True,
                      index=torch.int32, seed=0, cache=None):
    c = cache or ref.Cache(lens, kvh, d, bs, device=device, seed=seed, index=index)
    q = ref.query(sum(news), hq, d, dtype, device, seed=seed + 1)
    scale = d ** -0.5
    out, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, window, sinks)
    kw = dict(window=window, sinks=sinks, block_table_host=c.host)
    got = attend(q, *c.args(), lens, news, scale, **kw)
    ref.check_out(got, out, bound, dtype)
    if weigh:
        rows = list(np.random.default_rng(seed).permutation(len(lens) + 2)[: len(lens)])
        before = torch.rand(len(lens) + 2, kvh, max(max(lens), 1) + 5, device=device)
        after = before.clone()
        again = attend(q, *c.args(), lens, news, scale, weights=before, out_weights=after,
                       weight_rows=rows, **kw)
        assert torch.equal(again.isnan(), got.isnan())
        assert torch.equal(again.nan_to_num(), got.nan_to_num())
        ref.check_weights(before, after, sums, sum_bounds, rows, lens, news)
        same = before.clone()
        attend(q, *c.args(), lens, news, scale, weights=same, weight_rows=rows, **kw)
        assert torch.equal(same.nan_to_num(), after.nan_to_num())


LENGTHS = [
    # one token of one request, from the first position on
    ([1], [1]), ([2], [1]), ([63], [1]), ([64], [1]), ([65], [1]), ([600], [1]),
    # whole prompts, chunks, decodes and requests without rows or history, together
    ([7, 1, 130, 0, 257, 64], [7, 1, 2, 0, 100, 0]),
    ([300, 17, 1000], [300, 17, 1]),
    # more rows than history: the first ones see nothing
    ([5, 0, 40], [9, 3, 1]),
    ([1500], [333]),
]


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (100, 4), (37, 300), (5000, 2)])
@pytest.mark.parametrize("lens,news", LENGTHS)
def test_lengths_and_windows(gpu_device, lens, news, window, sinks):
    _attend_and_check(gpu_device, lens, news, 8, 2, 128, 32, BF16, window, sinks)


@pytest.mark.parametrize("hq,kvh,d,bs", [
    (8, 8, 64, 16), (14, 2, 64, 32), (10, 2, 128, 128), (32, 8, 128, 128), (7, 1, 128, 64),
    (16, 1, 128, 16), (8, 1, 256, 128), (10, 2, 256, 16), (3, 3, 256, 64),
    # what the matrix kernels leave to the general ones: other head sizes, pages
    # that end inside a group of 16 positions, groups of more than 16 heads
    (4, 2, 80, 16), (4, 1, 4, 16), (2, 1, 512, 32), (8, 2, 128, 24), (40, 2, 128, 16),
    (6, 2, 64, 1),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_head_layouts(gpu_device, hq, kvh, d, bs, dtype):
    lens, news = [200, 71, 33], [1, 71, 6]
    _attend_and_check(gpu_device, lens, news, hq, kvh, d, bs, dtype, 50, 3, seed=3)
    _attend_and_check(gpu_device, lens, news, hq, kvh, d, bs, dtype, None, 0, seed=4,
                      index=torch.int64)


def test_fp32_queries(gpu_device):
    _attend_and_check(gpu_device, [150, 40], [20, 1], 6, 2, 128, 16, FP32, 60, 4)


@pytest.mark.parametrize("news", [[1] * 3, [5, 2, 3], [700, 513, 64]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1024, 4)])
def test_long_histories(gpu_device, news, window, sinks):
    """Keys cut into parts and joined; several row tiles."""
    _attend_and_check(gpu_device, [9000, 5003, 2048], news, 16, 4, 128, 128, BF16, window, sinks)


@pytest.mark.parametrize("hq,kvh,d,bs,dtype", [
    (6, 2, 80, 16, BF16), (4, 1, 4, 16, FP16), (2, 1, 512, 32, BF16), (3, 1, 260, 16, FP16),
    (5, 5, 12, 1, BF16), (4, 2, 160, 64, BF16), (8, 2, 128, 24, FP16), (40, 2, 128, 16, BF16),
    (4, 2, 64, 16, FP32), (4, 2, 96, 128, FP32),
])
@pytest.mark.parametrize("news", [[1, 1, 1], [3, 1, 40], [300, 2, 0]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 130)])
def test_long_histories_of_any_geometry(gpu_device, hq, kvh, d, bs, dtype, news, window, sinks):
    """The general kernels' parts: rows that see more, fewer and none of a part's positions."""
    _attend_and_check(gpu_device, [5003, 1, 2048], news, hq, kvh, d, bs, dtype, window, sinks)


@pytest.mark.parametrize("news", [[12000], [3000], [700, 12000]])
def test_long_prompts(gpu_device, news):
    """Whole prompts: many tiles, columns in segments, few and many of them."""
    _attend_and_check(gpu_device, [12000] * len(news), news, 2, 1, 64, 64, BF16, None, 0)


@pytest.mark.parametrize("kvh,hq", [(1, 2), (1, 15), (1, 16)])
def test_one_request_over_many_positions(gpu_device, kvh, hq):
    """Hundreds of parts of a row; scores from the decode, and keys read again."""
    _attend_and_check(gpu_device, [150000], [1], hq, kvh, 64, 64, FP16, None, 0)
    _attend_and_check(gpu_device, [150000], [1], hq, kvh, 64, 64, BF16, 100000, 3000)


@pytest.mark.parametrize("d,hq,kvh", [(64, 4, 2), (256, 8, 1)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_long_chunks_other_heads(gpu_device, d, hq, kvh, dtype):
    _attend_and_check(gpu_device, [3000, 2999], [600, 1], hq, kvh, d, 64, dtype, 777, 33)


@pytest.mark.parametrize("window,sinks", [(None, 0), (3500, 20)])
@pytest.mark.parametrize("batch,n,hq,kvh,d", [(16, 8, 32, 8, 128), (64, 5, 20, 4, 64),
                                              (32, 4, 16, 2, 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_few_rows_of_a_large_batch(gpu_device, batch, n, hq, kvh, d, dtype, window, sinks):
    """25 or 32 rows and heads to a kv head, over enough positions for one pass over
    the codes, beside single tokens, a longer chunk and a request without history.
    The requests share pages, and values that are NaN: seen by all rows of some
    requests, by some rows of others, by none of others."""
    lens = [4000 - 9 * b for b in range(batch)] + [4000, 0, 37, 300]
    news = [n - (b % 3 == 1) for b in range(batch)] + [1, 0, 1, 50]
    c = ref.Cache([4000], kvh, d, 16, device=gpu_device, seed=5, spare=60)
    rng = np.random.default_rng(5)
    c.host = np.stack([rng.permutation(c.nb)[:250] for _ in lens]).astype(np.int64)
    c.table = torch.from_numpy(c.host).to(gpu_device, torch.int32)
    c.lens = lens
    for b, back, dim in ((0, 2, 3), (1, 1, d - 1), (2, 60, 17)):
        c.v.view(-1, kvh, d)[int(c.slots(b, lens[b] - back)), 0, dim] = 0xff
    _attend_and_check(gpu_device, lens, news, hq, kvh, d, 16, dtype, window, sinks, cache=c)


def test_many_requests(gpu_device):
    """More requests than one launch's argument holds, some without rows."""
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(1, 90, 300)]
    news = [int(min(n, m)) for n, m in zip(lens, rng.integers(0, 4, 300))]
    _attend_and_check(gpu_device, lens, news, 4, 2, 64, 16, BF16, 20, 2)


@pytest.mark.parametrize("n", [1, 4, 90])
@pytest.mark.parametrize("window,sinks", [(None, 0), (64, 5)])
def test_nan_in_masked_places_stays_there(gpu_device, n, window, sinks):
    """NaN codes and scales behind the sequence, and at seen positions, reach exactly
    the rows that see them."""
    lens = [300, 200]
    c = ref.Cache(lens, 2, 128, 32, device=gpu_device, seed=7)
    k, v = c.k.view(-1, 2, 128), c.v.view(-1, 2, 128)
    ks, vs = c.ks.view(-1, 2), c.vs.view(-1, 2)
    for b, length in enumerate(lens):  # stale rows behind the last position
        width = c.host.shape[1] * c.bs
        stale = torch.from_numpy(c.slots(b, np.arange(length, width))).to(gpu_device)
        k[stale], v[stale] = 0x7F, 0xFF
        ks[stale], vs[stale] = math.nan, math.inf
    # a NaN value element, a NaN key and a NaN value scale: near the end of request 0,
    # where only its last rows see them, and early in request 1
    s0 = c.slots(0, np.array([300 - max(1, n // 2)]))[0]
    v[s0, 0, 77] = 0x7F
    s1 = c.slots(1, np.array([90]))[0]
    vs[s1, 1] = math.nan
    if n > 1:
        s2 = c.slots(0, np.array([299]))[0]
        k[s2, 1, 3] = 0x7F
    _attend_and_check(gpu_device, lens, [n, n], 8, 2, 128, 32, BF16, window, sinks, cache=c)


def test_value_rows_of_any_size(gpu_device):
    """Value scales from 1e-6 to 1e4 side by side: the large rows' small weights count."""
    c = ref.Cache([700, 700], 2, 128, 32, device=gpu_device, seed=9, value_spread=4.0)
    for news in ([1, 1], [300, 40]):
        _attend_and_check(gpu_device, [700, 700], news, 8, 2, 128, 32, FP16, None, 0, cache=c)


def test_large_scores(gpu_device):
    """Scores in the hundreds: the offset follows the maximum wherever it comes."""
    c = ref.Cache([900], 1, 128, 32, device=gpu_device, seed=10)
    c.ks.mul_(torch.linspace(1.0, 40.0, c.nb * 32, device=gpu_device).view(c.nb, 32, 1, 1))
    for n in (1, 200):
        _attend_and_check(gpu_device, [900], [n], 4, 1, 128, 32, BF16, None, 0, cache=c)


def test_vanished_pages_and_padded_views(gpu_device):
    """Pages behind the window may have any id; rows of a fused projection and padded
    rows; rows of `out` behind the last request's stay."""
    lens, news, window, sinks = [2000, 900], [3, 70], 256, 20
    c = ref.Cache(lens, 2, 128, 32, device=gpu_device, seed=11)
    fused = ref.query(80, 8 + 4, 128, BF16, gpu_device)
    q = fused[:, :8]
    scale = 128 ** -0.5
    want, bound, _, _ = ref.attention64(q[:73], c, lens, news, scale, window, sinks)
    table, host = c.table.clone(), c.host.copy()
    for b in range(2):
        gone = range(-(-sinks // 32), (lens[b] - news[b] - window + 1) // 32)
        for i in gone:
            host[b, i] = (-1, 10**6)[i % 2]
    table.copy_(torch.from_numpy(host))
    out = torch.full((80, 8, 128), 7.0, dtype=BF16, device=gpu_device)
    got = attend(q, *c.args()[:4], table, lens, news, scale, window=window, sinks=sinks, out=out,
                 block_table_host=host)
    assert got is out and bool((out[73:] == 7.0).all())
    ref.check_out(out[:73], want, bound, BF16)
    fresh = attend(q, *c.args()[:4], table, lens, news, scale, window=window, sinks=sinks)
    assert torch.equal(fresh[:73], out[:73]) and not fresh[73:].any()
    # into the query's own memory, and into a wider type
    own = q[:73].contiguous()
    attend(own, *c.args()[:4], table, lens, news, scale, window=window, sinks=sinks, out=own)
    assert torch.equal(own, out[:73])
    wide = torch.zeros(73, 8, 128, device=gpu_device)
    attend(q[:73], *c.args()[:4], table, lens, news, scale, window=window, sinks=sinks, out=wide)
    assert torch.equal(wide, out[:73].float())


def test_caches_and_queries_at_odd_addresses(gpu_device):
    lens, news = [300, 90], [1, 40]
    c = ref.Cache(lens, 2, 128, 32, device=gpu_device, seed=12)
    def moved(t, by):
        buf = torch.zeros(t.numel() + 64, dtype=t.dtype, device=gpu_device)
        view = buf[by:by + t.numel()].view(t.shape)
        view.copy_(t)
        return view
    c.k, c.v = moved(c.k, 4), moved(c.v, 12)
    _attend_and_check(gpu_device, lens, news, 8, 2, 128, 32, BF16, 100, 4, cache=c)
    c.k, c.v = moved(c.k, 16), moved(c.v, 16)
    q = ref.query(sum(news), 8, 128, BF16, gpu_device)
    want = attend(q, *c.args(), lens, news, 0.1)
    odd = moved(q, 1)
    out = moved(torch.zeros_like(q), 3)
    attend(odd, *c.args(), lens, news, 0.1, out=out)
    assert torch.equal(out, want)


def test_another_stream_and_a_captured_call(gpu_device):
    lens, news = [2500, 700], [1, 130]
    c = ref.Cache(lens, 2, 128, 32, device=gpu_device, seed=13)
    q = ref.query(sum(news), 8, 128, BF16, gpu_device)
    w0 = torch.rand(2, 2, 2500, device=gpu_device)
    w1 = torch.zeros_like(w0)
    kw = dict(window=1500, sinks=4, block_table_host=c.host)
    want = attend(q, *c.args(), lens, news, 0.1, weights=w0, out_weights=w1, **kw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    w2 = torch.zeros_like(w0)
    with torch.cuda.stream(side):
        got = attend(q, *c.args(), lens, news, 0.1, weights=w0, out_weights=w2, **kw)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(w1, w2)
    out, w3 = torch.zeros_like(q), torch.zeros_like(w0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(q, *c.args(), lens, news, 0.1, weights=w0, out_weights=w3, out=out, **kw)
    for seed in range(3):
        q.copy_(ref.query(sum(news), 8, 128, BF16, gpu_device, seed=20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        again = attend(q, *c.args(), lens, news, 0.1, weights=w0, out_weights=w1, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(w3, w1)


@pytest.mark.parametrize("dtype,d", [(BF16, 96), (FP32, 128)])
def test_more_rows_than_history_in_any_geometry(gpu_device, dtype, d):
    _attend_and_check(gpu_device, [5, 0, 900], [9, 3, 1000], 6, 2, d, 16, dtype, None, 0)
    _attend_and_check(gpu_device, [5, 0, 900], [9, 3, 1000], 6, 2, d, 16, dtype, 70, 66)


def test_many_requests_of_any_geometry(gpu_device):
    """More than a launch takes, some of them in parts."""
    lens = [(97 * b) % 701 for b in range(250)]
    news = [(b * 7) % 4 for b in range(250)]
    _attend_and_check(gpu_device, lens, news, 4, 2, 80, 16, FP16, None, 0)
    _attend_and_check(gpu_device, lens, news, 4, 2, 80, 16, FP16, 130, 70)


@pytest.mark.parametrize("batch,lens,n,hq,kvh,d", [
    (16, 4000, 8, 32, 8, 128),  # two groups of columns
    (3, 900, 2, 6, 2, 96),      # the general kernels
    (2, 3000, 300, 8, 2, 128),  # tiles of 256 rows
])
def test_streams_and_graphs_of_every_kernel(gpu_device, batch, lens, n, hq, kvh, d):
    """Two calls at once on two streams, and replays of a captured one."""
    c = ref.Cache([lens] * batch, kvh, d, 32, device=gpu_device, seed=15)
    ls, ns = [lens] * batch, [n] * batch
    qs = [ref.query(sum(ns), hq, d, BF16, gpu_device, seed=s) for s in (1, 2)]
    w0 = torch.rand(batch, kvh, lens, device=gpu_device)

    def call(q, w, **kw):
        return attend(q, *c.args(), ls, ns, 0.1, weights=w0, out_weights=w,
                      block_table_host=c.host, **kw)

    wants, ws = [], [torch.zeros_like(w0) for _ in range(4)]
    for q, w in zip(qs, ws):
        wants.append(call(q, w))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    gots = []
    for q, w, stream in zip(qs, ws[2:], streams):
        with torch.cuda.stream(stream):
            gots.append(call(q, w))
    torch.cuda.synchronize()
    for a, b in zip(gots + ws[2:], wants + ws[:2]):
        assert torch.equal(a, b)
    q, out, w3 = qs[0].clone(), torch.zeros_like(qs[0]), torch.zeros_like(w0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q, w3, out=out)
    for k in (1, 0, 1):
        q.copy_(qs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wants[k]) and torch.equal(w3, ws[k])
        assert torch.equal(call(qs[1 - k], ws[2]), wants[1 - k])
        torch.cuda.synchronize()


def test_agrees_with_the_rounded_rows_of_the_older_call(gpu_device):
    lens = [1000, 77]
    c = ref.Cache(lens, 2, 128, 32, device=gpu_device, seed=14)
    q = ref.query(2, 8, 128, BF16, gpu_device)
    a = attend(q, *c.args(), lens, [1, 1], 0.1)
    b = fp8_ops.fp8_per_token_head_attention(q, *c.args(), lens, [1, 1], 0.1)
    assert torch.allclose(a.float(), b.float(), atol=2e-2, rtol=2e-2)


# ---- eviction -----------------------------------------------------------------------


def _weights(rows, kvh, cols, seed, kind):
    rng = np.random.default_rng(seed)
    w = rng.standard_normal((rows, kvh, cols)).astype(np.float32)
    if kind == "ties":
        w = np.round(w)
    elif kind == "heavy":
        w = np.where(w < -0.5, np.float32(0), np.exp(3 * w))
    elif kind == "special":
        w = np.where(rng.random(w.shape) < 0.5, np.round(w) * np.float32(1e-40), w)
        at = rng.random(w.shape)
        w[at < 0.02], w[(at > 0.02) & (at < 0.04)] = np.nan, -np.nan
        w[(at > 0.04) & (at < 0.06)], w[(at > 0.06) & (at < 0.08)] = np.inf, -np.inf
        w[(at > 0.08) & (at < 0.2)], w[(at > 0.2) & (at < 0.3)] = 0.0, -0.0
    elif kind == "equal":
        w[:] = 1.0
    return w


def _evict_and_check(device, lens, keep, sinks, recent, kvh, d, bs, kind, *, fresh, seed=0,
                     index=torch.int32):
    batch = len(lens)
    keeps = [keep] * batch if isinstance(keep, int) else keep
    c = ref.Cache(lens, kvh, d, bs, device=device, seed=seed, index=index,
                  spare=2 + (sum(-(-min(n, k) // bs) for n, k in zip(lens, keeps)) if fresh else 0))
    rows = [int(r) for r in np.random.default_rng(seed).permutation(batch + 1)[:batch]]
    host_w = _weights(batch + 1, kvh, max(max(lens), 1) + 3, seed, kind)
    w = torch.from_numpy(host_w).to(device)
    images = [t.cpu().clone() for t in (c.k, c.ks, c.v, c.vs)]
    stay = [min(n, k) for n, k in zip(lens, keeps)]
    kw, dst = {}, c.host
    out_w = w
    if fresh:
        width = max(1, max(-(-n // bs) for n in stay))
        free = iter(sorted(set(range(c.nb)) - {int(i) for b, n in enumerate(lens)
                                               for i in c.host[b, : -(-n // bs)]}, reverse=True))
        dst = np.full((batch, width), -5, dtype=np.int64)
        for b, n in enumerate(stay):
            dst[b, : -(-n // bs)] = [next(free) for _ in range(-(-n // bs))]
        out_w = torch.full_like(w, 3.0)
        kw = dict(out_block_table=torch.from_numpy(dst).to(device, index), out_weights=out_w)
    new_lens, kept = evict(*c.args(), lens, w, keep, sinks=sinks, recent=recent, weight_rows=rows,
                           **kw)
    torch.cuda.synchronize()
    assert new_lens == stay and kept.dtype == torch.int32
    kept = kept.cpu().numpy()
    assert kept.shape == (batch, kvh, max(stay))
    want_w = host_w.copy() if not fresh else np.full_like(host_w, 3.0)
    want = [t.clone() for t in images]
    for b, n in enumerate(lens):
        for h in range(kvh):
            ids = ref.kept_rows(host_w[rows[b], h], n, keeps[b], sinks, recent)
            np.testing.assert_array_equal(kept[b, h, : stay[b]], ids)
            assert (kept[b, h, stay[b]:] == -1).all()
            want_w[rows[b], h, : stay[b]] = host_w[rows[b], h, ids]
            src = torch.from_numpy(c.slots(b, ids))
            at = np.arange(stay[b])
            to = torch.from_numpy(dst[b, at // bs] * bs + at % bs)
            for t, old in zip(want, images):
                t.view(-1, kvh, t.shape[-1])[to, h] = old.view(-1, kvh, t.shape[-1])[src, h]
    for got, t in zip((c.k, c.ks, c.v, c.vs), want):  # whole images: nothing else moved
        assert torch.equal(got.cpu(), t)
    got_w = out_w.cpu().numpy()
    np.testing.assert_array_equal(got_w.view(np.uint32), want_w.view(np.uint32))


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("kind", ["plain", "ties", "heavy", "special", "equal"])
def test_eviction(gpu_device, kind, fresh):
    _evict_and_check(gpu_device, [700, 1, 0, 333, 64, 65], 64, 4, 17, 2, 128, 32, kind, fresh=fresh)
    _evict_and_check(gpu_device, [3000, 2049], [1500, 1024], 0, 0, 3, 64, 16, kind, fresh=fresh,
                     seed=1, index=torch.int64)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (8, 3, 5), (99, 0, 99),
                                               (99, 50, 0), (100, 60, 30), (101, 7, 2)])
def test_eviction_budgets(gpu_device, keep, sinks, recent, fresh):
    _evict_and_check(gpu_device, [100, 40], keep, sinks, recent, 2, 128, 16, "heavy", fresh=fresh)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("d,bs", [(4, 16), (80, 24), (256, 128), (64, 1), (20, 8)])
def test_eviction_head_sizes(gpu_device, d, bs, fresh):
    _evict_and_check(gpu_device, [500, 260], 130, 2, 30, 2, d, bs, "ties", fresh=fresh)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("keep", [500, 33000])
def test_eviction_of_long_rows(gpu_device, keep, fresh):
    """Rows of weights past what a workgroup keeps at hand, and just within."""
    _evict_and_check(gpu_device, [40003, 32768, 32769], keep, 16, 400, 1, 64, 64, "heavy",
                     fresh=fresh)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("kind", ["ties", "special", "equal"])
def test_eviction_of_long_rows_with_ties(gpu_device, kind, fresh):
    """Thresholds among equal weights and NaN, across the chunks of a long row."""
    _evict_and_check(gpu_device, [50001, 100, 33000], [20000, 100, 32000], 3, 7, 2, 16, 64, kind,
                     fresh=fresh)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("keep,sinks,recent", [(300, 100, 200), (1, 0, 0), (40000, 39990, 10),
                                               (40000, 0, 40000), (17000, 16500, 0)])
def test_eviction_budgets_of_long_rows(gpu_device, keep, sinks, recent, fresh):
    """Nothing to choose, one row, and rows that stay across chunks."""
    _evict_and_check(gpu_device, [50001], keep, sinks, recent, 1, 16, 64, "special", fresh=fresh)


def test_eviction_of_many_requests(gpu_device):
    rng = np.random.default_rng(3)
    lens = [int(n) for n in rng.integers(0, 60, 400)]
    _evict_and_check(gpu_device, lens, 20, 2, 3, 1, 16, 16, "ties", fresh=False)
    _evict_and_check(gpu_device, lens, 20, 2, 3, 1, 16, 16, "ties", fresh=True)


def test_captured_evictions(gpu_device):
    """Into fresh pages, short and long rows; replays follow the weights."""
    lens, keep = [40000, 900], 500
    c = ref.Cache(lens, 2, 64, 64, device=gpu_device, seed=6, spare=40)
    used = set(c.host.reshape(-1).tolist())
    free = [i for i in range(c.nb) if i not in used][:16]
    dst = torch.tensor(free, dtype=torch.int32, device=gpu_device).view(2, 8)
    w = torch.rand(2, 2, 40000, device=gpu_device)
    out_w = torch.zeros_like(w)
    kw = dict(sinks=4, recent=50, out_block_table=dst, out_weights=out_w, block_table_host=c.host,
              out_block_table_host=dst.cpu().numpy().astype(np.int64))
    evict(*c.args(), lens, w, keep, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, kept = evict(*c.args(), lens, w, keep, **kw)
    for seed in range(3):
        w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (kept, c.k, c.ks, c.v, c.vs, out_w)]
        _, again = evict(*c.args(), lens, w, keep, **kw)
        torch.cuda.synchronize()
        for a, b in zip(got, (again, c.k, c.ks, c.v, c.vs, out_w)):
            assert torch.equal(a, b)
        ids = ref.kept_rows(w[0, 1].cpu().numpy(), lens[0], keep, 4, 50)
        np.testing.assert_array_equal(again[0, 1].cpu().numpy(), ids)


def test_no_requests(gpu_device):
    c = ref.Cache([10], 1, 16, 16, device=gpu_device)
    new_lens, kept = evict(*c.args(), [], torch.ones(1, 1, 10, device=gpu_device), 4)
    assert new_lens == [] and kept.shape == (0, 1, 0)


def test_nothing_to_keep(gpu_device):
    c = ref.Cache([10], 1, 16, 16, device=gpu_device)
    w = torch.ones(1, 1, 10, device=gpu_device)
    new_lens, kept = evict(*c.args(), [10], w, 0)
    assert new_lens == [0] and kept.shape == (1, 1, 0)


def test_shared_prefix_pages_move_into_fresh_ones(gpu_device):
    c = ref.Cache([96, 96], 1, 64, 32, device=gpu_device, spare=6, seed=4)
    c.host[1, :2] = c.host[0, :2]  # a common prefix of two pages
    c.table.copy_(torch.from_numpy(c.host))
    w = torch.rand(2, 1, 96, device=gpu_device)
    used = set(c.host.reshape(-1).tolist())
    free = [i for i in range(c.nb) if i not in used][:4]
    dst = torch.tensor(free, dtype=torch.int32, device=gpu_device).view(2, 2)
    old = c.rows(0, 96)[0], c.rows(1, 96)[0]
    new_lens, kept = evict(*c.args(), [96, 96], w.clone(), 40, out_block_table=dst)
    assert new_lens == [40, 40]
    c.host, c.table = dst.cpu().numpy().astype(np.int64), dst
    for b in range(2):
        assert torch.equal(c.rows(b, 40)[0], old[b][kept[b, 0].long()])


def test_a_bounded_serving_loop(gpu_device):
    """Store, attend with weights, evict, go on: against 64 bits at every step."""
    kvh, hq, d, bs, budget = 2, 8, 128, 16, 96
    lens, rows, scale = [0, 0, 0], [2, 0, 1], 128 ** -0.5
    c = ref.Cache([256] * 3, kvh, d, bs, device=gpu_device, seed=21)
    c.lens = lens
    w = torch.rand(4, kvh, 256, device=gpu_device)
    spare = w[3].clone()
    g = torch.Generator().manual_seed(22)
    for step, news in enumerate([[150, 40, 7], [1, 1, 1], [1, 30, 1], [0, 64, 1], [20, 1, 100]]):
        n = sum(news)
        k = torch.randn(n, kvh, d, generator=g).to(BF16).to(gpu_device)
        v = torch.randn(n, kvh, d, generator=g).to(BF16).to(gpu_device)
        lens = [a + b for a, b in zip(lens, news)]
        slots = np.concatenate([c.slots(b, np.arange(lens[b] - news[b], lens[b]))
                                for b in range(3)])
        fp8_ops.fp8_per_token_head_store(k, v, torch.from_numpy(slots).to(gpu_device), c.k, c.ks,
                                         c.v, c.vs)
        q = ref.query(n, hq, d, BF16, gpu_device, seed=30 + step)
        window, sinks = (None, 0) if step % 2 else (80, 4)
        want, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, window, sinks)
        before = w.clone()
        got = attend(q, *c.args(), lens, news, scale, window=window, sinks=sinks, weights=w,
                     weight_rows=rows)
        ref.check_out(got, want, bound, BF16)
        ref.check_weights(before, w, sums, sum_bounds, rows, lens, news)
        old = [c.rows(b, lens[b]) for b in range(3)]
        old_w = w.cpu().numpy()
        new_lens, kept = evict(*c.args(), lens, w, budget, sinks=4, recent=16, weight_rows=rows)
        for b in range(3):
            assert new_lens[b] == min(lens[b], budget)
            now = c.rows(b, new_lens[b])
            for h in range(kvh):
                ids = ref.kept_rows(old_w[rows[b], h], lens[b], budget, 4, 16)
                np.testing.assert_array_equal(kept[b, h, : new_lens[b]].cpu().numpy(), ids)
                for a, z in zip(now, old[b]):
                    assert torch.equal(a[:, h], z[torch.from_numpy(ids).to(gpu_device), h])
        lens = new_lens
    assert torch.equal(w[3], spare)
