# SPDX-License-Identifier: Apache-2.0
"""Attention over pages with block scales, on the GPU against a 64-bit restatement
(``tests/_fp8_window.py`` derives the bounds), and a serving loop of store and attention."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests import _eight_bit as ref
from tests import _fp8_window as win
from vllm_ascend_quantized_kv_cache.ops.block8 import block8_attention, block8_store

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _check(device, lens, news, hq, kvh, d, bs, group, codes, dtype, window=None, sinks=0, *, seed=0,
           index=torch.int32, cache=None, q=None, host=True):
    c = cache or ref.Pages(lens, kvh, d, bs, group, codes, device=device, seed=seed, index=index)
    if q is None:
        q = win.query(sum(news), hq, d, dtype, device, seed=seed + 1)
    scale = d ** -0.5
    want, bound, _, _ = win.attention64(q, c, lens, news, scale, window, sinks)
    got = block8_attention(q, *c.args(), lens, news, scale, window=window, sinks=sinks,
                           block_table_host=c.host if host else None)
    win.check_out(got, want, bound, dtype)
    return got


LENGTHS = [
    ([1], [1]), ([2], [1]), ([15], [1]), ([16], [1]), ([17], [1]), ([64], [1]), ([65], [1]),
    ([600], [1]),
    # whole prompts, chunks, decodes and requests without rows or history, together
    ([7, 1, 130, 0, 257, 64], [7, 1, 2, 0, 100, 0]),
    ([300, 17, 1000], [300, 17, 1]),
    # more rows than history: the first ones see nothing
    ([5, 0, 40], [9, 3, 1]),
    ([1500], [333]),
]


@pytest.mark.parametrize("codes,group", [("e4m3", 32), ("int8", 16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (100, 4), (37, 300), (5000, 2)])
@pytest.mark.parametrize("lens,news", LENGTHS)
def test_lengths_and_windows(gpu_device, lens, news, window, sinks, codes, group):
    _check(gpu_device, lens, news, 8, 2, 128, 32, group, codes, BF16, window, sinks)


@pytest.mark.parametrize("hq,kvh,d,bs,group", [
    (8, 8, 64, 16, 16), (14, 2, 64, 32, 32), (10, 2, 128, 128, 128), (32, 8, 128, 128, 64),
    (7, 1, 128, 64, 32), (16, 1, 128, 16, 16), (8, 1, 256, 128, 128), (10, 2, 256, 48, 16),
    (3, 3, 256, 64, 32),
    # what the matrix kernels leave to the general one: other head sizes, pages or scales that
    # end inside a group of 16 positions, groups of more than 16 heads
    (4, 2, 80, 16, 16), (4, 1, 4, 16, 8), (2, 1, 512, 32, 32), (8, 2, 128, 24, 12),
    (40, 2, 128, 16, 16), (6, 2, 64, 1, 1), (8, 2, 128, 64, 8),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_head_layouts(gpu_device, hq, kvh, d, bs, group, dtype, codes):
    lens, news = [200, 71, 33], [1, 71, 6]
    _check(gpu_device, lens, news, hq, kvh, d, bs, group, codes, dtype, 50, 3, seed=3)
    _check(gpu_device, lens, news, hq, kvh, d, bs, group, codes, dtype, seed=4, index=torch.int64,
           host=False)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_fp32_queries(gpu_device, codes):
    _check(gpu_device, [150, 40], [20, 1], 6, 2, 128, 16, 16, codes, FP32, 60, 4)
    _check(gpu_device, [5003, 40], [2, 1], 6, 2, 128, 16, 16, codes, FP32)


@pytest.mark.parametrize("news", [[1] * 3, [5, 2, 3], [700, 513, 64]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1024, 4)])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_long_histories(gpu_device, news, window, sinks, codes):
    """Keys cut into parts and joined; several row tiles."""
    _check(gpu_device, [9000, 5003, 2048], news, 16, 4, 128, 128, 128, codes, BF16, window, sinks)


@pytest.mark.parametrize("d,hq,kvh", [(64, 4, 2), (256, 8, 1)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_long_chunks_other_heads(gpu_device, d, hq, kvh, dtype, codes):
    _check(gpu_device, [3000, 2999], [600, 1], hq, kvh, d, 64, 32, codes, dtype, 777, 33)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("d,hq,kvh,bs,group,news", [(80, 4, 2, 16, 16, [1, 3, 40]),
                                                  (128, 8, 2, 24, 8, [2, 1, 300])])
def test_long_histories_of_any_geometry(gpu_device, codes, d, hq, kvh, bs, group, news):
    _check(gpu_device, [5003, 1, 2048], news, hq, kvh, d, bs, group, codes, BF16, 700, 130)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("batch,n,hq,kvh,d", [(16, 8, 32, 8, 128), (64, 5, 20, 4, 64),
                                              (32, 4, 16, 2, 256)])
def test_a_few_rows_of_a_large_batch(gpu_device, batch, n, hq, kvh, d, codes):
    """25 or 32 rows and heads to a kv head, over enough positions for one pass over the codes;
    the requests share pages."""
    lens = [4000 - 9 * b for b in range(batch)] + [4000, 0, 37]
    news = [n - (b % 3 == 1) for b in range(batch)] + [1, 0, 1]
    c = ref.Pages([4000], kvh, d, 16, 16, codes, device=gpu_device, seed=5, spare=60)
    rng = np.random.default_rng(5)
    c.host = np.stack([rng.permutation(310)[:250] for _ in lens]).astype(np.int64)
    c.table = torch.from_numpy(c.host).to(gpu_device, torch.int32)
    _check(gpu_device, lens, news, hq, kvh, d, 16, 16, codes, BF16, 3500, 20, cache=c)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("news", [[1, 1], [70, 3]])
def test_scales_of_any_sign_and_size(gpu_device, codes, news):
    """Negative scales, and value scales from 2^-60 to 2^20 beside each other."""
    lens = [400, 90]
    c = ref.Pages(lens, 2, 128, 32, 16, codes, device=gpu_device, seed=8)
    g = torch.Generator().manual_seed(9)
    for i, s in enumerate(c.scale):
        sign = (torch.rand(s.shape, generator=g) < 0.5).float() * 2 - 1
        s *= sign.to(gpu_device)
        if i:
            s *= torch.exp2(torch.randint(-60, 20, s.shape, generator=g).float()).to(gpu_device)
    _check(gpu_device, lens, news, 8, 2, 128, 32, 16, codes, FP32, cache=c)
    for dtype in (BF16, FP16):
        q = win.query(sum(news), 8, 128, dtype, gpu_device)
        if dtype is FP16:
            c.scale[1] *= 2.0 ** -30  # results within its range
        _check(gpu_device, lens, news, 8, 2, 128, 32, 16, codes, dtype, 200, 5, cache=c, q=q)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 0.0, 2.0 ** -100])
@pytest.mark.parametrize("news", [[1, 2], [40, 3]])
def test_odd_value_scales(gpu_device, codes, value, news):
    """A block whose value scale is not finite spoils the rows that see it, and no others;
    one of nothing counts as nothing."""
    lens, d = [300, 60], 64
    c = ref.Pages(lens, 2, d, 16, 16, codes, device=gpu_device, seed=10)
    at = int(ref.slots_of(c.host, 0, [280], 16)[0]) // 16  # positions 272 - 287
    c.scale[1].view(-1, 2)[at, 1] = value
    if value == 2.0 ** -100:
        c.scale[1].view(-1, 2)[at, 1] = 0.0  # as the definition's bound takes it
    q = win.query(sum(news), 4, d, BF16, gpu_device)
    want, bound, _, _ = win.attention64(q, c, lens, news, 0.125)
    c.scale[1].view(-1, 2)[at, 1] = value
    got = block8_attention(q, *c.args(), lens, news, 0.125, block_table_host=c.host)
    if math.isfinite(value):
        win.check_out(got, want, bound, BF16)
        return
    sees = torch.zeros(got.shape[:2], dtype=torch.bool, device=gpu_device)
    for i in range(news[0]):
        sees[i, 2:] = 300 - news[0] + i >= 272
    assert not torch.isfinite(got[sees]).any()
    clean = ~sees
    win.check_out(got[clean], want[clean], bound[clean], BF16)


@pytest.mark.parametrize("news", [[1, 1], [40, 3], [5, 5]])
@pytest.mark.parametrize("window", [None, 30])
def test_nan_codes(gpu_device, news, window):
    """NaN codes reach the rows that see them and no others."""
    lens, d = [300, 60], 128
    c = ref.Pages(lens, 2, d, 16, 16, "e4m3", device=gpu_device, seed=11)
    for b, p, dim in ((0, 297, 3), (0, 250, 90), (1, 59, 127), (1, 10, 0)):
        c.data[1].view(-1, 2, d)[int(ref.slots_of(c.host, b, [p], 16)[0]), 1, dim] = 0xff
    c.data[0].view(-1, 2, d)[int(ref.slots_of(c.host, 0, [298], 16)[0]), 0, 5] = 0x7f
    _check(gpu_device, lens, news, 4, 2, d, 16, 16, "e4m3", BF16, window, 2 if window else 0, cache=c)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("news", [1, 40])
def test_stale_rows_and_pages(gpu_device, codes, news):
    """What lies behind a request's rows, and in pages that nobody sees, has no part in it."""
    lens, d = [301], 64
    c = ref.Pages(lens, 2, d, 16, 16, codes, device=gpu_device, seed=12)
    want = _check(gpu_device, lens, [news], 4, 2, d, 16, 16, codes, BF16, 50, 3, cache=c)
    last = int(ref.slots_of(c.host, 0, [300], 16)[0])
    for data in c.data:
        data.view(torch.uint8).view(-1, 2, d)[last + 1:last // 16 * 16 + 16] = 0x7f
    gone = c.host.copy()
    gone[0, 1:(301 - news - 50) // 16] = -1
    for scale in c.scale:
        scale[c.host[0, 2]] = math.nan
    table = torch.from_numpy(gone).to(gpu_device)
    q = win.query(news, 4, d, BF16, gpu_device)
    got = block8_attention(q, *c.args()[:4], table, lens, [news], d ** -0.5, window=50, sinks=3,
                           block_table_host=gone)
    assert torch.equal(got, want)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_queries_of_any_size(gpu_device, codes):
    """Rows far apart in size, beside each other: no row's size reaches another's result."""
    lens, news, d = [260, 33], [20, 1], 128
    c = ref.Pages(lens, 1, d, 16, 16, codes, device=gpu_device, seed=13)
    g = torch.Generator().manual_seed(14)
    q = torch.randn(21, 8, d, generator=g) * torch.exp2(
        torch.randint(-100, 6, (21, 8, 1), generator=g).float())
    q[3], q[4, 2] = 0.0, 2.0 ** -130
    q[5, :, ::2] *= 2.0 ** -12  # and dims within a row
    _check(gpu_device, lens, news, 8, 1, d, 16, 16, codes, BF16, cache=c,
           q=q.to(BF16).to(gpu_device))


def test_large_scores(gpu_device):
    """Scores of hundreds: a row's weight on a few positions, maxima that keep growing."""
    lens, d = [700], 128
    for codes in ("e4m3", "int8"):
        c = ref.Pages(lens, 2, d, 64, 64, codes, device=gpu_device, seed=15)
        for news in (1, 90):
            q = win.query(news, 8, d, FP16, gpu_device, size=40.0)
            _check(gpu_device, lens, [news], 8, 2, d, 64, 64, codes, FP16, cache=c, q=q)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("size", [2.0 ** 22, 2.0 ** 25, 2.0 ** 28, 2.0 ** 40])
def test_scores_beyond_their_steps(gpu_device, codes, size):
    """Where a score's step is 4, 16 and more, the weights of 16 bits stay finite."""
    lens, d = [300], 128
    c = ref.Pages(lens, 2, d, 64, 64, codes, device=gpu_device, seed=18)
    for news in (1, 60):
        q = win.query(news, 8, d, BF16, gpu_device, size=size)
        _check(gpu_device, lens, [news], 8, 2, d, 64, 64, codes, BF16, cache=c, q=q)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("shift", [1, 8])
def test_rows_off_their_bounds(gpu_device, codes, shift):
    """Queries and outputs at odd addresses; caches off a 16-byte bound."""
    lens, news, d, kvh = [130, 20], [9, 1], 64, 2
    c = ref.Pages(lens, kvh, d, 16, 16, codes, device=gpu_device, seed=16)
    q = win.query(10, 4, d, BF16, gpu_device)
    buf = torch.zeros(10 * 500 + shift, dtype=BF16, device=gpu_device)
    apart = buf[shift:].view(10, 500)[:, :256].view(10, 4, d)
    apart.copy_(q)
    want = _check(gpu_device, lens, news, 4, kvh, d, 16, 16, codes, BF16, cache=c, q=q)
    out = torch.zeros(10 * 256 + shift, dtype=BF16, device=gpu_device)[shift:].view(10, 4, d)
    got = block8_attention(apart, *c.args(), lens, news, d ** -0.5, out=out, block_table_host=c.host)
    assert got is out and torch.equal(out, want)
    moved = []
    for data in c.data:  # 4-byte bounds: the general kernel
        x = torch.zeros(data.numel() + 16, dtype=data.dtype, device=gpu_device)
        x[4:4 + data.numel()] = data.flatten()
        moved.append(x[4:4 + data.numel()].view(data.shape))
    c.data = moved
    _check(gpu_device, lens, news, 4, kvh, d, 16, 16, codes, BF16, cache=c, q=q)


def test_padded_batch_and_out(gpu_device):
    lens, news, d = [90, 40], [2, 1], 64
    c = ref.Pages(lens, 2, d, 16, 16, "int8", device=gpu_device, seed=17)
    q = win.query(7, 4, d, BF16, gpu_device)
    want, bound, _, _ = win.attention64(q[:3], c, lens, news, 0.125)
    got = block8_attention(q, *c.args(), lens, news, 0.125)
    win.check_out(got[:3], want, bound, BF16)
    assert (got[3:] == 0).all()
    for out in (torch.full((7, 4, d), 5.0, dtype=BF16, device=gpu_device),
                torch.full((7, d, 4), 5.0, dtype=BF16, device=gpu_device).transpose(1, 2),
                torch.full((7, 4, d), 5.0, dtype=FP32, device=gpu_device)):
        back = block8_attention(q, *c.args(), lens, news, 0.125, out=out)
        assert back is out and (out[3:] == 5.0).all()
        assert torch.equal(out[:3].to(BF16), got[:3])
    own = q.clone()
    assert torch.equal(block8_attention(own, *c.args(), lens, news, 0.125, out=own)[:3], got[:3])
    assert block8_attention(q[:0], *c.args(), [], [], 0.125).shape == (0, 4, d)
    assert (block8_attention(q, *c.args(), lens, [0, 0], 0.125) == 0).all()


@pytest.mark.parametrize("news", [[1, 1], [50, 1]])
def test_streams_and_graphs(gpu_device, news):
    lens, d = [2000, 700], 128
    c = ref.Pages(lens, 2, d, 128, 128, "e4m3", device=gpu_device, seed=18)
    q = win.query(sum(news), 8, d, BF16, gpu_device)
    want = _check(gpu_device, lens, news, 8, 2, d, 128, 128, "e4m3", BF16, cache=c, q=q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block8_attention(q, *c.args(), lens, news, d ** -0.5, block_table_host=c.host)
    also = block8_attention(q, *c.args(), lens, news, d ** -0.5, block_table_host=c.host)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(also, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one pool
        out = torch.zeros_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            block8_attention(q, *c.args(), lens, news, d ** -0.5, out=out, block_table_host=c.host)
        graphs.append(graph)
        outs.append(out)
    for i in range(3):
        q.copy_(win.query(sum(news), 8, d, BF16, gpu_device, seed=50 + i))
        for out in outs:
            out.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        want = block8_attention(q, *c.args(), lens, news, d ** -0.5, block_table_host=c.host)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("codes,group,d,bs", [("e4m3", 128, 128, 128), ("int8", 16, 64, 32)])
def test_a_serving_loop(gpu_device, codes, group, d, bs):
    """Prompts, then tokens: each step rotates, stores and attends.  Against rows quantized in
    one go from the definition, the results differ by what requantized rows add."""
    dev, kvh, hq = gpu_device, 2, 8
    prompts, steps = [150, 37, 1], 40
    lens = [n + steps for n in prompts]
    host, pages = ref.paged(lens, bs)
    host = host.astype(np.int64)
    cache = ref.BlockCache(pages, bs, kvh, d, group, codes, dev)
    table = torch.from_numpy(host).to(dev)
    cos_sin = ref.table(max(lens), d).to(dev)
    g = torch.Generator().manual_seed(20)
    at = [0] * len(prompts)
    for step in range(steps + 1):
        news = prompts if step == 0 else [1] * len(prompts)
        qkv = torch.randn(sum(news), hq + 2 * kvh, d, generator=g).to(BF16).to(dev)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + kvh], qkv[:, hq + kvh:]
        positions = [p for a, n in zip(at, news) for p in range(a, a + n)]
        slots = [s for b, (a, n) in enumerate(zip(at, news))
                 for s in ref.slots_of(host, b, range(a, a + n), bs).tolist()]
        at = [a + n for a, n in zip(at, news)]
        q = block8_store(k, v, torch.tensor(slots, device=dev), *cache.args(), query=q,
                         positions=torch.tensor(positions, device=dev), cos_sin=cos_sin)
        got = block8_attention(q, *cache.args(), table, at, news, d ** -0.5, block_table_host=host)
        if step % 13 == 0:
            view = ref.Pages.__new__(ref.Pages)
            view.__dict__.update(host=host, table=table, data=cache.data, scale=cache.scale,
                                 codes=codes, kvh=kvh, d=d, bs=bs, group=group)
            want, bound, _, _ = win.attention64(q, view, at, news, d ** -0.5)
            win.check_out(got, want, bound, BF16)
