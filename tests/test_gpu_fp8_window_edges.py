# SPDX-License-Identifier: Apache-2.0
"""Windowed attention, running weights and eviction over the paged E4M3 cache, on
the GPU: calls and values at the edges of what is allowed."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests import _fp8_window as ref
from vllm_ascend_quantized_kv_cache.ops import fp8_window

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
attend = fp8_window.fp8_per_token_head_window_attention
evict = fp8_window.fp8_per_token_head_evict


# ---- requests without new rows ---------------------------------------------------


@pytest.mark.parametrize("hq,kvh,d,bs,dtype", [(8, 2, 128, 32, BF16), (4, 2, 64, 16, FP16),
                                               (6, 2, 96, 16, BF16), (4, 1, 64, 16, FP32)])
@pytest.mark.parametrize("news", [[2, 0, 0, 70, 0], [0, 0, 0, 0, 1], [0] * 5])
def test_weights_of_idle_requests_go_on(gpu_device, hq, kvh, d, bs, dtype, news):
    """A step's ``out_weights`` hold every request's running weights: those of one
    without rows as they were, up to its length."""
    lens, rows, cols = [300, 1500, 0, 90, 1], [4, 0, 5, 2, 1], 1507
    c = ref.Cache(lens, kvh, d, bs, device=gpu_device, seed=31)
    q = ref.query(sum(news), hq, d, dtype, gpu_device)
    scale = d ** -0.5
    out, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, 200, 4)
    before = torch.rand(7, kvh, cols, device=gpu_device)
    start = torch.full_like(before, -3.0)
    for b, r in enumerate(rows):  # what the step leaves of the old weights, and where
        start[r, :, :lens[b]] = before[r, :, :lens[b]]
    after = torch.full_like(before, -3.0)
    got = attend(q, *c.args(), lens, news, scale, window=200, sinks=4, weights=before,
                 out_weights=after, weight_rows=rows, block_table_host=c.host)
    ref.check_out(got, out, bound, dtype)
    ref.check_weights(start, after, sums, sum_bounds, rows, lens, news)
    same = before.clone()
    attend(q, *c.args(), lens, news, scale, window=200, sinks=4, weights=same, weight_rows=rows,
           block_table_host=c.host)
    for b, r in enumerate(rows):
        assert torch.equal(same[r, :, :lens[b]], after[r, :, :lens[b]])
        assert torch.equal(same[r, :, lens[b]:], before[r, :, lens[b]:])


def test_weights_of_many_idle_requests(gpu_device):
    """More than a launch's argument holds, two buffers in turn."""
    lens = [(53 * b) % 97 for b in range(260)]
    c = ref.Cache(lens, 1, 64, 16, device=gpu_device, seed=32)
    w = [torch.rand(260, 1, 97, device=gpu_device), torch.full((260, 1, 97), -1.0,
                                                               device=gpu_device)]
    one = w[0].clone()
    for step in range(4):
        news = [int(b % 50 == step and lens[b] > 0) for b in range(260)]
        q = ref.query(sum(news), 2, 64, BF16, gpu_device, seed=step)
        attend(q, *c.args(), lens, news, 0.1, weights=w[step % 2], out_weights=w[1 - step % 2])
        attend(q, *c.args(), lens, news, 0.1, weights=one)
    for b, n in enumerate(lens):
        assert torch.equal(w[0][b, :, :n], one[b, :, :n])


# ---- probabilities of any size -----------------------------------------------------


def _constant_rows(device, length, d, heavy, light, every=64):
    """One request whose keys give the scores `heavy` (every `every`th position) and
    `light`, exact for a query of ones and a scale of 1 / D; the heavy rows' values
    are 1 in dim 0, the light ones' 448 in dim 1, zeros elsewhere."""
    c = ref.Cache([length], 1, d, 64, device=device, seed=33)
    c.k.fill_(0x38)
    at = torch.from_numpy(c.slots(0, np.arange(length))).to(device)
    big = torch.arange(length, device=device) % every == 0
    c.ks.view(-1)[at] = torch.where(big, heavy, light).float()
    c.vs.fill_(1.0)
    c.v.zero_()
    v = c.v.view(-1, d)
    v[at[big], 0] = 0x38
    v[at[~big], 1] = 0x7E
    return c


@pytest.mark.parametrize("n,hq,d", [(1, 8, 128), (60, 8, 64), (40, 8, 128), (100, 8, 128),
                                    (2, 64, 128), (40, 8, 256), (40, 8, 96)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("below", [16.0, 25.6, 31.0])
def test_small_weights_count_beside_large_ones(gpu_device, n, hq, d, dtype, below):
    """Weights of 2^-below of the largest: they alone fill dim 1 of the result.

    Off by half a step of the result; by the weights' rounding to 16 bits, 2^-11 of
    each, or 2^-32 of the largest where that is more; and by 2^-16 for the fp32
    arithmetic (exp2 of exponents up to 32: 32 2^-24, and sums of 700 terms)."""
    length = 700
    heavy = float(np.float32(below * math.log(2.0)))
    c = _constant_rows(gpu_device, length, d, heavy, 0.0)
    q = torch.ones(n, hq, d, dtype=dtype, device=gpu_device)
    got = attend(q, *c.args(), [length], [n], 1.0 / d, block_table_host=c.host).double()
    pos = torch.arange(length - n, length, device=gpu_device, dtype=torch.float64)
    big = torch.floor(pos / 64) + 1
    w = math.exp(-heavy)
    norm = big + (pos + 1 - big) * w
    want = torch.zeros(n, d, dtype=torch.float64, device=gpu_device)
    want[:, 0], want[:, 1] = big / norm, 448 * (pos + 1 - big) * w / norm
    off = (got - want[:, None]).abs()
    part = ref.HALF_STEP[dtype] + 2.0 ** -11 + 2.0 ** -16
    tiny = float(torch.finfo(dtype).smallest_normal) * ref.HALF_STEP[dtype] * 2
    limit = want * (part + torch.tensor([0, 2.0 ** -32 / w] + [0] * (d - 2), device=gpu_device))
    assert bool((off <= limit[:, None] + tiny).all()), (off - limit[:, None]).max().item()


# ---- value scales of any kind --------------------------------------------------------


@pytest.mark.parametrize("n,hq,kvh,d", [(1, 8, 2, 128), (3, 8, 2, 128), (40, 8, 2, 128),
                                        (300, 8, 2, 128), (60, 4, 2, 64), (40, 8, 1, 256),
                                        (40, 6, 2, 96)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 7)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_value_scales_of_any_sign(gpu_device, n, hq, kvh, d, window, sinks, dtype):
    """Negative scales, zero and tiny ones, whichever kernel the rows go to: V is
    code * scale."""
    lens = [500, 37]
    news = [n, min(n, 37)]
    c = ref.Cache(lens, kvh, d, 32, device=gpu_device, seed=34)
    vs = c.vs.view(-1, kvh)
    rng = np.random.default_rng(34)
    kind = torch.from_numpy(rng.integers(0, 6, vs.shape)).to(gpu_device)
    vs.copy_(torch.where(kind == 0, -vs, torch.where(kind == 1, torch.zeros_like(vs), vs)))
    vs.copy_(torch.where(kind == 2, vs * 2.0 ** -60, torch.where(kind == 3, vs * -0.0, vs)))
    # a request whose first positions have nothing but zero scales
    first = torch.from_numpy(c.slots(1, np.arange(20))).to(gpu_device)
    vs[first] = 0.0
    q = ref.query(sum(news), hq, d, dtype, gpu_device, seed=35)
    scale = d ** -0.5
    out, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, window, sinks)
    w = torch.zeros(2, kvh, 500, device=gpu_device)
    got = attend(q, *c.args(), lens, news, scale, window=window, sinks=sinks, weights=w)
    ref.check_out(got, out, bound, dtype)
    ref.check_weights(torch.zeros_like(w), w, sums, sum_bounds, [0, 1], lens, news)


@pytest.mark.parametrize("n", [1, 40, 300])
def test_a_value_scale_that_is_no_number_reaches_who_sees_it(gpu_device, n):
    """NaN and infinite scales: nothing finite from the rows that see one."""
    lens = [500]
    for value in (math.nan, math.inf, -math.inf):
        c = ref.Cache(lens, 1, 128, 32, device=gpu_device, seed=36)
        c.vs.view(-1)[int(c.slots(0, np.array([490]))[0])] = value
        q = ref.query(n, 8, 128, BF16, gpu_device, seed=37)
        got = attend(q, *c.args(), lens, [n], 0.1)
        see = torch.arange(500 - n, 500, device=gpu_device) >= 490
        assert not got[see].isfinite().any() and got[~see].isfinite().all()


# ---- numbers past 64 bits --------------------------------------------------------------


@pytest.mark.parametrize("past", [2 ** 31, 2 ** 63, 2 ** 64 + 1])
def test_windows_and_budgets_without_an_end(gpu_device, past):
    """A window, sinks or a budget past every length: everything is seen, or stays."""
    lens, news = [300, 90], [1, 40]
    c = ref.Cache(lens, 2, 64, 16, device=gpu_device, seed=38)
    q = ref.query(sum(news), 4, 64, BF16, gpu_device)
    want = attend(q, *c.args(), lens, news, 0.1)
    assert torch.equal(attend(q, *c.args(), lens, news, 0.1, window=past, sinks=1), want)
    assert torch.equal(attend(q, *c.args(), lens, news, 0.1, window=1, sinks=past), want)
    w = torch.rand(2, 2, 300, device=gpu_device)
    image = [t.clone() for t in (c.k, c.ks, c.v, c.vs, w)]
    for keep in (past, [past, past]):
        new_lens, kept = evict(*c.args(), lens, w, keep, sinks=past, recent=past)
        assert new_lens == lens
        for b, n in enumerate(lens):
            assert torch.equal(kept[b, 0, :n].cpu(), torch.arange(n, dtype=torch.int32))
            assert bool((kept[b, :, n:] == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(image, (c.k, c.ks, c.v, c.vs, w)))
    new_lens, _ = evict(*c.args(), lens, w, [past, 50], sinks=4)
    assert new_lens == [300, 50]


# ---- pages that are gone, NaN in tall tiles, fp32, captured evictions in place --------


@pytest.mark.parametrize("news,hq,kvh,d,bs,dtype", [
    ([70, 9], 8, 2, 128, 32, BF16),   # keys read for many columns
    ([1, 3], 8, 2, 128, 32, FP16),    # from the decode's scores
    ([300, 1], 16, 2, 128, 16, BF16),  # columns in segments
    ([3, 70], 6, 2, 96, 32, BF16),    # any geometry
    ([3, 70], 6, 2, 64, 24, FP32),
])
@pytest.mark.parametrize("sinks", [0, 20])
def test_weights_beside_vanished_pages(gpu_device, news, hq, kvh, d, bs, dtype, sinks):
    """Pages behind the window, gone from the table or given to others that hold NaN,
    reach neither results nor weights."""
    lens, window = [2000, 900], 256
    c = ref.Cache(lens, kvh, d, bs, device=gpu_device, seed=41)
    q = ref.query(sum(news), hq, d, dtype, gpu_device)
    scale = d ** -0.5
    out, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, window, sinks)
    host, live = c.host.copy(), set()
    for b in range(2):
        first = (lens[b] - news[b] - window + 1) // bs
        for i in range(c.host.shape[1]):
            if -(-sinks // bs) <= i < first or i >= -(-lens[b] // bs):
                host[b, i] = (-1, 10 ** 6, 0, c.nb - 1)[i % 4]
            else:
                live.add(int(c.host[b, i]))
    gone = torch.tensor([i for i in range(c.nb) if i not in live], device=gpu_device)
    c.k[gone], c.v[gone] = 0x7F, 0xFF
    c.ks[gone], c.vs[gone] = math.nan, math.nan
    table = torch.from_numpy(host).to(gpu_device, torch.int64)
    before = torch.rand(2, kvh, 2000, device=gpu_device)
    after = before.clone()
    got = attend(q, *c.args()[:4], table, lens, news, scale, window=window, sinks=sinks,
                 weights=before, out_weights=after, block_table_host=host)
    ref.check_out(got, out, bound, dtype)
    ref.check_weights(before, after, sums, sum_bounds, [0, 1], lens, news)


@pytest.mark.parametrize("window,sinks", [(None, 0), (64, 5), (333, 130)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_nan_in_tall_tiles(gpu_device, window, sinks, dtype):
    """256-row tiles at head size 128: NaN keys, values and scales at the edges of
    what their rows see, over more blocks than LDS holds."""
    lens, news, kvh, d = [1100, 700], [333, 290], 2, 128
    c = ref.Cache(lens, kvh, d, 32, device=gpu_device, seed=42)
    k, v = c.k.view(-1, kvh, d), c.v.view(-1, kvh, d)
    ks, vs = c.ks.view(-1, kvh), c.vs.view(-1, kvh)
    for b, length in enumerate(lens):  # stale rows behind the last position
        stale = torch.from_numpy(c.slots(b, np.arange(length, c.host.shape[1] * 32))).to(gpu_device)
        k[stale], v[stale] = 0x7F, 0xFF
        ks[stale], vs[stale] = math.nan, math.inf

    def at(b, p):
        return int(c.slots(b, np.array([p]))[0])

    for p, dim in ((1099, 0), (1000, 77), (868, 127), (800, 31), (3, 5)):
        v[at(0, p), 0, dim] = 0x7F
    vs[at(1, 650), 1] = math.nan
    vs[at(1, 470), 0] = math.inf
    k[at(1, 699), 0, 9] = 0xFF
    ks[at(0, 1050), 1] = math.nan
    q = ref.query(sum(news), 8, d, dtype, gpu_device)
    scale = d ** -0.5
    # (the infinite scale's row of values: none finite, as the other kind of scale)
    out, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, window, sinks)
    vs[at(1, 470), 0] = math.nan
    out = torch.where(out.isnan(), out, ref.attention64(q, c, lens, news, scale, window, sinks)[0])
    vs[at(1, 470), 0] = math.inf
    before = torch.rand(2, kvh, 1100, device=gpu_device)
    after = before.clone()
    got = attend(q, *c.args(), lens, news, scale, window=window, sinks=sinks, weights=before,
                 out_weights=after)
    ref.check_out(got, out, bound, dtype)
    ref.check_weights(before, after, sums, sum_bounds, [0, 1], lens, news)


@pytest.mark.parametrize("hq,kvh,d,bs", [(6, 2, 128, 16), (4, 1, 96, 8), (3, 3, 20, 16)])
def test_fp32_queries_keep_their_bits(gpu_device, hq, kvh, d, bs):
    """A few positions of alike weight, so that probabilities in 16 bits would show.

    Scores and weights as in ``ref.attention64``: a score off by (D + 16) 2^-24 of its
    magnitudes A, a weight relatively by twice that and (length + 200) 2^-24; p times
    the value scale one rounding, the sum over length positions one each, the norm a
    few: (length + 64) 2^-24."""
    lens, news = [5, 3, 7], [2, 3, 1]
    c = ref.Cache(lens, kvh, d, bs, device=gpu_device, seed=43)
    q = ref.query(sum(news), hq, d, FP32, gpu_device, size=0.1)
    scale, rep, row = d ** -0.5, hq // kvh, 0
    got = attend(q, *c.args(), lens, news, scale).double()
    told = False
    for b, (length, n) in enumerate(zip(lens, news)):
        k, v = c.rows(b, length)
        for i in range(n):
            m = length - n + i + 1
            for head in range(hq):
                kk, vv = k[:m, head // rep], v[:m, head // rep]
                x = q[row, head].double()
                p = torch.softmax(kk @ x * scale, 0)
                a = (kk.abs() @ x.abs()).max() * scale
                part = (2 * (d + 16) * a + 2 * length + 264) * 2.0 ** -24
                want, size = p @ vv, p @ vv.abs()
                limit = 2.0 ** -24 * want.abs() + (1 + 2.0 ** -24) * part * size + 2.0 ** -149
                assert bool(((got[row, head] - want).abs() <= limit).all())
                told |= bool(((p.half().double() @ vv - want).abs() > limit).any())
            row += 1
    assert told  # the limit is one that 16 bits break


def test_captured_evictions_in_place(gpu_device):
    """Short and long rows, codes, scales and weights moving within their own pages;
    replays follow what is there."""
    lens, keep = [40000, 900, 300], 500
    c = ref.Cache(lens, 2, 64, 64, device=gpu_device, seed=44)
    w = torch.rand(3, 2, 40000, device=gpu_device)
    parts = (c.k, c.ks, c.v, c.vs, w)
    image = [t.clone() for t in parts]
    kw = dict(sinks=4, recent=50, block_table_host=c.host)
    evict(*c.args(), lens, w, keep, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, kept = evict(*c.args(), lens, w, keep, **kw)
    for seed in range(3):
        new = torch.rand(w.shape, generator=torch.Generator().manual_seed(seed)).to(gpu_device)

        def restore():
            for t, old in zip(parts, image):
                t.copy_(old)
            w.copy_(new)

        restore()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (kept, *parts)]
        restore()
        new_lens, again = evict(*c.args(), lens, w, keep, **kw)
        torch.cuda.synchronize()
        assert new_lens == [500, 500, 300]
        for a, b in zip(got, (again, *parts)):
            assert torch.equal(a, b)
        ids = ref.kept_rows(new[0, 1].cpu().numpy(), lens[0], keep, 4, 50)
        np.testing.assert_array_equal(again[0, 1].cpu().numpy(), ids)


# ---- parts of uneven requests ------------------------------------------------------------


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16), (256, BF16), (96, FP16)])
@pytest.mark.parametrize("long,short,batch", [(1200, 8, 40), (3, 1, 150), (1, 900, 2)])
def test_joined_parts_of_uneven_requests(gpu_device, d, dtype, long, short, batch):
    """One request of many rows beside many of few, all of them or some in parts,
    requests of one part and without rows between them."""
    lens = [2500] + [(1500, 20, 2300)[b % 3] for b in range(batch)] + [3000]
    news = [long] + [(short, 1, 0, short)[b % 4] for b in range(batch)] + [short]
    c = ref.Cache([3000] * 4, 1, d, 16, device=gpu_device, seed=45)
    c.host = np.stack([c.host[b % 4] for b in range(len(lens))])
    c.table = torch.from_numpy(c.host).to(gpu_device, torch.int32)
    c.lens = lens
    q = ref.query(sum(news), 8, d, dtype, gpu_device)
    scale = d ** -0.5
    for window, sinks in ((None, 0), (1700, 3)):
        out, bound, sums, sum_bounds = ref.attention64(q, c, lens, news, scale, window, sinks)
        before = torch.rand(len(lens), 1, 3000, device=gpu_device)
        after = before.clone()
        got = attend(q, *c.args(), lens, news, scale, window=window, sinks=sinks, weights=before,
                     out_weights=after, block_table_host=c.host)
        ref.check_out(got, out, bound, dtype)
        ref.check_weights(before, after, sums, sum_bounds, list(range(len(lens))), lens, news)


# ---- offsets past 32 bits ------------------------------------------------------------------


@pytest.mark.parametrize("d,bs,hq,kvh", [(128, 128, 32, 8), (64, 64, 8, 8), (256, 128, 8, 4),
                                         (96, 128, 8, 8)])
def test_pages_and_weights_past_32_bits(gpu_device, d, bs, hq, kvh):
    """Caches of more than 2^32 bytes a side and 2^31 weights: the last pages and rows
    give what the first ones of a small cache do, bit for bit."""
    lens, news = [900, 300], [1, 70]
    c = ref.Cache(lens, kvh, d, bs, device=gpu_device, seed=46, spare=40)
    pages = (1 << 32) // (bs * kvh * d) + c.nb + 5
    rows, cols = 2 + (1 << 31) // (kvh * 901), 901
    base = pages - c.nb
    big = ref.Cache([1], kvh, d, bs, device=gpu_device)
    for name in ("k", "ks", "v", "vs"):
        small = getattr(c, name)
        t = torch.empty((pages, *small.shape[1:]), dtype=small.dtype, device=gpu_device)
        t[base:] = small
        setattr(big, name, t)
    big.host = c.host + base
    big.table = torch.from_numpy(big.host).to(gpu_device, torch.int32)
    w = torch.rand(2, kvh, cols, device=gpu_device)
    wide = torch.empty((rows, kvh, cols), device=gpu_device)
    at = [rows - 1, rows - 2]
    for b in range(2):
        wide[at[b]] = w[b]
    for window, sinks in ((None, 0), (200, 4)):
        for n in ([1, 70], [3, 1], [300, 0]):
            q = ref.query(sum(n), hq, d, BF16, gpu_device)
            kw = dict(window=window, sinks=sinks)
            want = attend(q, *c.args(), lens, n, 0.1, weights=w, **kw)
            got = attend(q, *big.args(), lens, n, 0.1, weights=wide, weight_rows=at, **kw)
            assert torch.equal(got, want)
            assert all(torch.equal(wide[at[b]], w[b]) for b in range(2))
    free = [i for i in range(c.nb) if i not in set(c.host.reshape(-1).tolist())]
    dst = np.array(free[:2 * -(-100 // bs)], dtype=np.int64).reshape(2, -1)
    for fresh in (True, False):
        for cache, weights, r, off in ((c, w, [0, 1], 0), (big, wide, at, base)):
            kw = dict(out_block_table=torch.from_numpy(dst + off).to(gpu_device, torch.int32),
                      out_weights=weights.clone()) if fresh and off == 0 else {}
            if fresh and off:
                kw = dict(out_block_table=torch.from_numpy(dst + off).to(gpu_device, torch.int32))
            evict(*cache.args(), lens, weights, 100, sinks=4, recent=20, weight_rows=r, **kw)
            if fresh and off:  # (in place, where the small cache's went to a copy)
                for b in range(2):
                    wide[at[b]] = w[b]
        for name in ("k", "ks", "v", "vs"):
            assert torch.equal(getattr(big, name)[base:], getattr(c, name))
    assert all(torch.equal(wide[at[b]], w[b]) for b in range(2))
