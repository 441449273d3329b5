# SPDX-License-Identifier: Apache-2.0
"""Attention over paged latent rows, on the GPU against a 64-bit restatement, and a serving
loop of store and attention."""

from __future__ import annotations

import pytest
import torch

from tests import _eight_bit as ref
from tests import _fp8_window as win
from vllm_ascend_quantized_kv_cache.ops.fp8_latent import fp8_latent_attention, fp8_latent_store

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SCALE = 192 ** -0.5


def _check(device, lens, news, heads, rank, dims, bs, dtype, *, seed=0, index=torch.int32,
           cache=None, q=None, host=True, size=0.5):
    c = cache or ref.Latents(lens, rank, dims, bs, dtype, device=device, seed=seed, index=index)
    if q is None:
        q = win.query(sum(news), heads, rank + dims, dtype, device, seed=seed + 1, size=size)
    want, bound = ref.latent64(q, c, lens, news, SCALE)
    got = fp8_latent_attention(q, *c.args(), lens, news, SCALE,
                               block_table_host=c.host if host else None)
    win.check_out(got, want, bound, dtype)
    return got


LENGTHS = [
    ([1], [1]), ([2], [1]), ([15], [1]), ([16], [1]), ([17], [1]), ([127], [1]), ([128], [1]),
    ([129], [1]), ([600], [1]),
    ([7, 1, 130, 0, 257, 64], [7, 1, 2, 0, 100, 0]),
    ([300, 17, 1000], [300, 17, 1]),
    # more rows than history: the first ones see nothing
    ([5, 0, 40], [9, 3, 1]),
    ([1500], [333]),
]


@pytest.mark.parametrize("heads", [3, 16, 40])
@pytest.mark.parametrize("lens,news", LENGTHS)
def test_lengths(gpu_device, lens, news, heads):
    _check(gpu_device, lens, news, heads, 512, 64, 32, BF16)


@pytest.mark.parametrize("heads,rank,dims,bs", [
    (1, 512, 64, 16), (16, 512, 64, 128), (32, 512, 64, 64), (128, 512, 64, 128), (17, 512, 32, 48),
    (8, 256, 64, 16), (16, 256, 32, 64), (64, 256, 64, 32),
    # what the matrix kernel leaves to the general one
    (4, 128, 64, 16), (3, 100, 10, 8), (2, 512, 64, 24), (5, 512, 128, 16), (1, 4, 2, 1),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_layouts(gpu_device, heads, rank, dims, bs, dtype):
    lens, news = [200, 71, 33], [1, 71, 6]
    _check(gpu_device, lens, news, heads, rank, dims, bs, dtype, seed=3)
    _check(gpu_device, lens, [1, 1, 1], heads, rank, dims, bs, dtype, seed=4, index=torch.int64,
           host=False)


def test_fp32_queries(gpu_device):
    _check(gpu_device, [150, 40], [20, 1], 6, 512, 64, 16, FP32)
    _check(gpu_device, [5003, 40], [2, 1], 6, 256, 32, 16, FP32)


@pytest.mark.parametrize("news", [[1] * 3, [2, 1, 2], [300, 64, 1]])
@pytest.mark.parametrize("heads", [8, 16, 64])
def test_long_histories(gpu_device, news, heads):
    _check(gpu_device, [9000, 5003, 2048], news, heads, 512, 64, 128, BF16)


@pytest.mark.parametrize("batch,heads", [(1, 16), (100, 16), (130, 33)])
def test_batches(gpu_device, batch, heads):
    """More requests than a launch takes; parts of some."""
    lens = [(37 * b) % 700 + 1 for b in range(batch)] + [9000]
    news = [1 + b % 2 for b in range(batch)] + [1]
    _check(gpu_device, lens, news, heads, 256, 64, 16, FP16)


@pytest.mark.parametrize("news", [[1, 1], [70, 3]])
def test_scales_of_any_sign_and_size(gpu_device, news):
    lens = [400, 90]
    for dtype in (FP32, BF16):
        c = ref.Latents(lens, 512, 64, 32, dtype, device=gpu_device, seed=8)
        g = torch.Generator().manual_seed(9)
        sign = (torch.rand(c.scale.shape, generator=g) < 0.5).float() * 2 - 1
        spread = torch.exp2(torch.randint(-60, 3, c.scale.shape, generator=g).float())
        c.scale *= (sign * spread).to(gpu_device)
        _check(gpu_device, lens, news, 8, 512, 64, 32, dtype, cache=c)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 0.0])
@pytest.mark.parametrize("news", [[1, 2], [40, 3]])
def test_odd_scales(gpu_device, value, news):
    lens = [300, 60]
    c = ref.Latents(lens, 512, 64, 16, BF16, device=gpu_device, seed=10)
    at = int(ref.slots_of(c.host, 0, [280], 16)[0])
    c.scale.view(-1)[at] = 0.0
    q = win.query(sum(news), 4, 576, BF16, gpu_device, size=0.5)
    want, bound = ref.latent64(q, c, lens, news, SCALE)
    c.scale.view(-1)[at] = value
    got = fp8_latent_attention(q, *c.args(), lens, news, SCALE, block_table_host=c.host)
    sees = torch.zeros(sum(news), dtype=torch.bool, device=gpu_device)
    if value != 0.0:
        for i in range(news[0]):
            sees[i] = 300 - news[0] + i >= 280
        assert not torch.isfinite(got[sees]).any()
    win.check_out(got[~sees], want[~sees], bound[~sees], BF16)


@pytest.mark.parametrize("heads", [4, 32])
@pytest.mark.parametrize("news", [[1, 1], [40, 3]])
def test_nan_codes_and_parts(gpu_device, news, heads):
    """A position that holds a NaN spoils the rows that see it and no others."""
    lens = [300, 60]
    c = ref.Latents(lens, 512, 64, 16, BF16, device=gpu_device, seed=11)
    c.data.view(-1, 512)[int(ref.slots_of(c.host, 0, [270], 16)[0]), 77] = 0xff
    c.data.view(-1, 512)[int(ref.slots_of(c.host, 0, [290], 16)[0]), 500] = 0x7f
    c.rope.view(-1, 64)[int(ref.slots_of(c.host, 1, [58], 16)[0]), 3] = float("nan")
    _check(gpu_device, lens, news, heads, 512, 64, 16, BF16, cache=c)


@pytest.mark.parametrize("news", [1, 40])
def test_stale_rows(gpu_device, news):
    """What lies behind a request's rows has no part in it."""
    c = ref.Latents([301], 512, 64, 16, BF16, device=gpu_device, seed=12)
    want = _check(gpu_device, [301], [news], 16, 512, 64, 16, BF16, cache=c)
    last = int(ref.slots_of(c.host, 0, [300], 16)[0])
    behind = slice(last + 1, last // 16 * 16 + 16)
    c.data.view(-1, 512)[behind] = 0x7f
    c.scale.view(-1)[behind] = float("nan")
    c.rope.view(-1, 64)[behind] = float("inf")
    q = win.query(news, 16, 576, BF16, gpu_device, seed=1, size=0.5)
    got = fp8_latent_attention(q, *c.args(), [301], [news], SCALE, block_table_host=c.host)
    assert torch.equal(got, want)


def test_large_scores(gpu_device):
    for news in (1, 90):
        _check(gpu_device, [700], [news], 8, 512, 64, 64, FP16, size=12.0)


@pytest.mark.parametrize("heads", [4, 32, 33, 64, 65, 96])
@pytest.mark.parametrize("growth", [2.0 ** 0.1, 2.0 ** -0.1, 64.0])
def test_scores_that_grow(gpu_device, heads, growth):
    """Maxima that outgrow the offsets again and again, or stay the first ones, by rows that
    get larger or smaller from position to position."""
    lens, news = [500, 129], [1, 2]
    for rank, dims in ((512, 64), (256, 32)):
        c = ref.Latents(lens, rank, dims, 64, BF16, device=gpu_device, seed=14)
        for b, n in enumerate(lens):
            at = torch.from_numpy(ref.slots_of(c.host, b, torch.arange(n).numpy(), 64))
            steps = torch.arange(n) // 48 if growth == 64.0 else torch.arange(n) % 300
            size = torch.exp2(torch.log2(torch.tensor(growth)) * steps).clamp(2.0 ** -40, 2.0 ** 40)
            c.scale.view(-1)[at.to(gpu_device)] = (2.0 ** -6 * size).to(gpu_device)
        _check(gpu_device, lens, news, heads, rank, dims, 64, BF16, cache=c, size=0.1)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_few_and_many_columns(gpu_device, dtype):
    """Requests of both kernels in one call, between those without rows."""
    lens, news = [70, 2000, 0, 300, 900, 64, 5], [1, 3, 0, 2, 40, 0, 1]
    _check(gpu_device, lens, news, 16, 512, 64, 16, dtype, seed=15)


@pytest.mark.parametrize("shift", [1, 8])
def test_rows_off_their_bounds(gpu_device, shift):
    lens, news = [130, 20], [9, 1]
    c = ref.Latents(lens, 512, 64, 16, BF16, device=gpu_device, seed=16)
    q = win.query(10, 4, 576, BF16, gpu_device, size=0.5)
    buf = torch.zeros(10 * 3000 + shift, dtype=BF16, device=gpu_device)
    apart = buf[shift:].view(10, 3000)[:, :2304].view(10, 4, 576)
    apart.copy_(q)
    want = _check(gpu_device, lens, news, 4, 512, 64, 16, BF16, cache=c, q=q)
    out = torch.zeros(10 * 2048 + shift, dtype=BF16, device=gpu_device)[shift:].view(10, 4, 512)
    got = fp8_latent_attention(apart, *c.args(), lens, news, SCALE, out=out, block_table_host=c.host)
    assert got is out and torch.equal(out, want)
    x = torch.zeros(c.data.numel() + 16, dtype=torch.uint8, device=gpu_device)
    x[4:4 + c.data.numel()] = c.data.flatten()
    c.data = x[4:4 + c.data.numel()].view(c.data.shape)  # 4-byte bounds: the general kernel
    _check(gpu_device, lens, news, 4, 512, 64, 16, BF16, cache=c, q=q)


def test_padded_batch_and_out(gpu_device):
    lens, news = [90, 40], [2, 1]
    c = ref.Latents(lens, 256, 64, 16, BF16, device=gpu_device, seed=17)
    q = win.query(7, 4, 320, BF16, gpu_device, size=0.5)
    want, bound = ref.latent64(q[:3], c, lens, news, SCALE)
    got = fp8_latent_attention(q, *c.args(), lens, news, SCALE)
    win.check_out(got[:3], want, bound, BF16)
    assert (got[3:] == 0).all()
    for out in (torch.full((7, 4, 256), 5.0, dtype=BF16, device=gpu_device),
                torch.full((7, 256, 4), 5.0, dtype=BF16, device=gpu_device).transpose(1, 2),
                torch.full((7, 4, 256), 5.0, dtype=FP32, device=gpu_device)):
        back = fp8_latent_attention(q, *c.args(), lens, news, SCALE, out=out)
        assert back is out and (out[3:] == 5.0).all()
        assert torch.equal(out[:3].to(BF16), got[:3])
    own = q.clone()
    part = own[..., :256]
    assert torch.equal(fp8_latent_attention(own, *c.args(), lens, news, SCALE, out=part)[:3], got[:3])
    assert fp8_latent_attention(q[:0], *c.args(), [], [], SCALE).shape == (0, 4, 256)
    assert (fp8_latent_attention(q, *c.args(), lens, [0, 0], SCALE) == 0).all()


@pytest.mark.parametrize("news", [[1, 1], [50, 1]])
def test_streams_and_graphs(gpu_device, news):
    lens = [2000, 700]
    c = ref.Latents(lens, 512, 64, 128, BF16, device=gpu_device, seed=18)
    q = win.query(sum(news), 16, 576, BF16, gpu_device, size=0.5)
    want = _check(gpu_device, lens, news, 16, 512, 64, 128, BF16, cache=c, q=q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp8_latent_attention(q, *c.args(), lens, news, SCALE, block_table_host=c.host)
    also = fp8_latent_attention(q, *c.args(), lens, news, SCALE, block_table_host=c.host)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(also, want)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of one pool
        out = torch.zeros_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            fp8_latent_attention(q, *c.args(), lens, news, SCALE, out=out, block_table_host=c.host)
        graphs.append(graph)
        outs.append(out)
    for i in range(3):
        q.copy_(win.query(sum(news), 16, 576, BF16, gpu_device, seed=50 + i, size=0.5))
        for out in outs:
            out.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        want = fp8_latent_attention(q, *c.args(), lens, news, SCALE, block_table_host=c.host)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_a_serving_loop(gpu_device):
    """Prompts, then tokens: each step rotates, stores and attends."""
    dev, heads, rank, dims, bs = gpu_device, 16, 512, 64, 16
    prompts, steps = [150, 37, 1], 20
    lens = [n + steps for n in prompts]
    c = ref.Latents(lens, rank, dims, bs, BF16, device=dev, seed=20)
    cos_sin = ref.table(max(lens), dims).to(dev)
    g = torch.Generator().manual_seed(21)
    at = [0] * len(prompts)
    for step in range(steps + 1):
        news = prompts if step == 0 else [1] * len(prompts)
        rows = sum(news)
        down = torch.randn(rows, rank + dims, generator=g).to(BF16).to(dev)
        q = (0.5 * torch.randn(rows, heads, rank + dims, generator=g)).to(BF16).to(dev)
        positions = [p for a, n in zip(at, news) for p in range(a, a + n)]
        slots = [s for b, (a, n) in enumerate(zip(at, news))
                 for s in ref.slots_of(c.host, b, range(a, a + n), bs).tolist()]
        at = [a + n for a, n in zip(at, news)]
        turned = q[..., rank:]
        fp8_latent_store(down[:, :rank], down[:, rank:], torch.tensor(positions, device=dev), cos_sin,
                         torch.tensor(slots, device=dev), c.data, c.scale, c.rope, query=turned,
                         interleaved=True, out_query=turned)
        if step % 10 == 0:
            _check(dev, at, news, heads, rank, dims, bs, BF16, cache=c, q=q)
