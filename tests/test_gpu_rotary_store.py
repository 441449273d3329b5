# SPDX-License-Identifier: Apache-2.0
"""The rotating stores on the GPU, against their definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from tests import _eight_bit as ref
from vllm_ascend_quantized_kv_cache.ops.block8 import block8_store
from vllm_ascend_quantized_kv_cache.ops.fp8_latent import fp8_latent_store
from vllm_ascend_quantized_kv_cache.ops.fp8_ops import fp8_per_token_head_store
from vllm_ascend_quantized_kv_cache.ops.fp8_rotary import fp8_per_token_head_rotary_store

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rows(tokens, hq, kvh, d, dtype, dev, seed, shift=0):
    """Queries, keys and values as views of one projection, `shift` elements off its start."""
    g = torch.Generator().manual_seed(seed)
    wide = (hq + 2 * kvh) * d
    x = torch.randn(tokens, wide, generator=g) * torch.exp(0.5 * torch.randn(wide, generator=g))
    x *= torch.exp(0.5 * torch.randn(tokens, 1, generator=g))
    buf = torch.zeros(tokens * wide + shift + 8, dtype=dtype, device=dev)
    buf[shift:shift + tokens * wide] = x.to(dtype).flatten().to(dev)
    qkv = buf[shift:shift + tokens * wide].view(tokens, hq + 2 * kvh, d)
    return qkv[:, :hq], qkv[:, hq:hq + kvh], qkv[:, hq + kvh:]


def _positions(tokens, limit, seed, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, limit, (tokens,), generator=g).to(dtype).to(dev)


ROTATIONS = [
    # tokens, hq, kvh, d, rot, interleaved, dtype, table, index, shift
    (1, 10, 2, 128, 128, False, BF16, F32, torch.int64, 0),
    (37, 14, 2, 64, 32, True, F16, F32, torch.int32, 0),
    (300, 8, 1, 256, 256, False, BF16, BF16, torch.int64, 0),
    (5, 3, 3, 96, 64, False, F32, F32, torch.int32, 0),
    (19, 4, 2, 128, 128, True, F16, F16, torch.int64, 0),
    (70, 5, 1, 512, 512, False, BF16, F32, torch.int64, 0),
    (1100, 40, 8, 128, 128, False, BF16, F32, torch.int64, 0),  # four heads a thread
    # any geometry: dims off 16, a rotation off 16, rows off 16 bytes
    (33, 6, 2, 20, 20, False, BF16, F32, torch.int64, 0),
    (21, 4, 4, 100, 34, True, F32, F32, torch.int32, 0),
    (17, 2, 1, 128, 72, False, F16, F32, torch.int64, 0),
    (29, 4, 2, 64, 64, False, BF16, F32, torch.int64, 3),
    (9, 2, 1, 508, 254, False, BF16, F32, torch.int64, 0),
]


@pytest.mark.parametrize("tokens,hq,kvh,d,rot,inter,dtype,table,index,shift", ROTATIONS)
def test_token_scales(gpu_device, tokens, hq, kvh, d, rot, inter, dtype, table, index, shift):
    dev = gpu_device
    q, k, v = _rows(tokens, hq, kvh, d, dtype, dev, 1, shift)
    kept = [x.clone() for x in (q, k, v)]
    cos_sin = ref.table(500, rot, table).to(dev)
    positions = _positions(tokens, 500, 2, index, dev)
    bs, pages = 16, tokens // 16 + 3
    slots = torch.randperm(pages * bs, generator=torch.Generator().manual_seed(3))[:tokens]
    slots[::5] = -1
    if tokens > 7:
        slots[7] = pages * bs  # outside the cache
    data = [torch.full((pages, bs, kvh, d), 7, dtype=torch.uint8, device=dev) for _ in range(2)]
    scale = [torch.full((pages, bs, kvh, 1), 3.0, device=dev) for _ in range(2)]
    got = fp8_per_token_head_rotary_store(q, k, v, positions, cos_sin, slots.to(dev, index), data[0],
                                          scale[0], data[1], scale[1], interleaved=inter)
    for x, y in zip((q, k, v), kept):
        assert torch.equal(x, y), "the inputs stay as they are"
    y, amp = ref.rotate(q, cos_sin, positions, inter)
    ref.check_rotated(got, y, amp, "queries")
    live = (slots >= 0) & (slots < pages * bs)
    at, tok = slots[live].to(dev), live.nonzero()[:, 0].to(dev)
    rest = torch.ones(pages * bs, dtype=torch.bool, device=dev)
    rest[at] = False
    for side, (y, amp) in enumerate((ref.rotate(k, cos_sin, positions, inter),
                                     (v.double(), v.double().abs()))):
        y, amp = y[tok], amp[tok]
        s = scale[side].view(-1, kvh, 1)[at].double()
        want = (y.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-6)
        assert ((s - want).abs() <= want * ref.TOP).all()
        codes = data[side].view(-1, kvh, d)
        ref.check_codes(codes[at].view(ref.E4M3).double() * s, s, y, amp, f"side {side}", "e4m3")
        assert (codes[rest] == 7).all() and (scale[side].view(-1, kvh)[rest] == 3.0).all()


def test_token_scales_are_the_stores(gpu_device):
    """Values, which are not rotated, and keys at angle 0: bit for bit the store without it."""
    dev = gpu_device
    q, k, v = _rows(200, 4, 2, 128, BF16, dev, 5)
    slots = torch.randperm(256)[:200].to(dev)
    out = []
    for rotate in (False, True):
        data = [torch.zeros(16, 16, 2, 128, dtype=torch.uint8, device=dev) for _ in range(2)]
        scale = [torch.zeros(16, 16, 2, 1, device=dev) for _ in range(2)]
        if rotate:
            still = torch.cat([torch.ones(1, 64), torch.zeros(1, 64)], 1).to(dev)
            zero = torch.zeros(200, dtype=torch.int64, device=dev)
            same = fp8_per_token_head_rotary_store(q, k, v, zero, still, slots, data[0], scale[0],
                                                   data[1], scale[1])
            assert torch.equal(same, q)
        else:
            fp8_per_token_head_store(k, v, slots, data[0], scale[0], data[1], scale[1])
        out.append([*data, *scale])
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("where", ["self", "own", "strided", "inside"])
def test_out_query(gpu_device, where):
    dev = gpu_device
    q, k, v = _rows(23, 6, 2, 64, BF16, dev, 6)
    cos_sin = ref.table(50, 64).to(dev)
    positions = _positions(23, 50, 7, torch.int64, dev)
    y, amp = ref.rotate(q, cos_sin, positions, False)
    data = [torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device=dev) for _ in range(2)]
    scale = [torch.zeros(4, 16, 2, 1, device=dev) for _ in range(2)]
    out = {"self": lambda: q, "own": lambda: torch.empty(23, 6, 64, dtype=BF16, device=dev),
           "strided": lambda: torch.empty(23, 64, 6, dtype=BF16, device=dev).transpose(1, 2),
           # memory of the projection, but not the queries': behind them
           "inside": lambda: q.as_strided(q.shape, q.stride(), q.storage_offset() + 64)}[where]()
    ky, _ = ref.rotate(k, cos_sin, positions, False)
    got = fp8_per_token_head_rotary_store(q, k, v, positions, cos_sin, torch.arange(23, device=dev),
                                          data[0], scale[0], data[1], scale[1], out_query=out)
    assert got is out
    ref.check_rotated(got, y, amp, "queries")
    back = data[0].view(-1, 2, 64)[:23].view(ref.E4M3).double() * scale[0].view(-1, 2, 1)[:23].double()
    assert ((back - ky).abs() <= ky.abs() * 2.0 ** -4 + ky.abs().amax(-1, keepdim=True) * 2.0 ** -8).all()


def test_positions_outside_the_table(gpu_device):
    dev = gpu_device
    q, k, v = _rows(4, 2, 1, 64, BF16, dev, 8)
    cos_sin = ref.table(10, 32).to(dev)
    positions = torch.tensor([3, 10, -1, 9], device=dev)
    data = [torch.full((1, 16, 1, 64), 9, dtype=torch.uint8, device=dev) for _ in range(2)]
    scale = [torch.full((1, 16, 1, 1), 2.0, device=dev) for _ in range(2)]
    got = fp8_per_token_head_rotary_store(q, k, v, positions, cos_sin, torch.arange(4, device=dev),
                                          data[0], scale[0], data[1], scale[1])
    bad = torch.tensor([1, 2], device=dev)
    assert torch.isnan(got[bad, :, :32]).all() and torch.equal(got[bad, :, 32:], q[bad, :, 32:])
    assert not torch.isnan(got[[0, 3]]).any()
    for side in (0, 1):
        assert (data[side][0, bad] == 9).all() and (scale[side][0, bad] == 2.0).all()
        assert (scale[side][0, [0, 3]] != 2.0).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_rows_that_are_not_finite(gpu_device, value):
    dev = gpu_device
    _, k, v = _rows(20, 1, 2, 64, BF16, dev, 9)
    k = k.clone()
    k[3, 1, 40] = value
    data = [torch.zeros(2, 16, 2, 64, dtype=torch.uint8, device=dev) for _ in range(2)]
    scale = [torch.zeros(2, 16, 2, 1, device=dev) for _ in range(2)]
    fp8_per_token_head_rotary_store(None, k, v, torch.arange(20, device=dev), ref.table(20, 64).to(dev),
                                    torch.arange(20, device=dev), data[0], scale[0], data[1], scale[1])
    back = data[0].view(ref.E4M3).float() * scale[0]
    bad = torch.isnan(back).view(32, 2, 64)
    assert bad[3, 1].all() and not bad[:3].any() and not bad[4:].any() and not bad[3, 0].any()
    c = ref.BlockCache(2, 16, 2, 64, 16, "int8", dev)
    block8_store(k, v, torch.arange(20, device=dev), *c.args())
    bad = ~torch.isfinite(c.data[0].float() * c.scale[0].view(2, 1, 2, 1))
    assert bad[0, 3, 1].any() and not bad[1].any() and not bad[0, :, 0].any()


BLOCKS = [
    # (before, new) of requests, pad, hq, kvh, d, bs, group, rot, inter, dtype, codes, shift
    ([(600, 1)], 0, 10, 2, 128, 128, 128, 128, False, BF16, "int8", 0),
    ([(0, 1), (127, 1), (128, 1), (5, 1), (255, 1)], 3, 4, 8, 128, 128, 128, 128, False, BF16, "e4m3", 0),
    ([(0, 300), (70, 129), (128, 128), (1, 2)], 0, 4, 2, 128, 128, 128, 128, False, BF16, "e4m3", 0),
    ([(0, 300), (70, 129), (128, 128), (1, 2)], 5, 4, 2, 64, 64, 16, 32, True, F16, "int8", 0),
    ([(3, 200), (130, 5)], 0, 2, 1, 256, 128, 64, 256, False, BF16, "int8", 0),
    ([(3, 200), (130, 7)], 0, 2, 1, 512, 128, 128, 512, False, F32, "e4m3", 0),  # rows read twice
    ([(i % 17, 1 + i % 3) for i in range(700)], 0, 2, 1, 64, 16, 16, 64, False, BF16, "e4m3", 0),
    ([(0, 1500), (9, 100)], 0, 4, 2, 64, 32, 32, 64, False, BF16, "int8", 0),
    # any geometry
    ([(2, 50), (30, 4)], 2, 3, 3, 20, 24, 12, 20, False, BF16, "int8", 0),
    ([(2, 50), (30, 4)], 2, 3, 1, 100, 18, 6, 34, True, F32, "e4m3", 0),
    ([(2, 50), (30, 4)], 0, 4, 2, 64, 32, 32, 64, False, F16, "e4m3", 5),
    ([(0, 20)], 0, 0, 2, 64, 16, 1, 64, False, BF16, "e4m3", 0),  # a scale for each token
]


@pytest.mark.parametrize("requests,pad,hq,kvh,d,bs,group,rot,inter,dtype,codes,shift", BLOCKS)
def test_block_scales(gpu_device, requests, pad, hq, kvh, d, bs, group, rot, inter, dtype, codes,
                      shift):
    dev = gpu_device
    host, pages = ref.paged([a + n for a, n in requests], bs)
    slots, positions = [], []
    for b, (a, n) in enumerate(requests):
        positions += range(a, a + n)
        slots += ref.slots_of(host, b, range(a, a + n), bs).tolist()
    if pad:  # behind the batch and inside a block's rows
        slots[3:3] = [-1] * pad
        positions[3:3] = [0] * pad
        slots += [pages * bs] * pad
        positions += [0] * pad
    tokens = len(slots)
    q, k, v = _rows(tokens, hq, kvh, d, dtype, dev, 11, shift)
    cos_sin = ref.table(max(positions) + 1, rot).to(dev)
    positions = torch.tensor(positions, device=dev)
    before = ref.BlockCache(pages, bs, kvh, d, group, codes, dev)
    after = before.clone()
    got = block8_store(k, v, torch.tensor(slots, device=dev), *after.args(), query=q if hq else None,
                       positions=positions, cos_sin=cos_sin, interleaved=inter)
    if hq:
        y, amp = ref.rotate(q, cos_sin, positions, inter)
        ref.check_rotated(got, y, amp, "queries")
    else:
        assert got is None
    rows = [ref.rotate(k, cos_sin, positions, inter), (v.double(), v.double().abs())]
    ref.check_block_store(before, after, rows, slots, [0 <= s < pages * bs for s in slots])


@pytest.mark.parametrize("gaps", [(3, 200, 700), (0, 40, 1300), (1000, 70, 2500)])
def test_block_scales_among_padding(gpu_device, gaps):
    """Runs of a block whose rows lie far apart in the call, past a workgroup's tokens."""
    dev = gpu_device
    d, kvh, bs, group = 64, 1, 32, 32
    slots = []
    for i in range(9):  # two and a half blocks, cut by padding wherever it falls
        slots += [-1] * gaps[i % 3] + list(range(100 + 9 * i, 100 + 9 * (i + 1)))
    slots += [-1] * gaps[0]
    tokens = len(slots)
    _, k, v = _rows(tokens, 1, kvh, d, BF16, dev, 17)
    before = ref.BlockCache(8, bs, kvh, d, group, "int8", dev)
    after = before.clone()
    block8_store(k, v, torch.tensor(slots, device=dev), *after.args())
    rows = [(x.double(), x.double().abs()) for x in (k, v)]
    ref.check_block_store(before, after, rows, slots, [x >= 0 for x in slots])


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("steps", [[1] * 40, [16, 1, 30, 2, 100], [7, 70, 3]])
def test_a_block_in_several_calls(gpu_device, codes, steps):
    """Rows of growing size: each call's scale and requantized rows follow from the last."""
    dev = gpu_device
    d, kvh, bs, group = 64, 2, 64, 32
    total = sum(steps)
    host, pages = ref.paged([total], bs)
    _, k, v = _rows(total, 1, kvh, d, BF16, dev, 12)
    grow = torch.exp(torch.arange(total, device=dev) * 0.05)[:, None, None]
    k, v = (k * grow).to(BF16), (v * grow).to(BF16)
    cos_sin = ref.table(total, d).to(dev)
    cache = ref.BlockCache(pages, bs, kvh, d, group, codes, dev)
    at = 0
    for n in steps:
        slots = ref.slots_of(host, 0, range(at, at + n), bs).tolist()
        positions = torch.arange(at, at + n, device=dev)
        before = cache.clone()
        block8_store(k[at:at + n], v[at:at + n], torch.tensor(slots, device=dev, dtype=torch.int32),
                     *cache.args(), positions=positions, cos_sin=cos_sin)
        rows = [ref.rotate(k[at:at + n], cos_sin, positions, False),
                (v[at:at + n].double(), v[at:at + n].double().abs())]
        ref.check_block_store(before, cache, rows, slots, [True] * n)
        at += n


def test_block_store_without_rotation(gpu_device):
    dev = gpu_device
    _, k, v = _rows(50, 1, 2, 64, F16, dev, 13)
    before = ref.BlockCache(4, 16, 2, 64, 16, "int8", dev)
    after = before.clone()
    slots = list(range(5, 55))
    assert block8_store(k, v, torch.tensor(slots, device=dev), *after.args()) is None
    rows = [(x.double(), x.double().abs()) for x in (k, v)]
    ref.check_block_store(before, after, rows, slots, [True] * 50)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_empty_and_tiny_rows(gpu_device, codes):
    """Rows of zeros take the least scale; amounts at the edge of a scale stay in range."""
    dev = gpu_device
    edge = 448.0 if codes == "e4m3" else 127.0
    x = torch.zeros(6, 1, 64, device=dev)
    x[1, 0, 3], x[2, 0, 3], x[3, 0, 3] = edge, edge * (1 + 2.0 ** -23), edge * (1 - 2.0 ** -24)
    x[4, 0, 3], x[5, 0, 3] = 1e-30, -3e38
    before = ref.BlockCache(6, 16, 1, 64, 16, codes, dev)
    after = before.clone()
    slots = [16 * i for i in range(6)]
    block8_store(x, x, torch.tensor(slots, device=dev), *after.args())
    ref.check_block_store(before, after, [(x.double(), x.double().abs())] * 2, slots, [True] * 6)
    if codes == "e4m3":
        assert after.scale[0][:, 0, 0].tolist()[:5] == [2.0 ** -20, 1.0, 2.0, 1.0, 2.0 ** -20]


LATENTS = [
    # tokens, heads, rank, part, interleaved, dtype, shift
    (1, 16, 512, 64, True, BF16, 0),
    (64, 16, 512, 64, True, BF16, 0),
    (333, 128, 512, 64, False, F16, 0),
    (41, 8, 256, 32, True, F32, 0),
    (13, 0, 512, 64, True, BF16, 0),
    (27, 3, 100, 10, True, BF16, 0),
    (27, 3, 512, 64, False, BF16, 1),
]


@pytest.mark.parametrize("tokens,heads,rank,dims,inter,dtype,shift", LATENTS)
def test_latent_store(gpu_device, tokens, heads, rank, dims, inter, dtype, shift):
    dev = gpu_device
    g = torch.Generator().manual_seed(14)
    wide = rank + dims
    buf = torch.randn(tokens * wide + shift, generator=g).to(dtype).to(dev)
    down = buf[shift:].view(tokens, wide)
    latent, part = down[:, :rank], down[:, rank:]
    q = torch.randn(tokens, max(heads, 1), 24 + dims, generator=g).to(dtype).to(dev)[..., 24:]
    cos_sin = ref.table(200, dims).to(dev)
    positions = _positions(tokens, 200, 15, torch.int64, dev)
    bs, pages = 16, tokens // 16 + 2
    slots = torch.randperm(pages * bs, generator=g)[:tokens]
    slots[1::4] = -1
    data = torch.full((pages, bs, rank), 5, dtype=torch.uint8, device=dev)
    scale = torch.full((pages, bs, 1), 3.0, device=dev)
    rope = torch.full((pages, bs, dims), 4.0, dtype=dtype, device=dev)
    # the rotated parts land behind the absorbed dims
    full = torch.zeros(tokens, max(heads, 1), wide, dtype=dtype, device=dev)
    got = fp8_latent_store(latent, part, positions, cos_sin, slots.to(dev), data, scale, rope,
                           query=q if heads else None, interleaved=inter,
                           out_query=full[..., rank:] if heads else None)
    if heads:
        y, amp = ref.rotate(q, cos_sin, positions, inter)
        ref.check_rotated(full[..., rank:], y, amp, "queries")
        assert (full[..., :rank] == 0).all()
    else:
        assert got is None
    live = slots >= 0
    at, tok = slots[live].to(dev), live.nonzero()[:, 0].to(dev)
    rest = torch.ones(pages * bs, dtype=torch.bool, device=dev)
    rest[at] = False
    x = latent[tok].double()
    s = scale.view(-1, 1)[at].double()
    want = (x.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-6)
    assert ((s - want).abs() <= want * ref.TOP).all()
    ref.check_codes(data.view(-1, rank)[at].view(ref.E4M3).double() * s, s, x, x.abs(), "latent", "e4m3")
    y, amp = ref.rotate(part[:, None], cos_sin, positions, inter)
    ref.check_rotated(rope.view(-1, dims)[at], y[tok, 0], amp[tok, 0], "position part")
    assert (data.view(-1, rank)[rest] == 5).all() and (scale.view(-1)[rest] == 3.0).all()
    assert (rope.view(-1, dims)[rest] == 4.0).all()


def test_latent_out_query(gpu_device):
    """Heads first, in place, rows of two tensors' memory; rows that share elements are refused."""
    dev, tokens, heads, dims = gpu_device, 6, 3, 16
    g = torch.Generator().manual_seed(18)
    latent, part, q = (torch.randn(shape, generator=g).to(BF16).to(dev) for shape in (
        (tokens, 32), (tokens, dims), (tokens, heads, dims)))
    cache = (torch.zeros(1, 16, 32, dtype=torch.uint8, device=dev), torch.zeros(1, 16, 1, device=dev),
             torch.zeros(1, 16, dims, dtype=BF16, device=dev))
    at = torch.arange(tokens, device=dev)
    args = (latent, part, at, ref.table(tokens, dims).to(dev), at, *cache)
    want = fp8_latent_store(*args, query=q)
    first = torch.zeros(heads, tokens, dims, dtype=BF16, device=dev).transpose(0, 1)
    assert fp8_latent_store(*args, query=q, out_query=first) is first and torch.equal(first, want)
    shared = torch.zeros(tokens, 1, dims, dtype=BF16, device=dev).expand(tokens, heads, dims)
    with pytest.raises(RuntimeError):
        fp8_latent_store(*args, query=q, out_query=shared)
    buf = torch.zeros(tokens, heads, dims + 8, dtype=BF16, device=dev)
    buf[..., :dims] = q
    fp8_latent_store(*args, query=buf[..., :dims], out_query=buf[..., 8:])
    assert torch.equal(buf[..., 8:], want)
    assert fp8_latent_store(*args, query=q, out_query=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("which", ["token", "block", "latent"])
def test_captured_and_replayed(gpu_device, which):
    """The slots and positions are the device's: a replay takes what they hold then."""
    dev = gpu_device
    bs, d, kvh, tokens = 16, 64, 2, 6
    q, k, v = _rows(tokens, 4, kvh, d, BF16, dev, 16)
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=dev)
    positions = torch.zeros(tokens, dtype=torch.int64, device=dev)
    cos_sin = ref.table(64, d).to(dev)
    out = torch.empty(tokens, 4, d, dtype=BF16, device=dev)

    def make():
        if which == "latent":
            return [torch.zeros(8, bs, 128, dtype=torch.uint8, device=dev),
                    torch.zeros(8, bs, 1, device=dev), torch.zeros(8, bs, d, dtype=BF16, device=dev)]
        if which == "token":
            return [x for _ in range(2) for x in (
                torch.zeros(8, bs, kvh, d, dtype=torch.uint8, device=dev),
                torch.zeros(8, bs, kvh, 1, device=dev))]
        return list(ref.BlockCache(8, bs, kvh, d, 16, "int8", dev).args())

    def call(cache, into):
        if which == "latent":
            fp8_latent_store(v.reshape(tokens, 128), k[:, 0], positions, cos_sin, slots, *cache,
                             query=q, out_query=into)
        elif which == "token":
            fp8_per_token_head_rotary_store(q, k, v, positions, cos_sin, slots, *cache, out_query=into)
        else:
            block8_store(k, v, slots, *cache, query=q, positions=positions, cos_sin=cos_sin,
                         out_query=into)

    cache, eager = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(cache, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(cache, out)
    for step in range(4):
        slots.copy_(torch.arange(tokens) * bs + step)
        positions.fill_(step)
        graph.replay()
        want = torch.empty_like(out)
        call(eager, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(cache, eager):
            assert torch.equal(a, b), step


def test_on_another_stream(gpu_device):
    dev = gpu_device
    q, k, v = _rows(400, 8, 2, 128, BF16, dev, 17)
    cos_sin, positions = ref.table(400, 128).to(dev), torch.arange(400, device=dev)
    side = torch.cuda.Stream()
    caches = [ref.BlockCache(4, 128, 2, 128, 128, "e4m3", dev) for _ in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    a = block8_store(k, v, positions, *caches[0].args(), query=q, positions=positions, cos_sin=cos_sin)
    with torch.cuda.stream(side):
        b = block8_store(k, v, positions, *caches[1].args(), query=q, positions=positions,
                         cos_sin=cos_sin)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    for x, y in zip(caches[0].args(), caches[1].args()):
        assert torch.equal(x, y)


def test_no_tokens(gpu_device):
    dev = gpu_device
    c = ref.BlockCache(2, 16, 2, 64, 16, "e4m3", dev)
    q = torch.zeros(0, 4, 64, dtype=BF16, device=dev)
    kv = torch.zeros(0, 2, 64, dtype=BF16, device=dev)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    got = block8_store(kv, kv, none, *c.args(), query=q, positions=none,
                       cos_sin=ref.table(4, 64).to(dev))
    assert got.shape == (0, 4, 64)
