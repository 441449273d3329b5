# SPDX-License-Identifier: Apache-2.0
"""Serving loops over the cache with block scales and the latent cache, held against the rows
that went in: prompts, then tokens, some of them speculated and taken back.

A row is off by what its quantization rounds, and by every later growth of its block's scale:
half a step of INT8 codes at each new scale, and of E4M3 codes what becomes subnormal (half of
2^-9 of the new scale).  The scales follow from the rows by the definition, in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import _eight_bit as ref
from tests import _fp8_window as win
from vllm_ascend_quantized_kv_cache.ops.block8 import block8_attention, block8_store
from vllm_ascend_quantized_kv_cache.ops.fp8_latent import fp8_latent_attention, fp8_latent_store

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


class Side:
    """One side (keys or values) of one cache, followed row by row: what went in, and how far
    what is there may be off."""

    def __init__(self, cache, slots):
        self.cache, shape = cache, (slots, cache.kvh, cache.d)
        self.row, self.off = torch.zeros(shape).double(), torch.zeros(shape).double()
        self.scale = torch.zeros(slots // cache.group, cache.kvh).double()
        self.growths = 0

    def store(self, slots, y, amp, scale_after):
        """Rows y at slots; the scales that the cache has behind it, [blocks, heads]."""
        c, g = self.cache, self.cache.group
        blocks = slots // g
        for block in dict.fromkeys(blocks.tolist()):
            at = torch.from_numpy(np.flatnonzero(blocks == block))
            first = int(slots[blocks == block].min()) - block * g
            for h in range(c.kvh):
                top = y[at, h].abs().max().item()
                was = self.scale[block, h].item() if first else 0.0
                want = {max(ref.block_scale(top * f, c.codes), was) for f in (1 - ref.TOP, 1 + ref.TOP)}
                got = scale_after[block, h].item()
                assert any(abs(got - w) <= w * ref.TOP for w in want), (block, h, got, want)
                there = slice(block * g, block * g + first)
                if first and got != was:
                    self.growths += 1
                    self.off[there, h] += got * (2.0 ** -10 if c.codes == "e4m3" else 0.5 + 2.0 ** -14)
                self.scale[block, h] = got
                at_slot = torch.from_numpy(slots)[at]
                if c.codes == "e4m3":
                    half = torch.clamp(y[at, h].abs() * 2.0 ** -4, min=got * 2.0 ** -10)
                else:
                    half = torch.full_like(y[at, h], got * 0.5)
                self.row[at_slot, h] = y[at, h]
                self.off[at_slot, h] = half * (1 + 2.0 ** -14) + amp[at, h] * ref.FP32

    def check(self, side, slots):
        c = self.cache
        there = c.codes64(side).cpu()[slots]
        there = there * c.scale[side].double().cpu().view(-1, c.kvh)[slots // c.group][..., None]
        over = (there - self.row[slots]).abs() - self.off[slots]
        assert (over <= 0).all(), over.max().item()


@pytest.mark.parametrize("codes,group,d,bs,size", [
    ("e4m3", 128, 128, 128, 0.0), ("int8", 16, 64, 32, 0.0), ("int8", 128, 128, 128, 0.03),
    ("e4m3", 32, 64, 32, 0.1)])
def test_block_scales(gpu_device, codes, group, d, bs, size):
    """`size`: the rows' size grows by e to that a token, so that scales grow within blocks."""
    dev, kvh, hq = gpu_device, 2, 8
    prompts, steps = [150, 37, 1], 60
    host, pages = ref.paged([n + steps + 3 for n in prompts], bs)
    host = host.astype(np.int64)
    cache = ref.BlockCache(pages, bs, kvh, d, group, codes, dev)
    sides = [Side(cache, pages * bs) for _ in range(2)]
    table = torch.from_numpy(host).to(dev)
    cos_sin = ref.table(max(prompts) + steps + 3, d).to(dev)
    g = torch.Generator().manual_seed(30)
    at = [0] * len(prompts)
    for step in range(steps + 1):
        # every seventh step two more tokens than are kept
        spare = 2 if step % 7 == 6 else 0
        news = prompts if step == 0 else [1 + spare] * len(prompts)
        positions = np.concatenate([np.arange(a, a + n) for a, n in zip(at, news)])
        slots = np.concatenate([ref.slots_of(host, b, np.arange(a, a + n), bs)
                                for b, (a, n) in enumerate(zip(at, news))])
        qkv = torch.randn(sum(news), hq + 2 * kvh, d, generator=g)
        qkv[:, hq:] *= torch.from_numpy(np.exp(size * positions)).float()[:, None, None]
        qkv = qkv.to(BF16).to(dev)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + kvh], qkv[:, hq + kvh:]
        places = torch.from_numpy(positions).to(dev)
        turned = block8_store(k, v, torch.from_numpy(slots).to(dev), *cache.args(), query=q,
                              positions=places, cos_sin=cos_sin)
        ref.check_rotated(turned, *ref.rotate(q, cos_sin, places, False), "queries")
        rows = [ref.rotate(k, cos_sin, places, False), (v.double(), v.double().abs())]
        for i, (y, amp) in enumerate(rows):
            sides[i].store(slots, y.cpu(), amp.cpu(), cache.scale[i].double().cpu().view(-1, kvh))
        lens = [a + n for a, n in zip(at, news)]
        if step % 10 == 0 or step % 7 == 6:
            live = torch.from_numpy(np.concatenate(
                [ref.slots_of(host, b, np.arange(n), bs) for b, n in enumerate(lens)]))
            for i in range(2):
                sides[i].check(i, live)
            got = block8_attention(turned, *cache.args(), table, lens, news, d ** -0.5,
                                   block_table_host=host)
            view = ref.Pages.__new__(ref.Pages)
            view.__dict__.update(host=host, table=table, data=cache.data, scale=cache.scale,
                                 codes=codes, kvh=kvh, d=d, bs=bs, group=group)
            want, bound, _, _ = win.attention64(turned, view, lens, news, d ** -0.5)
            win.check_out(got, want, bound, BF16)
        at = [n - spare for n in lens]
    # (a power of two seldom grows among rows of one size: their maxima lie within an octave)
    least = 10 if size or codes == "int8" else 1
    assert all(side.growths >= least for side in sides), "scales did grow within blocks"


def test_latent_rows(gpu_device):
    dev, heads, rank, dims, bs = gpu_device, 16, 512, 64, 16
    prompts, steps = [150, 37, 1], 24
    c = ref.Latents([n + steps for n in prompts], rank, dims, bs, BF16, device=dev, seed=31)
    cos_sin = ref.table(max(prompts) + steps, dims).to(dev)
    g = torch.Generator().manual_seed(32)
    at = [0] * len(prompts)
    total = c.data.shape[0] * bs
    kept = torch.zeros(total, rank).double(), torch.zeros(total, dims).double()
    amps = torch.zeros(total, dims).double()
    for step in range(steps + 1):
        news = prompts if step == 0 else [1] * len(prompts)
        positions = np.concatenate([np.arange(a, a + n) for a, n in zip(at, news)])
        slots = torch.from_numpy(np.concatenate([ref.slots_of(c.host, b, np.arange(a, a + n), bs)
                                                 for b, (a, n) in enumerate(zip(at, news))]))
        at = [a + n for a, n in zip(at, news)]
        down = torch.randn(sum(news), rank + dims, generator=g).to(BF16).to(dev)
        q = (0.5 * torch.randn(sum(news), heads, rank + dims, generator=g)).to(BF16).to(dev)
        places = torch.from_numpy(positions).to(dev)
        y, amp = ref.rotate(down[:, None, rank:], cos_sin, places, True)
        kept[0][slots], kept[1][slots] = down[:, :rank].double().cpu(), y[:, 0].cpu()
        amps[slots] = amp[:, 0].cpu()
        turned = q[..., rank:]
        y, amp = ref.rotate(turned, cos_sin, places, True)
        fp8_latent_store(down[:, :rank], down[:, rank:], places, cos_sin, slots.to(dev), c.data,
                         c.scale, c.rope, query=turned, interleaved=True, out_query=turned)
        ref.check_rotated(turned, y, amp, "queries")
        if step % 6:
            continue
        live = torch.from_numpy(np.concatenate(
            [ref.slots_of(c.host, b, np.arange(n), bs) for b, n in enumerate(at)]))
        scale = c.scale.view(-1, 1).cpu().double()[live]
        x = kept[0][live]
        assert ((scale - x.abs().amax(-1, keepdim=True) / 448).abs() <= scale * ref.TOP).all()
        codes = c.data.view(-1, rank).cpu()[live].view(ref.E4M3).double()
        ref.check_codes(codes * scale, scale, x, x.abs(), "latent", "e4m3")
        ref.check_rotated(c.rope.view(-1, dims).cpu()[live], kept[1][live], amps[live], "parts")
        want, bound = ref.latent64(q, c, at, news, 192 ** -0.5)
        got = fp8_latent_attention(q, *c.args(), at, news, 192 ** -0.5, block_table_host=c.host)
        win.check_out(got, want, bound, BF16)
