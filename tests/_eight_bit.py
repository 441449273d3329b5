# SPDX-License-Identifier: Apache-2.0
"""Inputs, 64-bit restatements and derived bounds for the tests of the rotating stores, the
cache with block scales and the latent cache."""

from __future__ import annotations

import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def table(rows, rot, dtype=torch.float32, base=10000.0):
    """[rows, rot]: the cosines, then the sines, of each position."""
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * torch.pow(
        base, -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype)


def rotate(x, cos_sin, positions, interleaved):
    """(64-bit rotated rows [T, H, D], the sizes of the products that each dim sums)."""
    x = x.double()
    rot = cos_sin.shape[1]
    row = cos_sin.double()[positions.long()][:, None]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y, amp = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    amp[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    amp[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, amp


#: fp32 products, a sum and a quotient, each off by 2^-24 at most, of terms of size amp
FP32 = 2.0 ** -22
#: what that makes of a row's largest: a pair's amp is at most twice its larger result
TOP = 2.0 ** -21


def check_rotated(got, y, amp, what):
    bound = y.abs() * HALF_STEP[got.dtype] + amp * FP32 + torch.finfo(got.dtype).tiny
    off = (got.double() - y).abs() - bound
    assert (off <= 0).all(), f"{what}: {off.max().item()} past the bound"


def check_codes(values, scale, y, amp, what, codes):
    """Values (code * scale) of rows y: within half a step of the codes."""
    if codes == "e4m3":  # 3 bits behind the leading one, subnormal under 2^-6
        half = torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    else:
        half = scale.expand_as(y) * 0.5
    off = (values - y).abs() - half * (1 + 2.0 ** -14) - amp * FP32
    assert (off <= 0).all(), f"{what}: {off.max().item()} past the bound"


def block_scale(top, codes):
    """s(a) in 64 bits, for a number."""
    if codes == "int8":
        return max(top / 127.0, 1e-6)
    if top <= 0:
        return 2.0 ** -20
    return max(2.0 ** -20, 2.0 ** math.ceil(math.log2(top / 448.0)))


class BlockCache:
    """Empty (or random) pages with block scales."""

    def __init__(self, pages, bs, kvh, d, group, codes, device="cpu", seed=0):
        g = torch.Generator().manual_seed(seed)
        self.codes, self.bs, self.kvh, self.d, self.group = codes, bs, kvh, d, group
        dtype = torch.uint8 if codes == "e4m3" else torch.int8
        low, high = (0, 127) if codes == "e4m3" else (-127, 128)
        shape = (pages, bs, kvh, d)
        self.data = [torch.randint(low, high, shape, generator=g).to(dtype).to(device)
                     for _ in range(2)]
        self.scale = [torch.exp2(torch.randint(-9, -6, (pages, bs // group, kvh), generator=g).float())
                      .to(device) for _ in range(2)]

    def args(self):
        return self.data[0], self.scale[0], self.data[1], self.scale[1]

    def codes64(self, side):
        x = self.data[side]
        x = x.view(E4M3) if self.codes == "e4m3" else x
        return x.double().view(-1, self.kvh, self.d)

    def clone(self):
        c = object.__new__(BlockCache)
        c.__dict__.update(self.__dict__)
        c.data, c.scale = [t.clone() for t in self.data], [t.clone() for t in self.scale]
        return c


def check_block_store(before, after, rows, slots, live):
    """``after`` holds ``before`` and the rows (y, amp) of both sides at their slots."""
    g, codes = before.group, before.codes
    slots = [int(s) if ok else -1 for s, ok in zip(slots, live)]
    runs: dict[int, list[int]] = {}
    for t, s in enumerate(slots):
        if s >= 0:
            runs.setdefault(s // g, []).append(t)
    for side, (y, amp) in enumerate(rows):
        y, amp = y.cpu(), amp.cpu()
        old, new = before.codes64(side).cpu(), after.codes64(side).cpu()
        s0 = before.scale[side].double().view(-1, before.kvh).cpu()
        s1 = after.scale[side].double().view(-1, before.kvh).cpu()
        touched = torch.zeros(s0.shape[0], dtype=torch.bool)
        same = torch.ones(old.shape[0], dtype=torch.bool)
        for block, tokens in runs.items():
            touched[block] = True
            first = min(slots[t] for t in tokens) - block * g
            at = torch.tensor([slots[t] for t in tokens])
            same[at] = False
            for h in range(before.kvh):
                top = y[tokens, h].abs().max().item()
                was = s0[block, h].item()
                want = {max(block_scale(top * f, codes), was if first else 0.0)
                        for f in (1 - TOP, 1 + TOP)}
                got = s1[block, h].item()
                assert any(abs(got - w) <= w * TOP for w in want), (side, block, h, got, want)
                check_codes(new[at, h] * got, torch.tensor(got).double(), y[tokens, h],
                            amp[tokens, h], f"side {side} block {block} head {h}", codes)
                if first:
                    there = slice(block * g, block * g + first)
                    if got == was:
                        assert torch.equal(new[there, h], old[there, h])
                    else:
                        half = got * (2.0 ** -10 if codes == "e4m3" else 0.5 + 2.0 ** -14)
                        off = (new[there, h] * got - old[there, h] * was).abs().max().item()
                        assert off <= half, (side, block, h, off, half)
                    same[there] = False
        assert torch.equal(s1[~touched], s0[~touched])
        raw0 = before.data[side].view(torch.uint8).view(old.shape).cpu()
        raw1 = after.data[side].view(torch.uint8).view(old.shape).cpu()
        assert torch.equal(raw1[same], raw0[same]), f"side {side}: rows that nobody wrote"


def paged(lens, bs, seed=0, spare=3):
    """Pages of requests of these lengths, anywhere: (table [B, width], pages)."""
    rng = np.random.default_rng(seed)
    width = max(1, max(-(-n // bs) for n in lens))
    pages = len(lens) * width + spare
    return rng.permutation(pages)[: len(lens) * width].reshape(len(lens), width), pages


def slots_of(host, b, positions, bs):
    p = np.asarray(positions, dtype=np.int64)
    return host[b, p // bs].astype(np.int64) * bs + p % bs


class Pages:
    """Keys and values of requests of these lengths in a cache with block scales, quantized as
    the store does (for ``_fp8_window.attention64``)."""

    def __init__(self, lens, kvh, d, bs, group, codes, *, device="cpu", seed=0, index=torch.int32,
                 spare=2):
        self.host, pages = paged(lens, bs, seed, spare)
        self.host = self.host.astype(np.int64)
        self.table = torch.from_numpy(self.host).to(device, index)
        g = torch.Generator().manual_seed(seed)
        channel = torch.exp(0.5 * torch.randn(kvh, d, generator=g))
        size = torch.exp(torch.randn(pages * bs, kvh, 1, generator=g))
        self.data, self.scale = [], []
        for x in (channel, size):
            x = (torch.randn(pages * bs, kvh, d, generator=g) * x).view(-1, group, kvh, d)
            top = x.abs().amax((1, 3))
            if codes == "e4m3":
                s = torch.exp2(torch.ceil(torch.log2(top / 448.0))).clamp_min(2.0 ** -20)
                x = (x / s[:, None, :, None]).to(E4M3).view(torch.uint8)
            else:
                s = (top / 127.0).clamp_min(1e-6)
                x = (x / s[:, None, :, None]).round().to(torch.int8)
            self.data.append(x.view(pages, bs, kvh, d).to(device).contiguous())
            self.scale.append(s.view(pages, bs // group, kvh).to(device).contiguous())
        self.codes, self.kvh, self.d, self.bs, self.group = codes, kvh, d, bs, group

    def rows(self, b, length):
        at = torch.from_numpy(slots_of(self.host, b, np.arange(length), self.bs)).to(
            self.table.device)
        out = []
        for data, scale in zip(self.data, self.scale):
            x = data.view(E4M3) if self.codes == "e4m3" else data
            x = x.double().view(-1, self.kvh, self.d)[at]
            out.append(x * scale.double().view(-1, self.kvh, 1)[at // self.group])
        return out

    def args(self):
        return self.data[0], self.scale[0], self.data[1], self.scale[1], self.table


class Latents:
    """Latent rows and position parts of requests of these lengths, quantized as the store does."""

    def __init__(self, lens, rank, dims, bs, dtype, *, device="cpu", seed=0, index=torch.int32,
                 spare=2):
        self.host, pages = paged(lens, bs, seed, spare)
        self.host = self.host.astype(np.int64)
        self.table = torch.from_numpy(self.host).to(device, index)
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(pages * bs, rank, generator=g) * torch.exp(
            0.5 * torch.randn(rank, generator=g)) * torch.exp(torch.randn(pages * bs, 1, generator=g))
        s = (x.abs().amax(-1, keepdim=True) / 448.0).clamp_min(1e-6)
        self.data = (x / s).clamp(-448, 448).to(E4M3).view(torch.uint8).view(pages, bs, rank).to(device)
        self.scale = s.view(pages, bs, 1).to(device)
        self.rope = torch.randn(pages, bs, dims, generator=g).to(dtype).to(device)
        self.rank, self.dims, self.bs = rank, dims, bs

    def rows(self, b, length):
        """64-bit ([length, R], [length, P])."""
        at = torch.from_numpy(slots_of(self.host, b, np.arange(length), self.bs)).to(
            self.table.device)
        c = self.data.view(E4M3).double().view(-1, self.rank)[at]
        return c * self.scale.double().view(-1, 1)[at], self.rope.double().view(-1, self.dims)[at]

    def args(self):
        return self.data, self.scale, self.rope, self.table


def latent64(q, cache, lens, news, scale):
    """(out, bound) in 64 bits; the bound as ``_fp8_window.attention64`` derives it: a score is
    R + P exact products summed in fp32, two products, two sums and a logarithm behind them,
    a weight goes through the matrix units in 16 bits."""
    heads, wide = q.shape[1:]
    rank = cache.rank
    out, bound = q.new_zeros((2, q.shape[0], heads, rank), dtype=torch.float64)
    row0 = 0
    for b, (length, n) in enumerate(zip(lens, news)):
        if n and length:
            c, r = cache.rows(b, length)
            k = torch.cat([c, r], 1).T.contiguous()
            pos = (length - n + torch.arange(n, device=q.device))[:, None]
            mask = (torch.arange(length, device=q.device) <= pos).repeat_interleave(heads, 0)
            x = q[row0:row0 + n].double().reshape(n * heads, wide)
            s = (x @ k * scale).masked_fill(~mask, -math.inf)
            size = torch.where(mask, (x.abs() @ k.abs() * scale).nan_to_num(0.0, 0.0, 0.0), 0.0)
            a = size.amax(-1, keepdim=True)
            top = s.amax(-1, keepdim=True)
            p = torch.where(mask, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            norm = p.sum(-1, keepdim=True)
            p = torch.where(mask, p / torch.where(norm == 0, 1.0, norm), 0.0)
            bad = (mask.double() @ c.isnan().double()) > 0
            v = torch.where(c.isfinite(), c, 0.0)
            o = torch.where(bad, math.nan, p @ v)
            o = torch.where(norm.isnan(), math.nan, o)
            off = 2 * (wide + 16) * 2.0 ** -24 * a + (length + 200) * 2.0 ** -24
            peak = (p * v.abs().amax(-1)).amax(-1, keepdim=True)
            ob = (off + 2.0 ** -11) * (p @ v.abs()) + length * 2.0 ** -24 * peak
            out[row0:row0 + n] = o.view(n, heads, rank)
            bound[row0:row0 + n] = ob.view(n, heads, rank)
        row0 += n
    return out, bound
