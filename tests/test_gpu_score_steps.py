# SPDX-License-Identifier: Apache-2.0
"""Attention among scores whose own step, in fp32 and the log2 domain, is near the offsets that
keep weights within fp16's range, or far past them: results stay finite, and follow from the
scores' differences.

The scores here are whole steps apart and exact in fp32: the queries hold a large number A and
its step B in two dims, the cached rows 1 and a whole number k of 0 .. 15, and the scale is the
fp32 number whose product with fp32(log2(e)) is 1.  A + B k then is the kernels' score whatever
the order of its sum, and a weight is 2^(B k) relative to another up to what exp2, sums and
16-bit weights add:
  weights in 16 bits 2^-11, exp2 and the norm (L + 200) 2^-24, the scale's own rounding
  2^-24 of the largest difference, 15 B; 2^-24 of the row's largest weight where they are
  subnormal.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests import _eight_bit as ref
from tests import _fp8_window as win
from vllm_ascend_quantized_kv_cache.ops.block8 import block8_attention
from vllm_ascend_quantized_kv_cache.ops.fp8_latent import fp8_latent_attention
from vllm_ascend_quantized_kv_cache.ops.fp8_window import fp8_per_token_head_window_attention

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
LN2 = float(np.float32(math.log(2.0)))
SIZES = [2.0 ** e for e in (20, 23, 24, 25, 26, 27, 28, 30, 34, 40)]
PATTERNS = ("random", "grow", "fall")


def _steps(length, pattern, seed):
    """Whole numbers of 0 .. 15 for the positions."""
    g = torch.Generator().manual_seed(seed)
    if pattern == "random":
        return torch.randint(0, 16, (length,), generator=g)
    k = torch.arange(length) * 16 // length - torch.randint(0, 3, (length,), generator=g)
    return k.clamp(0, 15) if pattern == "grow" else 15 - k.clamp(0, 15)


def _queries(rows, heads, wide, size, dtype, device):
    """Half of the heads with the steps up, half with them down."""
    q = torch.zeros(rows, heads, wide)
    q[..., 0], q[..., 1] = size, size * 2.0 ** -23
    q[:, heads // 2:, 1] *= -1.0
    return q.to(dtype).to(device)


def _expected(k, values, q, n):
    """(out, bound) [n, heads, D] of one request's last n rows; values [L, heads, D] in 64 bits."""
    length, heads = values.shape[:2]
    step = q[0, :, 1].double()[:, None]  # [heads, 1]
    k = k.to(values.device).double()[None]
    out, bound = [], []
    for i in range(n):
        end = length - n + i + 1
        d = step * k[:, :end]
        p = torch.exp(LN2 * (d - d.amax(-1, keepdim=True)))
        p = p / p.sum(-1, keepdim=True)
        v = values[:end].permute(1, 0, 2).contiguous()
        off = 2.0 ** -11 + (length + 200) * 2.0 ** -24 + 15 * step.abs()[..., None] * 2.0 ** -24
        out.append((p[:, None] @ v)[:, 0])
        low = length * 2.0 ** -24 * p.amax(-1) * v.abs().amax((1, 2))
        bound.append(((p[:, None] @ v.abs()) * off)[:, 0] + low[:, None])
    return torch.stack(out), torch.stack(bound)


def _codes(rows, dims, k, seed):
    """E4M3 codes of rows [.., dims] whose first two dims are 1 and k."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dims, generator=g)
    x[:, 0] = 1.0
    x[:, 1] = k
    return x.to(ref.E4M3).view(torch.uint8)


@pytest.mark.parametrize("heads,dtype", [(4, BF16), (16, BF16), (33, BF16), (64, BF16), (96, BF16),
                                         (3, FP32)])
@pytest.mark.parametrize("size", SIZES)
def test_latent_rows(gpu_device, size, heads, dtype):
    dev, rank, dims, bs = gpu_device, 512, 64, 64
    for length, n in ((700, 1), (700, 41), (6000, 2)):
        c = ref.Latents([length], rank, dims, bs, dtype, device=dev, seed=1)
        c.scale.fill_(1.0)
        q = _queries(n, heads, rank + dims, size, dtype, dev)
        at = torch.from_numpy(ref.slots_of(c.host, 0, np.arange(length), bs)).to(dev)
        for seed, pattern in enumerate(PATTERNS):
            k = _steps(length, pattern, seed)
            c.data.view(-1, rank)[at] = _codes(length, rank, k, seed).to(dev)
            rows, _ = c.rows(0, length)
            want, bound = _expected(k, rows[:, None].expand(-1, heads, -1), q, n)
            got = fp8_latent_attention(q, *c.args(), [length], [n], LN2, block_table_host=c.host)
            win.check_out(got, want, bound, dtype)


@pytest.mark.parametrize("heads", [4, 32, 33, 64, 96])
@pytest.mark.parametrize("size", [2.0 ** e for e in (22, 25, 28, 31, 34, 40)])
def test_latent_rows_of_any_scores(gpu_device, size, heads):
    """Scores of every size up to `size`, of both signs: whatever is seen stays finite."""
    for lens, news in (([700, 300], [1, 2]), ([700], [60]), ([6000], [300 if heads == 4 else 2])):
        c = ref.Latents(lens, 512, 64, 64, BF16, device=gpu_device, seed=18)
        q = win.query(sum(news), heads, 576, BF16, gpu_device, size=size)
        scale = 192 ** -0.5
        want, bound = ref.latent64(q, c, lens, news, scale)
        got = fp8_latent_attention(q, *c.args(), lens, news, scale, block_table_host=c.host)
        win.check_out(got, want, bound, BF16)


@pytest.mark.parametrize("codes,dtype", [("e4m3", BF16), ("int8", BF16), ("e4m3", FP32)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", SIZES)
def test_block_scales(gpu_device, size, d, codes, dtype):
    dev, hq, kvh, bs = gpu_device, 8, 2, 64
    for length, n in ((700, 1), (700, 41), (6000, 2)):
        c = ref.Pages([length], kvh, d, bs, 16, codes, device=dev, seed=2)
        for scale in c.scale:
            scale.fill_(1.0)
        q = _queries(n, hq, d, size, dtype, dev)
        at = torch.from_numpy(ref.slots_of(c.host, 0, np.arange(length), bs)).to(dev)
        for seed, pattern in enumerate(PATTERNS):
            k = _steps(length, pattern, seed)
            if codes == "e4m3":
                rows = _codes(length * kvh, d, k.repeat_interleave(kvh), seed)
            else:
                rows = torch.zeros(length * kvh, d, dtype=torch.int8)
                rows[:, 0], rows[:, 1] = 1, k.repeat_interleave(kvh)
            c.data[0].view(-1, kvh, d)[at] = rows.view(length, kvh, d).to(dev)
            _, values = c.rows(0, length)
            want, bound = _expected(k, values.repeat_interleave(hq // kvh, 1), q, n)
            got = block8_attention(q, *c.args(), [length], [n], LN2, block_table_host=c.host)
            win.check_out(got, want, bound, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", SIZES)
def test_windowed_attention(gpu_device, size, d, dtype):
    dev, hq, kvh, bs = gpu_device, 8, 2, 64
    for length, n in ((700, 1), (700, 41), (6000, 2), (1200, 300)):
        c = win.Cache([length], kvh, d, bs, device=dev, seed=3)
        c.ks.fill_(1.0)
        c.vs.fill_(1.0)
        q = _queries(n, hq, d, size, dtype, dev)
        at = torch.from_numpy(c.slots(0, np.arange(length))).to(dev)
        for seed, pattern in enumerate(PATTERNS):
            k = _steps(length, pattern, seed)
            rows = _codes(length * kvh, d, k.repeat_interleave(kvh), seed)
            c.k.view(-1, kvh, d)[at] = rows.view(length, kvh, d).to(dev)
            _, values = c.rows(0, length)
            want, bound = _expected(k, values.repeat_interleave(hq // kvh, 1), q, n)
            got = fp8_per_token_head_window_attention(q, *c.args(), [length], [n], LN2,
                                                      block_table_host=c.host)
            win.check_out(got, want, bound, dtype)
