# SPDX-License-Identifier: Apache-2.0
"""Caches of more than 2^32 bytes: a request whose pages lie behind that bound is stored and
read as one in a small cache is, bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import _eight_bit as ref
from vllm_ascend_quantized_kv_cache.ops.block8 import block8_attention, block8_store
from vllm_ascend_quantized_kv_cache.ops.fp8_latent import fp8_latent_attention, fp8_latent_store
from vllm_ascend_quantized_kv_cache.ops.fp8_rotary import fp8_per_token_head_rotary_store

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
BS, TOKENS, PAGES = 128, 300, 3


def _rows(shape, seed, device):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(BF16).to(device)


def _places(first, device):
    """(slots, table, its host's copy) of a request in pages `first` .., last one first."""
    host = np.arange(first + PAGES - 1, first - 1, -1, dtype=np.int64)[None]
    slots = torch.from_numpy(ref.slots_of(host, 0, np.arange(TOKENS), BS)).to(device)
    return slots, torch.from_numpy(host).to(device, torch.int32), host


def _both(pages, device, run):
    near = run(PAGES, *_places(0, device))
    far = run(pages, *_places(pages - PAGES, device))
    for a, b in zip(near, far):
        assert torch.equal(a, b)
    assert all(torch.isfinite(x.float()).all() for x in near)


@pytest.mark.parametrize("codes", [torch.uint8, torch.int8])
def test_block_scales(gpu_device, codes):
    dev, kvh, d = gpu_device, 8, 128
    k, v = _rows((TOKENS, kvh, d), 1, dev), _rows((TOKENS, kvh, d), 2, dev)
    cos_sin, positions = ref.table(TOKENS, d).to(dev), torch.arange(TOKENS, device=dev)

    def run(pages, slots, table, host):
        cache = [x for _ in range(2) for x in (
            torch.empty(pages, BS, kvh, d, dtype=codes, device=dev),
            torch.empty(pages, BS // 64, kvh, device=dev))]
        q = block8_store(k, v, slots, *cache, query=_rows((TOKENS, 16, d), 3, dev),
                         positions=positions, cos_sin=cos_sin)
        for news in (1, 90):
            yield block8_attention(q[-news:], *cache, table, [TOKENS], [news], d ** -0.5,
                                   block_table_host=host)
        yield block8_attention(q[-2:].float(), *cache, table, [TOKENS], [2], d ** -0.5,
                               block_table_host=host)

    _both(2 ** 32 // (BS * kvh * d) + 10, dev, lambda *a: list(run(*a)))


def test_token_scales(gpu_device):
    dev, kvh, d = gpu_device, 8, 128
    k, v = _rows((TOKENS, kvh, d), 1, dev), _rows((TOKENS, kvh, d), 2, dev)
    cos_sin, positions = ref.table(TOKENS, d).to(dev), torch.arange(TOKENS, device=dev)

    def run(pages, slots, table, host):
        cache = [x for _ in range(2) for x in (
            torch.empty(pages, BS, kvh, d, dtype=torch.uint8, device=dev),
            torch.empty(pages, BS, kvh, 1, device=dev))]
        fp8_per_token_head_rotary_store(None, k, v, positions, cos_sin, slots, *cache)
        return [x.flatten(0, 1)[slots].float() for x in cache]

    _both(2 ** 32 // (BS * kvh * d) + 10, dev, run)


def test_latent_rows(gpu_device):
    dev, rank, dims = gpu_device, 512, 64
    latent, part = _rows((TOKENS, rank), 1, dev), _rows((TOKENS, dims), 2, dev)
    cos_sin, positions = ref.table(TOKENS, dims).to(dev), torch.arange(TOKENS, device=dev)

    def run(pages, slots, table, host):
        for dtype in (BF16, torch.float32):
            cache = (torch.empty(pages, BS, rank, dtype=torch.uint8, device=dev),
                     torch.empty(pages, BS, 1, device=dev),
                     torch.empty(pages, BS, dims, dtype=dtype, device=dev))
            fp8_latent_store(latent.to(dtype), part.to(dtype), positions, cos_sin, slots, *cache)
            for news in (1, 20):
                q = _rows((news, 16, rank + dims), 3, dev).to(dtype)
                yield fp8_latent_attention(q, *cache, table, [TOKENS], [news], 192 ** -0.5,
                                           block_table_host=host)

    _both(2 ** 32 // (BS * rank) + 10, dev, lambda *a: list(run(*a)))
