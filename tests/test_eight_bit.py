# SPDX-License-Identifier: Apache-2.0
"""The rotating stores, the cache with block scales and the latent cache, without a GPU:
what is refused, and the host's page checks."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from tests import _eight_bit as ref
from vllm_ascend_quantized_kv_cache.ops import _native
from vllm_ascend_quantized_kv_cache.ops.block8 import block8_attention, block8_store
from vllm_ascend_quantized_kv_cache.ops.fp8_latent import fp8_latent_attention, fp8_latent_store
from vllm_ascend_quantized_kv_cache.ops.fp8_rotary import fp8_per_token_head_rotary_store

BF16 = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _built():
    if not _native.library_path().exists():
        pytest.skip("libkvq_hip.so not built (run __graft_entry__.build())")


def _refused(call, args, kw, match):
    with pytest.raises(RuntimeError, match=match):
        call(**{**args, **kw})


# ---- the per-token store with a rotation ------------------------------------------


def _rotary():
    return dict(
        query=torch.zeros(3, 4, 64, dtype=BF16), key=torch.zeros(3, 2, 64, dtype=BF16),
        value=torch.zeros(3, 2, 64, dtype=BF16), positions=torch.arange(3),
        cos_sin=torch.zeros(9, 64), slot_mapping=torch.arange(3),
        k_data=torch.zeros(2, 16, 2, 64, dtype=torch.uint8), k_scale=torch.zeros(2, 16, 2, 1),
        v_data=torch.zeros(2, 16, 2, 64, dtype=torch.uint8), v_scale=torch.zeros(2, 16, 2, 1))


ROTATIONS = [
    (dict(positions=torch.arange(4)), "positions must be 1D of 3"),
    (dict(positions=torch.zeros(3, 1, dtype=torch.int64)), "positions must be 1D of 3"),
    (dict(positions=torch.zeros(3)), "int32/int64"),
    (dict(cos_sin=torch.zeros(9)), "cos_sin must be contiguous"),
    (dict(cos_sin=torch.zeros(0, 64)), "cos_sin must be contiguous"),
    (dict(cos_sin=torch.zeros(64, 9).T), "cos_sin must be contiguous"),
    (dict(cos_sin=torch.zeros(9, 64, dtype=torch.float64)), "unsupported floating dtype"),
    (dict(cos_sin=torch.zeros(9, 0)), "rotates 0 dims"),
    (dict(cos_sin=torch.zeros(9, 33)), "rotates 33 dims"),
    (dict(cos_sin=torch.zeros(9, 66)), "rotates 66 dims"),
    (dict(positions=None), "needs positions and cos_sin"),
]
QUERIES = [
    (dict(query=torch.zeros(2, 4, 64, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(3, 4, 32, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(3, 0, 64, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(3, 256, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(3, 4, 64)), "query is torch.float32"),
    (dict(out_query=torch.zeros(3, 4, 64)), "out_query is torch.float32"),
    (dict(out_query=torch.zeros(3, 5, 64, dtype=BF16)), "does not match query"),
    (dict(query=None, out_query=torch.zeros(3, 4, 64, dtype=BF16)), "out_query needs query"),
]


@pytest.mark.parametrize("kw,match", [
    *ROTATIONS, *QUERIES,
    (dict(cos_sin=None), "needs positions and cos_sin"),
    (dict(key=torch.zeros(3, 128, dtype=BF16)), "key and value must be"),
    (dict(value=torch.zeros(3, 2, 64)), "value is torch.float32"),
    (dict(value=torch.zeros(3, 3, 64, dtype=BF16)), "key"),
    (dict(slot_mapping=torch.arange(4)), "slot_mapping must be 1D of 3"),
    (dict(slot_mapping=torch.zeros(3)), "slot_mapping must be int32/int64"),
    (dict(key=torch.zeros(3, 2, 64, dtype=torch.float64),
          value=torch.zeros(3, 2, 64, dtype=torch.float64)), "unsupported floating dtype"),
    (dict(k_data=torch.zeros(2, 16, 3, 64, dtype=torch.uint8)), "key data cache must be uint8"),
    (dict(v_data=torch.zeros(2, 16, 2, 64, dtype=torch.int8)), "value data cache must be uint8"),
    (dict(v_scale=torch.zeros(2, 16, 2, 1, dtype=torch.float16)), "value scale"),
    ({}, "no CPU fallback"),
])
def test_rotary_store_refuses(kw, match):
    _refused(fp8_per_token_head_rotary_store, _rotary(), kw, match)


def test_a_store_without_tokens_needs_no_gpu():
    a = _rotary()
    for name in ("query", "key", "value", "positions", "slot_mapping"):
        a[name] = a[name][:0]
    assert fp8_per_token_head_rotary_store(**a) is a["query"]
    out = a["query"].clone()
    assert fp8_per_token_head_rotary_store(**a, out_query=out) is out
    assert fp8_per_token_head_rotary_store(**{**a, "query": None}) is None
    b = _block()
    for name in ("query", "key", "value", "positions", "slot_mapping"):
        b[name] = b[name][:0]
    assert block8_store(**b) is b["query"]
    c = _latent()
    for name in ("query", "latent", "part", "positions", "slot_mapping"):
        c[name] = c[name][:0]
    assert fp8_latent_store(**c) is c["query"]


# ---- the cache with block scales ----------------------------------------------------


def _block(dtype=torch.uint8):
    a = _rotary()
    for side in ("k", "v"):
        a[side + "_data"] = torch.zeros(2, 16, 2, 64, dtype=dtype)
        a[side + "_scale"] = torch.zeros(2, 1, 2)
    return a


CACHES = [
    (dict(k_data=torch.zeros(2, 16, 128, dtype=torch.uint8)), "data caches must be uint8"),
    (dict(k_data=torch.zeros(2, 16, 2, 64)), "data caches must be uint8"),
    (dict(v_data=torch.zeros(2, 16, 2, 64, dtype=torch.int8)), "data caches must be uint8"),
    (dict(v_data=torch.zeros(3, 16, 2, 64, dtype=torch.uint8)), "views disagree"),
    (dict(k_scale=torch.zeros(2, 2)), "views disagree"),
    (dict(k_scale=torch.zeros(2, 1, 3), v_scale=torch.zeros(2, 1, 3)), "views disagree"),
    (dict(v_scale=torch.zeros(2, 2, 2)), "views disagree"),
    (dict(k_scale=torch.zeros(2, 3, 2), v_scale=torch.zeros(2, 3, 2)), "3 scales do not divide"),
    (dict(k_scale=torch.zeros(2, 0, 2), v_scale=torch.zeros(2, 0, 2)), "0 scales do not divide"),
    (dict(k_scale=torch.zeros(2, 1, 2, dtype=BF16)), "scale caches must be float32"),
    (dict(v_scale=torch.zeros(2, 1, 4)[..., ::2]), "value scale must be contiguous"),
    (dict(k_data=torch.zeros(2, 2, 16, 64, dtype=torch.uint8).transpose(1, 2)),
     "key data must be contiguous"),
]


@pytest.mark.parametrize("kw,match", [
    *ROTATIONS, *QUERIES, *CACHES,
    (dict(cos_sin=None, positions=None), "queries need positions"),
    (dict(cos_sin=None, query=None), "needs positions and cos_sin"),
    (dict(key=torch.zeros(3, 2, 32, dtype=BF16)), "key and value must be"),
    (dict(value=torch.zeros(2, 2, 64, dtype=BF16)), "key and value must be"),
    (dict(value=torch.zeros(3, 2, 64)), "value is torch.float32"),
    (dict(slot_mapping=torch.zeros(3, 1, dtype=torch.int64)), "slot_mapping must be 1D of 3"),
    (dict(slot_mapping=torch.zeros(3)), "int32/int64"),
    ({}, "no CPU fallback"),
    (dict(query=None, cos_sin=None, positions=None), "no CPU fallback"),
])
def test_block_store_refuses(kw, match):
    _refused(block8_store, _block(), kw, match)


def _attend(codes="e4m3"):
    c = ref.Pages([40, 17], 2, 64, 16, 16, codes)
    return dict(query=torch.zeros(4, 4, 64, dtype=BF16), k_data=c.data[0], k_scale=c.scale[0],
                v_data=c.data[1], v_scale=c.scale[1], block_table=c.table, seq_lens=[40, 17],
                query_lens=[1, 3], scale=0.1)


LENGTHS = [
    (dict(seq_lens=[40, -1]), "negative seq_lens"),
    (dict(query_lens=[5, -1]), "negative query_lens"),
    (dict(query_lens=[4]), "1 query_lens for 2"),
    (dict(query_lens=[2, 3]), "sum to 5"),
    (dict(seq_lens=[40, 49]), "does not cover the longest"),
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int32)), "2D with a row per request"),
    (dict(block_table=torch.zeros(2, 3)), "int32/int64"),
    (dict(block_table_host=np.zeros((1, 3))), "the host's copy is \\(1, 3\\)"),
    (dict(block_table=torch.full((2, 3), 100, dtype=torch.int32)), "request 0 sees"),
    (dict(block_table=torch.tensor([[0, 1, 2], [3, -1, 4]])), "request 1 sees"),
]


@pytest.mark.parametrize("kw,match", [
    *LENGTHS,
    (dict(query=torch.zeros(4, 4, 32, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(4, 256, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(4, 3, 64, dtype=BF16)), "3 query heads over 2"),
    (dict(query=torch.zeros(4, 0, 64, dtype=BF16)), "0 query heads over 2"),
    (dict(query=torch.zeros(4, 4, 64, dtype=torch.float64)), "unsupported floating dtype"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(scale=float("inf")), "scale must be positive"),
    (dict(window=0), "window must be at least 1"),
    (dict(sinks=-1), "sinks must not be negative"),
    (dict(out=torch.zeros(5, 4, 64, dtype=BF16)), "does not match query"),
    (dict(k_data=torch.zeros(8, 16, 2, 64)), "data caches must be uint8"),
    (dict(k_scale=torch.zeros(8, 3, 2)), "views disagree"),
    ({}, "no CPU fallback"),
])
def test_block_attention_refuses(kw, match):
    _refused(block8_attention, _attend(), kw, match)


def test_pages_that_nobody_sees_may_be_gone():
    a = _attend()
    host = a["block_table"].numpy().astype(np.int64)
    host[1, 2] = host[0, 0] = -1  # behind the last position, and behind the window
    _refused(block8_attention, a, dict(block_table_host=host), "request 0 sees")
    _refused(block8_attention, a, dict(block_table_host=host, window=17), "no CPU fallback")
    _refused(block8_attention, a, dict(block_table_host=host, window=17, sinks=1), "request 0 sees")


def test_a_call_without_rows_needs_no_gpu():
    a = _attend("int8")
    a["query_lens"] = [0, 0]
    assert not block8_attention(**a).any()
    out = torch.ones(4, 4, 64)
    assert block8_attention(**a, out=out) is out and (out == 1).all()
    b = _latents()
    b["query_lens"] = [0, 0]
    got = fp8_latent_attention(**b)
    assert got.shape == (4, 4, 32) and not got.any()


# ---- the latent cache ---------------------------------------------------------------


def _latent():
    return dict(
        latent=torch.zeros(3, 32, dtype=BF16), part=torch.zeros(3, 16, dtype=BF16),
        positions=torch.arange(3), cos_sin=torch.zeros(9, 16), slot_mapping=torch.arange(3),
        data=torch.zeros(2, 16, 32, dtype=torch.uint8), scale=torch.zeros(2, 16, 1),
        rope=torch.zeros(2, 16, 16, dtype=BF16), query=torch.zeros(3, 4, 16, dtype=BF16))


LATENT_CACHES = [
    (dict(data=torch.zeros(2, 16, 32)), "data must be uint8"),
    (dict(data=torch.zeros(2, 16, 1, 32, dtype=torch.uint8)), "data must be uint8"),
    (dict(data=torch.zeros(2, 32, 16, dtype=torch.uint8).transpose(1, 2)),
     "data must be contiguous"),
    (dict(scale=torch.zeros(2, 16)), "scale must be float32"),
    (dict(scale=torch.zeros(2, 16, 1, dtype=BF16)), "scale must be float32"),
    (dict(rope=torch.zeros(2, 15, 16, dtype=BF16)), "rope must be"),
    (dict(rope=torch.zeros(2, 16, 16, dtype=torch.int8)), "unsupported floating dtype"),
]


@pytest.mark.parametrize("kw,match", [
    *LATENT_CACHES,
    (dict(latent=torch.zeros((), dtype=BF16)), "latent and part must be"),
    (dict(latent=torch.zeros(3, 33, dtype=BF16)), "latent and part must be"),
    (dict(part=torch.zeros(2, 16, dtype=BF16)), "latent and part must be"),
    (dict(part=torch.zeros(3, 16)), "part torch.float32"),
    (dict(rope=torch.zeros(2, 16, 16)), "rope torch.float32"),
    (dict(slot_mapping=torch.arange(2)), "slot_mapping must be 1D of 3"),
    (dict(slot_mapping=torch.zeros(3)), "int32/int64"),
    (dict(positions=torch.arange(2)), "positions must be 1D of 3"),
    (dict(cos_sin=None), "needs positions and cos_sin"),
    (dict(cos_sin=torch.zeros(9, 8)), "rotates 8 dims, the position part has 16"),
    (dict(cos_sin=torch.zeros(9, 18)), "rotates 18 dims"),
    (dict(query=torch.zeros(3, 4, 32, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(3, 4, 16)), "query is torch.float32"),
    (dict(out_query=torch.zeros(3, 2, 16, dtype=BF16)), "does not match query"),
    (dict(query=None, out_query=torch.zeros(3, 2, 16, dtype=BF16)), "out_query needs query"),
    ({}, "no CPU fallback"),
])
def test_latent_store_refuses(kw, match):
    _refused(fp8_latent_store, _latent(), kw, match)


def test_rows_that_share_elements_are_seen():
    from vllm_ascend_quantized_kv_cache.ops.fp8_latent import _apart

    x = torch.zeros(5, 4, 48)
    for t in (x, x[..., 32:], x.transpose(0, 1), x[::2, 1:3], x[:1], x[:, :1, 8:24],
              x[:1].expand(1, 4, 48), x[:, :1].transpose(0, 1), torch.zeros(1, 1, 8)):
        assert _apart(t), (t.shape, t.stride())
    for t in (x[:1].expand(5, 4, 48), x[:, :1].expand(5, 4, 48), x[..., ::2],
              x.flatten().as_strided((5, 4, 48), (16, 240, 1)),
              x.flatten().as_strided((2, 4, 48), (100, 48, 1))):
        assert not _apart(t), (t.shape, t.stride())


def _latents():
    c = ref.Latents([40, 17], 32, 16, 16, BF16)
    return dict(query=torch.zeros(4, 4, 48, dtype=BF16), data=c.data, scale=c.scale, rope=c.rope,
                block_table=c.table, seq_lens=[40, 17], query_lens=[1, 3], softmax_scale=0.1)


@pytest.mark.parametrize("kw,match", [
    *LENGTHS,
    (dict(query=torch.zeros(4, 4, 32, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(4, 0, 48, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(4, 192, dtype=BF16)), "query must be"),
    (dict(query=torch.zeros(4, 4, 48)), "query is torch.float32, rope torch.bfloat16"),
    (dict(softmax_scale=0.0), "softmax_scale must be positive"),
    (dict(softmax_scale=-1.0), "softmax_scale must be positive"),
    (dict(softmax_scale=float("nan")), "softmax_scale must be positive"),
    (dict(out=torch.zeros(4, 4, 48, dtype=BF16)), "out must be"),
    ({}, "no CPU fallback"),
])
def test_latent_attention_refuses(kw, match):
    _refused(fp8_latent_attention, _latents(), kw, match)


@pytest.mark.parametrize("kw,match", LATENT_CACHES)
def test_latent_attention_refuses_caches(kw, match):
    args = _latents()
    args.update((k, _latent()[k]) for k in ("data", "scale", "rope"))
    _refused(fp8_latent_attention, args, kw, match)


# ---- the C entries, which every caller reaches ----------------------------------------


def test_sizing_calls_refuse():
    lib = _native.lib()
    lens, news = (ctypes.c_int64 * 2)(40, 17), (ctypes.c_int64 * 2)(1, 3)
    bf16, e4m3 = _native.dtype_code(BF16), _native.KVQ_CODES_E4M3

    def block(lens=lens, news=news, batch=2, dtype=bf16, hq=4, kvh=2, d=64, bs=16, group=16,
              codes=e4m3, window=0, sinks=0):
        return lib.kvq_block8_attn_workspace_bytes(
            lens, news, batch, dtype, hq, kvh, d, bs, group, codes, window, sinks)

    for bad in (dict(lens=None), dict(news=None), dict(batch=-1), dict(dtype=99), dict(hq=3),
                dict(kvh=0), dict(hq=0), dict(d=0), dict(d=516), dict(bs=0), dict(group=5),
                dict(group=0), dict(codes=7), dict(window=-1), dict(sinks=-1),
                dict(lens=(ctypes.c_int64 * 2)(-1, 1)), dict(news=(ctypes.c_int64 * 2)(1, -1)),
                dict(lens=(ctypes.c_int64 * 2)(1 << 40, 1))):
        assert block(**bad) < 0, bad

    def latent(lens=lens, news=news, batch=2, dtype=bf16, heads=4, rank=32, part=16, bs=16):
        return lib.kvq_fp8_latent_attn_workspace_bytes(
            lens, news, batch, dtype, heads, rank, part, bs)

    for bad in (dict(lens=None), dict(news=None), dict(batch=-1), dict(dtype=99), dict(heads=0),
                dict(heads=1 << 20), dict(rank=0), dict(rank=30), dict(rank=516), dict(part=0),
                dict(part=300), dict(bs=0), dict(lens=(ctypes.c_int64 * 2)(-1, 1)),
                dict(news=(ctypes.c_int64 * 2)(1 << 40, 1))):
        assert latent(**bad) < 0, bad


def test_calls_refuse_null_pointers():
    lib = _native.lib()
    lens, news = (ctypes.c_int64 * 1)(40), (ctypes.c_int64 * 1)(1)
    bf16 = _native.dtype_code(BF16)
    i64 = _native.index_code(torch.int64)
    assert lib.kvq_fp8_latent_attn(
        None, bf16, 192, lens, news, 1, 4, 32, 16, 0.1, None, None, None, 4, 16, None, i64, 3, None,
        0, None, None) < 0
    assert lib.kvq_block8_attn(
        None, bf16, 256, lens, news, 1, 4, 2, 64, 0.1, 0, 0, _native.KVQ_CODES_E4M3, None, None,
        None, None, 4, 16, 16, None, i64, 3, None, 0, None, None) < 0
    assert lib.kvq_block8_store(
        None, 0, None, 0, None, 128, None, 128, bf16, None, 0, None, 0, 0, 0, 0, None, i64, 1, 0, 2,
        64, _native.KVQ_CODES_E4M3, None, None, None, None, 2, 16, 16, None) < 0
    assert lib.kvq_fp8_latent_store(
        None, 0, 0, None, 0, 0, None, 32, None, 16, bf16, None, i64, None, 0, 9, 0, None, i64, 1, 0,
        32, 16, None, None, None, 2, 16, None) < 0
