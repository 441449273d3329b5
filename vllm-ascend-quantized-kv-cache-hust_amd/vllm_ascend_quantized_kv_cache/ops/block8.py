# SPDX-License-Identifier: Apache-2.0
"""A paged cache of 8-bit codes with a scale for each block of positions and head
(``kvq_block8_*``): the store, with the position rotation applied on the way, and
causal attention straight over the codes.

Codes are ``[NB, Bs, KVH, D]``, E4M3 (``torch.uint8``) or INT8 (``torch.int8``),
scales fp32 ``[NB, Bs // G, KVH]``: one for ``G`` positions of a page and a head,
``G`` a divisor of the page.  A page of 128 positions then keeps 4 bytes of scale
for each head and side where ``fp8_per_token_head`` keeps 512.  The reference has
no counterpart.

A block's rows may come in several calls (a token a step): its scale grows with
them, and the rows that are there are requantized when it does.  That costs E4M3
codes nothing but subnormals; INT8 codes are rounded once more each time (rows of
one size, a token a call: 1.25 times the error of one call, rms, in blocks of 16
positions, 1.30 in blocks of 128).
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native
from .fp8_rotary import (
    _check_devices,
    _check_query,
    _check_rotation,
    _rows,
    _target,
    _token_stride,
)
from .fp8_window import _MOST, _lengths, _on_device, _table

_STORE = "block8_store"
_ATTENTION = "block8_attention"
_CODES = {torch.uint8: _native.KVQ_CODES_E4M3, torch.int8: _native.KVQ_CODES_INT8}


def _check_cache(what: str, k_data, k_scale, v_data, v_scale):
    """(pages, positions a page, heads, head size, positions a scale, kind of codes)."""
    shape, dtype = k_data.shape, k_data.dtype
    if len(shape) != 4 or dtype not in _CODES or v_data.dtype is not dtype:
        raise RuntimeError(
            f"{what}: data caches must be uint8 (E4M3) or int8 [NB, Bs, KVH, D], got "
            f"{tuple(shape)} / {dtype} and {v_data.dtype}."
        )
    nb, bs, kvh, d = shape
    scales = k_scale.shape
    if v_data.shape != shape or v_scale.shape != scales or len(scales) != 3 or (
            scales[0] != nb or scales[2] != kvh):
        raise RuntimeError(
            f"{what}: cache views disagree: k_data {tuple(shape)}, k_scale {tuple(scales)}, "
            f"v_data {tuple(v_data.shape)}, v_scale {tuple(v_scale.shape)}."
        )
    if scales[1] == 0 or bs == 0 or bs % scales[1]:
        raise RuntimeError(f"{what}: {scales[1]} scales do not divide a page of {bs} positions.")
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
        raise RuntimeError(
            f"{what}: scale caches must be float32, got {k_scale.dtype} and {v_scale.dtype}.")
    device = k_data.device
    for name, t in (("key data", k_data), ("key scale", k_scale), ("value data", v_data),
                    ("value scale", v_scale)):
        if not t.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be contiguous.")
        if t.device != device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, key data on {device}.")
    return nb, bs, kvh, d, bs // scales[1], _CODES[dtype]


def block8_store(
    key: torch.Tensor,
    value: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_data: torch.Tensor,
    k_scale: torch.Tensor,
    v_data: torch.Tensor,
    v_scale: torch.Tensor,
    *,
    query: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    cos_sin: torch.Tensor | None = None,
    interleaved: bool = False,
    out_query: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write ``[T, KVH, D]`` keys and values into the cache by slot; with ``cos_sin``,
    rotated to ``positions`` on the way (keys), as
    ``fp8_per_token_head_rotary_store`` rotates, and ``query [T, Hq, D]`` with them.
    Returns the rotated queries: ``out_query``, which may be ``query`` itself, or a
    fresh tensor; None without queries.

    With ``a`` the largest ``|y|`` of a block's new rows and head,
    ``s(a) = max(2^-20, least 2^e with a <= 448 * 2^e)`` for E4M3 codes (which float:
    a power of two loses them nothing) and ``max(a / 127, 1e-6)`` for INT8.  The
    block's scale becomes ``s(a)``, or, where the first new row lies behind the
    block's start, the larger of that and what it was; the rows before them are
    requantized when it grows.  Codes are ``y / scale`` rounded to nearest even.

    The rows of one block are neighbours in the call and each slot is given once.
    A row written at a block's start begins it anew; rows behind the last one
    written (a speculation taken back) stay as they were and count as gone.  What
    they did to the scale stays: it grows only, until a row at the block's start.
    Negative slots, and slots outside the cache, are padding; so are rows whose
    position is outside the table.  A row that is not finite makes its block
    NaN (INT8: its scale), for good likewise.  bf16, fp16 or fp32 rows, which may
    lie apart.
    """
    nb, bs, kvh, d, group, codes = _check_cache(_STORE, k_data, k_scale, v_data, v_scale)
    if key.dim() != 3 or key.shape != value.shape or key.shape[1:] != (kvh, d):
        raise RuntimeError(
            f"{_STORE}: key and value must be [tokens, {kvh}, {d}], got {tuple(key.shape)} and "
            f"{tuple(value.shape)}."
        )
    tokens = key.shape[0]
    dtype = _native.dtype_code(key.dtype)
    if value.dtype != key.dtype:
        raise RuntimeError(f"{_STORE}: value is {value.dtype}, key {key.dtype}.")
    if slot_mapping.shape != (tokens,):
        raise RuntimeError(
            f"{_STORE}: slot_mapping must be 1D of {tokens} slots, got {tuple(slot_mapping.shape)}.")
    slot_type = _native.index_code(slot_mapping.dtype)
    _check_devices(_STORE, key, value=value, slot_mapping=slot_mapping, cache=k_data)
    pos_type = table_type = table_rows = rot = 0
    if cos_sin is not None or positions is not None:
        pos_type, table_type, table_rows, rot = _check_rotation(
            _STORE, positions, cos_sin, interleaved, tokens, d, key)
    if query is not None:
        if cos_sin is None:
            raise RuntimeError(f"{_STORE}: queries need positions and cos_sin.")
        _check_query(_STORE, query, out_query, tokens, d, key)
    elif out_query is not None:
        raise RuntimeError(f"{_STORE}: out_query needs query.")
    if tokens == 0:
        return query if out_query is None else out_query
    _native.require_gpu_tensors(_STORE, key)
    k, k_stride = _rows(key)
    v, v_stride = _rows(value)
    q, q_stride, target = None, 0, None
    if query is not None:
        q, q_stride = _rows(query)
        target = _target(query, out_query, (key, value))
    slots = slot_mapping.contiguous()
    places = None if positions is None else positions.contiguous()
    with _on_device(k_data):
        rc = _native.lib().kvq_block8_store(
            _native.ptr(q), q_stride, _native.ptr(target),
            0 if q is None else _token_stride(target), k.data_ptr(), k_stride, v.data_ptr(),
            v_stride, dtype, _native.ptr(places), pos_type, _native.ptr(cos_sin), table_type,
            table_rows, rot, 1 if interleaved else 0, slots.data_ptr(), slot_type, tokens,
            0 if q is None else q.shape[1], kvh, d, codes, k_data.data_ptr(), k_scale.data_ptr(),
            v_data.data_ptr(), v_scale.data_ptr(), nb, bs, group, _native.stream_of(k_data),
        )
    _native.check(rc, "kvq_block8_store")
    if out_query is not None and target is not out_query:
        out_query.copy_(target)
        return out_query
    return target


def block8_attention(
    query: torch.Tensor,
    k_data: torch.Tensor,
    k_scale: torch.Tensor,
    v_data: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int],
    query_lens: Sequence[int],
    scale: float,
    *,
    window: int | None = None,
    sinks: int = 0,
    out: torch.Tensor | None = None,
    block_table_host=None,
) -> torch.Tensor:
    """Causal attention of TND ``query [sum query_lens, Hq, D]`` straight over the
    codes, through an optional sliding window.

    Each request's rows are its last ``query_lens[b]`` of ``seq_lens[b]`` cached
    positions (their keys and values are stored already).  A row at position ``p``
    sees positions ``j <= p``; with ``window``, of those the last ``window`` and the
    first ``sinks``.  A row that sees nothing gives zeros.  Keys and values are
    ``code * scale`` of their block, not rounded to the query's type (value scales
    under 2^-90 may count as 0; one that is not finite leaves no finite number in
    the rows that see its block).  Sums are fp32; with bf16 and fp16 queries a
    weight times its value's scale is rounded to fp16 once, which puts fp16 results
    up to 1.4 times as far off as their own rounding does (bf16: 1.01).

    Pages that no row sees any more may be gone from the table (any id).
    ``block_table_host`` is the host's copy of the table, by which the pages are
    checked; without it the table is copied from the device and waited for.  The
    lengths are host values that travel with the launches: a call captured in a
    graph replays the lengths it was captured with.

    ``query`` may have rows behind the last request's (a padded batch), and its
    rows may lie apart (a view of a fused projection); rows of ``out`` behind the
    last request's stay as they were, zeros in a fresh one.  bf16, fp16 or fp32
    queries, head sizes up to 512.
    """
    nb, bs, kvh, d, group, codes = _check_cache(_ATTENTION, k_data, k_scale, v_data, v_scale)
    if query.dim() != 3 or query.shape[2] != d:
        raise RuntimeError(
            f"{_ATTENTION}: query must be [tokens, heads, {d}], got {tuple(query.shape)}.")
    tokens, hq = query.shape[:2]
    dtype = _native.dtype_code(query.dtype)
    if kvh == 0 or hq == 0 or hq % kvh:
        raise RuntimeError(f"{_ATTENTION}: {hq} query heads over {kvh} kv heads.")
    if not 0 < scale < float("inf"):
        raise RuntimeError(f"{_ATTENTION}: scale must be positive, got {scale}.")
    if window is not None and window < 1:
        raise RuntimeError(f"{_ATTENTION}: window must be at least 1, got {window}.")
    if sinks < 0:
        raise RuntimeError(f"{_ATTENTION}: sinks must not be negative, got {sinks}.")
    lens, totals = _lengths(_ATTENTION, seq_lens, "seq_lens")
    news, counts = _lengths(_ATTENTION, query_lens, "query_lens")
    batch = len(totals)
    if len(counts) != batch:
        raise RuntimeError(f"{_ATTENTION}: {len(counts)} query_lens for {batch} seq_lens.")
    rows = sum(counts)
    if rows > tokens:
        raise RuntimeError(f"{_ATTENTION}: query_lens sum to {rows}, the query has {tokens} rows.")
    _check_devices(_ATTENTION, k_data, query=query, block_table=block_table)
    if out is not None:
        if out.shape != query.shape:
            raise RuntimeError(
                f"{_ATTENTION}: out {tuple(out.shape)} does not match query {tuple(query.shape)}.")
        _check_devices(_ATTENTION, k_data, out=out)
    win, sinks = 0 if window is None else min(int(window), _MOST), min(int(sinks), _MOST)
    table = _checked_table(_ATTENTION, block_table, block_table_host, totals, lens, news, nb, bs,
                           win, sinks)
    width = table.shape[1]
    # straight into `out` unless it is laid out otherwise or is the query's own memory
    direct = out is None or (
        out.is_contiguous() and out.dtype == query.dtype
        and out.untyped_storage().data_ptr() != query.untyped_storage().data_ptr())
    if rows:
        _native.require_gpu_tensors(_ATTENTION, query, k_data)
    q, q_stride = _rows(query)
    result = out if out is not None and direct else torch.empty(
        query.shape, dtype=q.dtype, device=q.device)
    if rows < tokens and out is None:
        result[rows:].zero_()
    if rows == 0:
        return result if out is None else out
    lib = _native.lib()
    with _on_device(k_data):
        nbytes = lib.kvq_block8_attn_workspace_bytes(
            lens, news, batch, dtype, hq, kvh, d, bs, group, codes, win, sinks)
        _native.check(nbytes if nbytes < 0 else 0, "kvq_block8_attn_workspace_bytes")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        rc = lib.kvq_block8_attn(
            q.data_ptr(), dtype, q_stride, lens, news, batch, hq, kvh, d, scale, win, sinks,
            codes, k_data.data_ptr(), k_scale.data_ptr(), v_data.data_ptr(), v_scale.data_ptr(), nb,
            bs, group, table.data_ptr(), _native.index_code(table.dtype), width, _native.ptr(ws),
            nbytes, result.data_ptr(), _native.stream_of(k_data),
        )
    _native.check(rc, "kvq_block8_attn")
    if not direct:
        out[:rows].copy_(result[:rows])
        return out
    return result


def _checked_table(what, block_table, block_table_host, totals, lens, news, nb, bs, window, sinks):
    """The device's rows of the table, its pages checked by the host's copy."""
    table, host = _table(block_table, block_table_host, len(totals))
    width = table.shape[1]
    bad = _native.lib().kvq_fp8_pth_window_check(
        host.ctypes.data, 1, width, lens, news, len(totals), nb, bs, window, sinks)
    if bad == _native.KVQ_ERR_CAPACITY:
        raise RuntimeError(
            f"{what}: block_table does not cover the longest sequence: "
            f"max_seq_len={max(totals)}, max_blocks={width}, block_size={bs}."
        )
    if bad > 0:
        raise RuntimeError(
            f"{what}: block_table has a block id outside the cache among the pages that request "
            f"{bad - 1} sees."
        )
    _native.check(bad, what)
    return table


__all__ = ["block8_attention", "block8_store"]
