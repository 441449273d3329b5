# SPDX-License-Identifier: Apache-2.0
"""Bounded contexts over the paged E4M3 cache (``kvq_fp8_pth_window_attn``,
``kvq_fp8_pth_evict``): attention of new rows through a sliding window with
sinks, the running attention weights of the cached positions, and eviction by
them.

Beside ``fp8_ops``: the same pages, scales and block tables.  The reference has
no counterpart (its fp8 scheme stops at the store); the rows attended to are the
values of ``pkg/methods/fp8_per_token_head/semantics.py:63-65``.

A serving loop that bounds its cache stores each step's rows
(``fp8_per_token_head_store``), attends with ``weights=`` and, when a request
outgrows its budget, evicts and goes on with the lengths that come back.

The lengths, and the checked page tables, are host values that travel with the
launches: a call captured in a graph replays the lengths it was captured with.
"""

from __future__ import annotations

import contextlib
import ctypes
from collections.abc import Sequence

import numpy as np
import torch

from . import _native
from .fp8_ops import _check_contiguous, _check_same_device

_ATTENTION = "fp8_per_token_head_window_attention"
_EVICT = "fp8_per_token_head_evict"
#: the most cached positions of a request (the library's limit); windows, sinks and
#: budgets past it are as good as it
_MOST = 0x7FFF0000


def _on_device(t: torch.Tensor):
    """Launches go to ``t``'s device, whichever is current."""
    if t.get_device() == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(t.device)


_HERE = contextlib.nullcontext()


def _check_cache(k_data, k_scale, v_data, v_scale) -> torch.Size:
    shape = k_data.shape
    if len(shape) != 4 or k_data.dtype is not torch.uint8 or v_data.dtype is not torch.uint8:
        raise RuntimeError(
            "fp8_per_token_head data caches must be uint8 [NB, Bs, KVH, D], got "
            f"{tuple(shape)} / {k_data.dtype} and {v_data.dtype}."
        )
    if v_data.shape != shape or k_scale.shape != (*shape[:3], 1) or v_scale.shape != k_scale.shape:
        raise RuntimeError(
            "fp8_per_token_head cache views disagree: "
            f"k_data {tuple(shape)}, k_scale {tuple(k_scale.shape)}, "
            f"v_data {tuple(v_data.shape)}, v_scale {tuple(v_scale.shape)}."
        )
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
        raise RuntimeError(
            f"fp8_per_token_head scale caches must be float32, got {k_scale.dtype} and "
            f"{v_scale.dtype}."
        )
    device = k_data.device
    for name, t in (("key data", k_data), ("key scale", k_scale), ("value data", v_data),
                    ("value scale", v_scale)):
        if not t.is_contiguous() or t.device != device:
            _check_contiguous(name, t)
            _check_same_device(name, t, k_data)
    return shape


def _lengths(what: str, values, name: str):
    """(int64 array for a call, the numbers)."""
    if not isinstance(values, (list, tuple)):
        values = [int(n) for n in values]
    try:
        out = (ctypes.c_int64 * len(values))(*values)
    except TypeError:  # numpy integers
        values = [int(n) for n in values]
        out = (ctypes.c_int64 * len(values))(*values)
    if values and min(values) < 0:
        raise RuntimeError(f"{what}: negative {name}.")
    if values and max(values) > _MOST:
        raise RuntimeError(f"{what}: {name} past {_MOST}: {max(values)}.")
    return out, values


def _table(block_table, host, batch: int, name: str = "block_table"):
    """(device rows, the host's copy of them as a contiguous int64 array)."""
    if block_table.dim() != 2 or block_table.shape[0] < batch:
        raise RuntimeError(
            f"fp8_per_token_head {name} must be 2D with a row per request, got "
            f"{tuple(block_table.shape)} for {batch} requests."
        )
    _native.index_code(block_table.dtype)
    # (rows behind the batch are not read)
    table = block_table if block_table.is_contiguous() else block_table.contiguous()
    rows = host if host is not None else table[:batch].cpu().numpy()
    if isinstance(rows, torch.Tensor):
        rows = rows.cpu().numpy()
    if not (isinstance(rows, np.ndarray) and rows.dtype == np.int64 and rows.flags.c_contiguous):
        rows = np.ascontiguousarray(rows, dtype=np.int64)
    width = table.shape[1]
    if rows.ndim != 2 or rows.shape[1] != width or rows.shape[0] < batch:
        raise RuntimeError(
            f"fp8_per_token_head {name}: the host's copy is {rows.shape}, the table "
            f"{tuple(block_table.shape)} for {batch} requests."
        )
    return table, rows


def _weight_rows(what: str, weights, out_weights, weight_rows, batch: int, longest: int, kvh: int,
                 like):
    """(where the weights go, their rows as an int64 array for a call)."""
    target = weights if out_weights is None else out_weights
    for name, t in (("weights", weights), ("out_weights", target)):
        if t.dim() != 3 or t.dtype is not torch.float32 or t.shape[1] != kvh:
            raise RuntimeError(
                f"{what}: {name} must be float32 [rows, {kvh}, positions], got "
                f"{tuple(t.shape)} / {t.dtype}."
            )
        _check_contiguous(name, t)
        _check_same_device(name, t, like)
    if target is not weights:
        if target.shape != weights.shape:
            raise RuntimeError(
                f"{what}: out_weights {tuple(target.shape)} does not match weights "
                f"{tuple(weights.shape)}."
            )
        apart = abs(target.data_ptr() - weights.data_ptr())
        if 0 < apart < 4 * weights.numel():
            raise RuntimeError(f"{what}: out_weights overlaps weights.")
    if weight_rows is None:
        rows = range(batch)
        array = (ctypes.c_int64 * batch)(*rows)
    else:
        array, rows = _lengths(what, weight_rows, "weight_rows")
        if len(rows) != batch:
            raise RuntimeError(f"{what}: {len(rows)} weight_rows for {batch} requests.")
    if batch and (max(rows) >= weights.shape[0]
                  or (weight_rows is not None and len(set(rows)) != batch)):
        raise RuntimeError(
            f"{what}: weight_rows must be distinct rows of the {weights.shape[0]} in weights, got "
            f"{list(rows)}."
        )
    if longest > weights.shape[2]:
        raise RuntimeError(
            f"{what}: weights hold {weights.shape[2]} positions, the longest request has {longest}."
        )
    return target, array


def fp8_per_token_head_window_attention(
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
    weights: torch.Tensor | None = None,
    out_weights: torch.Tensor | None = None,
    weight_rows: Sequence[int] | None = None,
    out: torch.Tensor | None = None,
    block_table_host=None,
) -> torch.Tensor:
    """Causal attention of TND ``query [sum query_lens, Hq, D]`` straight over the
    paged E4M3 rows, through an optional sliding window.

    Each request's rows are its last ``query_lens[b]`` of ``seq_lens[b]`` cached
    positions (their keys and values are stored already).  A row at position
    ``p`` sees positions ``j <= p``; with ``window``, of those the last
    ``window`` and the first ``sinks``.  A row that sees nothing gives zeros.
    Positions are places in the cache: after an eviction a window counts the rows
    that were kept, other ones for each kv head.
    Pages that no row sees any more may be gone from the table (any id).
    ``block_table_host`` is the host's copy of the table, by which the pages are
    checked; without it the table is copied from the device and waited for.
    Keys and values are ``code * scale``, whatever the scale's sign (value scales
    under 2^-90 may count as 0; one that is not finite leaves no finite number in
    the rows that see it), not rounded to the query's type, so without a window the result is nearer to that definition than
    ``fp8_per_token_head_attention``'s, which attends to rounded rows.

    ``weights`` (fp32 ``[rows, KVH, positions]``, request ``b`` in row
    ``weight_rows[b]``, by default ``b``) are the running attention weights:
    every cached position gains the sum of its weights over the request's rows
    and the query heads of the kv head; the new rows' own positions start from
    nothing.  They are updated in place, or written to ``out_weights``, where a
    request without new rows has its old ones; positions past a request's length
    and rows of other requests stay as they were there.

    ``query`` may have rows behind the last request's (a padded batch), and its
    rows may lie apart (a view of a fused projection); rows of ``out`` behind
    the last request's stay as they were, zeros in a fresh one.  bf16, fp16 or
    fp32 queries, head sizes up to 512.
    """
    nb, bs, kvh, d = _check_cache(k_data, k_scale, v_data, v_scale)
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
    longest = max(totals, default=0)
    w_rows = target = None
    if weights is not None:
        target, w_rows = _weight_rows(_ATTENTION, weights, out_weights, weight_rows, batch, longest,
                                      kvh, k_data)
    elif out_weights is not None or weight_rows is not None:
        raise RuntimeError(f"{_ATTENTION}: out_weights and weight_rows need weights.")
    _check_same_device("query", query, k_data)
    _check_same_device("block_table", block_table, k_data)
    if out is not None:
        if out.shape != query.shape:
            raise RuntimeError(
                f"{_ATTENTION}: out {tuple(out.shape)} does not match query {tuple(query.shape)}.")
        _check_same_device("out", out, k_data)
    table, host = _table(block_table, block_table_host, batch)
    width = table.shape[1]
    lib = _native.lib()
    win, sinks = 0 if window is None else min(int(window), _MOST), min(int(sinks), _MOST)
    bad = lib.kvq_fp8_pth_window_check(host.ctypes.data, 1, width, lens, news, batch, nb, bs, win,
                                       sinks)
    if bad == _native.KVQ_ERR_CAPACITY:
        raise RuntimeError(
            "fp8_per_token_head block_table does not cover the longest sequence: "
            f"max_seq_len={longest}, max_blocks={width}, block_size={bs}."
        )
    if bad > 0:
        raise RuntimeError(
            f"fp8_per_token_head block_table has a block id outside the cache among the pages that "
            f"request {bad - 1} sees."
        )
    _native.check(bad, _ATTENTION)
    # straight into `out` unless it is laid out otherwise or is the query's own memory
    direct = out is None or (
        out.is_contiguous() and out.dtype == query.dtype
        and out.untyped_storage().data_ptr() != query.untyped_storage().data_ptr())
    # weights that go to another tensor go there of requests without rows too
    apart = target is not None and longest > 0 and target.data_ptr() != weights.data_ptr()
    if rows or apart:
        _native.require_gpu_tensors(_ATTENTION, query, k_data)
    q = query
    strides = q.stride()
    if strides[2] != 1 or strides[1] != d or (tokens > 1 and strides[0] < hq * d):
        q = q.contiguous()
        strides = q.stride()
    result = torch.empty(query.shape, dtype=q.dtype, device=q.device) if (
        out is None or not direct) else out
    if rows < tokens and out is None:
        result[rows:].zero_()
    if rows == 0 and not apart:
        return result if out is None else out
    with _on_device(k_data):
        nbytes = lib.kvq_fp8_pth_window_attn_workspace_bytes(
            lens, news, batch, dtype, hq, kvh, d, bs, win, sinks, 0 if target is None else 1)
        _native.check(nbytes if nbytes < 0 else 0, "kvq_fp8_pth_window_attn_workspace_bytes")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        rc = lib.kvq_fp8_pth_window_attn(
            q.data_ptr(), dtype, strides[0] if tokens > 1 else hq * d, lens, news, batch, hq, kvh,
            d, scale, win, sinks, k_data.data_ptr(), k_scale.data_ptr(), v_data.data_ptr(),
            v_scale.data_ptr(), nb, bs, table.data_ptr(), _native.index_code(table.dtype), width,
            None if target is None else weights.data_ptr(), _native.ptr(target), w_rows,
            0 if target is None else weights.shape[2], _native.ptr(ws), nbytes, result.data_ptr(),
            _native.stream_of(k_data),
        )
    _native.check(rc, "kvq_fp8_pth_window_attn")
    if not direct:
        out[:rows].copy_(result[:rows])
        return out
    return result


def fp8_per_token_head_evict(
    k_data: torch.Tensor,
    k_scale: torch.Tensor,
    v_data: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int],
    weights: torch.Tensor,
    keep: int | Sequence[int],
    *,
    sinks: int = 0,
    recent: int = 0,
    weight_rows: Sequence[int] | None = None,
    out_block_table: torch.Tensor | None = None,
    out_weights: torch.Tensor | None = None,
    block_table_host=None,
    out_block_table_host=None,
) -> tuple[list[int], torch.Tensor]:
    """Shrinks requests of more than ``keep`` cached rows to that many.

    Such a request keeps, per kv head, its first ``sinks`` rows, its last
    ``recent`` and the heaviest of the rest by ``weights`` (as
    ``fp8_per_token_head_window_attention`` keeps them; of equal weights the
    earliest, NaN before all), in the order of their positions; others keep all.
    Codes, scales and weights move to the front of the request's own pages and
    weights row, or to ``out_block_table``'s pages and to ``out_weights``, where
    given (requests that keep all are copied there too).

    Returns the new lengths (host) and the positions kept, int32 ``[B, KVH, max
    new length]`` with -1 behind a request's rows.  Rows behind the new lengths
    stay as they were.  A page that rows move within or to may belong to one
    request only; pages shared between requests (a common prefix) can be read
    from with ``out_block_table``.  The tables' host copies are as in
    ``fp8_per_token_head_window_attention``; positions, and so windows, count the
    rows kept from here on.
    """
    nb, bs, kvh, d = _check_cache(k_data, k_scale, v_data, v_scale)
    if kvh == 0 or d == 0:
        raise RuntimeError(f"{_EVICT}: an empty cache {tuple(k_data.shape)}.")
    if sinks < 0 or recent < 0:
        raise RuntimeError(f"{_EVICT}: sinks and recent must not be negative.")
    lens, totals = _lengths(_EVICT, seq_lens, "seq_lens")
    batch = len(totals)
    longest = max(totals, default=0)
    stay = sinks + recent
    if isinstance(keep, (int, np.integer)):
        keep = min(int(keep), _MOST)
        if keep < 0:
            raise RuntimeError(f"{_EVICT}: negative keep.")
        keeps = (ctypes.c_int64 * batch)(*[keep] * batch)
        new_lens = [n if n < keep else keep for n in totals]
        short = keep < stay and longest > keep
    else:
        keeps, budgets = _lengths(_EVICT, [min(int(k), _MOST) for k in keep], "keep")
        if len(budgets) != batch:
            raise RuntimeError(f"{_EVICT}: {len(budgets)} budgets for {batch} requests.")
        new_lens = [n if n < k else k for n, k in zip(totals, budgets)]
        short = any(k < stay and n > k for n, k in zip(totals, budgets))
    if short:
        raise RuntimeError(f"{_EVICT}: a budget under sinks + recent = {stay}: {keep}.")
    target, rows = _weight_rows(_EVICT, weights, out_weights, weight_rows, batch, longest, kvh,
                                k_data)
    _check_same_device("block_table", block_table, k_data)
    table, host = _table(block_table, block_table_host, batch)
    out_table = out_host = None
    if out_block_table is not None:
        _check_same_device("out_block_table", out_block_table, k_data)
        if out_block_table.dtype != block_table.dtype:
            raise RuntimeError(
                f"{_EVICT}: out_block_table is {out_block_table.dtype}, block_table "
                f"{block_table.dtype}."
            )
        out_table, out_host = _table(out_block_table, out_block_table_host, batch,
                                     "out_block_table")
    lib = _native.lib()
    width, out_width = table.shape[1], 0 if out_table is None else out_table.shape[1]
    bad = lib.kvq_fp8_pth_evict_check(
        host.ctypes.data, None if out_host is None else out_host.ctypes.data, 1, width, out_width,
        lens, keeps, batch, nb, bs) if batch else 0
    if bad == _native.KVQ_ERR_CAPACITY:
        raise RuntimeError(
            f"{_EVICT}: a block table does not cover its rows (block_size={bs}, longest={longest}).")
    if bad > 0:
        why = "outside the cache" if bad % 2 else "in use twice"
        raise RuntimeError(f"{_EVICT}: request {(bad - 1) // 2} has a page {why}.")
    _native.check(bad, _EVICT)
    most = max(new_lens, default=0)
    _native.require_gpu_tensors(_EVICT, k_data)
    with _on_device(k_data):
        kept = torch.empty((batch, kvh, most), dtype=torch.int32, device=k_data.device)
        nbytes = lib.kvq_fp8_pth_evict_workspace_bytes(lens, keeps, batch, kvh)
        _native.check(nbytes if nbytes < 0 else 0, "kvq_fp8_pth_evict_workspace_bytes")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=k_data.device) if nbytes else None
        rc = lib.kvq_fp8_pth_evict(
            k_data.data_ptr(), k_scale.data_ptr(), v_data.data_ptr(), v_scale.data_ptr(), nb, bs,
            kvh, d, table.data_ptr(), _native.ptr(out_table), _native.index_code(table.dtype),
            width, out_width, lens, keeps, batch, min(sinks, _MOST), min(recent, _MOST), weights.data_ptr(),
            target.data_ptr(), rows, weights.shape[2], kept.data_ptr(), most, _native.ptr(ws),
            nbytes, _native.stream_of(k_data),
        ) if most else 0
    _native.check(rc, "kvq_fp8_pth_evict")
    return new_lens, kept


__all__ = ["fp8_per_token_head_evict", "fp8_per_token_head_window_attention"]
