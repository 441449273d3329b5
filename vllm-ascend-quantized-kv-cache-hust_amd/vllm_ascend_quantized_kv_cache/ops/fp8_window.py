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
from collections.abc import Sequence

import numpy as np
import torch

from . import _native
from .fp8_ops import _check_contiguous, _check_same_device

_ATTENTION = "fp8_per_token_head_window_attention"
_EVICT = "fp8_per_token_head_evict"


def _on_device(t: torch.Tensor):
    """Launches go to ``t``'s device, whichever is current."""
    if t.get_device() == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _check_cache(k_data, k_scale, v_data, v_scale) -> None:
    if k_data.dim() != 4 or k_data.dtype is not torch.uint8 or v_data.dtype is not torch.uint8:
        raise RuntimeError(
            "fp8_per_token_head data caches must be uint8 [NB, Bs, KVH, D], got "
            f"{tuple(k_data.shape)} / {k_data.dtype} and {v_data.dtype}."
        )
    nb, bs, kvh, _ = k_data.shape
    if v_data.shape != k_data.shape or k_scale.shape != (nb, bs, kvh, 1) or (
            v_scale.shape != k_scale.shape):
        raise RuntimeError(
            "fp8_per_token_head cache views disagree: "
            f"k_data {tuple(k_data.shape)}, k_scale {tuple(k_scale.shape)}, "
            f"v_data {tuple(v_data.shape)}, v_scale {tuple(v_scale.shape)}."
        )
    if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
        raise RuntimeError(
            f"fp8_per_token_head scale caches must be float32, got {k_scale.dtype} and "
            f"{v_scale.dtype}."
        )
    for name, t in (("key data", k_data), ("key scale", k_scale), ("value data", v_data),
                    ("value scale", v_scale)):
        _check_contiguous(name, t)
        _check_same_device(name, t, k_data)


def _lengths(what: str, values, name: str) -> np.ndarray:
    out = np.array([int(n) for n in values], dtype=np.int64)
    if out.size and int(out.min()) < 0:
        raise RuntimeError(f"{what}: negative {name}.")
    return out


def _table(block_table, host, batch: int, name: str = "block_table"):
    """(device rows, the host's copy of them as a contiguous array)."""
    if block_table.dim() != 2 or block_table.shape[0] < batch:
        raise RuntimeError(
            f"fp8_per_token_head {name} must be 2D with a row per request, got "
            f"{tuple(block_table.shape)} for {batch} requests."
        )
    _native.index_code(block_table.dtype)
    table = block_table[:batch].contiguous()
    rows = host if host is not None else table.cpu().numpy()
    if isinstance(rows, torch.Tensor):
        rows = rows.cpu().numpy()
    rows = np.ascontiguousarray(rows, dtype=np.int64)
    rows = rows.reshape(rows.shape[0] if rows.ndim == 2 else -1, table.shape[1])[:batch]
    if rows.shape[0] != batch:
        raise RuntimeError(
            f"fp8_per_token_head {name}: the host's copy has {rows.shape[0]} rows for {batch} "
            "requests."
        )
    return table, rows


def _weight_rows(what: str, weights, out_weights, weight_rows, batch: int, longest: int, kvh: int,
                 like) -> tuple[torch.Tensor, np.ndarray]:
    target = weights if out_weights is None else out_weights
    for name, t in (("weights", weights), ("out_weights", target)):
        if t.dim() != 3 or t.dtype is not torch.float32 or t.shape[1] != kvh:
            raise RuntimeError(
                f"{what}: {name} must be float32 [rows, {kvh}, positions], got "
                f"{tuple(t.shape)} / {t.dtype}."
            )
        _check_contiguous(name, t)
        _check_same_device(name, t, like)
    if target.shape != weights.shape:
        raise RuntimeError(
            f"{what}: out_weights {tuple(target.shape)} does not match weights "
            f"{tuple(weights.shape)}."
        )
    if target is not weights and target.data_ptr() != weights.data_ptr():
        n = 4 * weights.numel()
        if abs(target.data_ptr() - weights.data_ptr()) < n:
            raise RuntimeError(f"{what}: out_weights overlaps weights.")
    rows = np.arange(batch, dtype=np.int64) if weight_rows is None else np.array(
        [int(r) for r in weight_rows], dtype=np.int64)
    if rows.shape[0] != batch:
        raise RuntimeError(f"{what}: {rows.shape[0]} weight_rows for {batch} requests.")
    if batch and (int(rows.min()) < 0 or int(rows.max()) >= weights.shape[0]
                  or len(set(rows.tolist())) != batch):
        raise RuntimeError(
            f"{what}: weight_rows must be distinct rows of the {weights.shape[0]} in weights, got "
            f"{rows.tolist()}."
        )
    if longest > weights.shape[2]:
        raise RuntimeError(
            f"{what}: weights hold {weights.shape[2]} positions, the longest request has {longest}."
        )
    return target, rows


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
    Pages that no row sees any more may be gone from the table (any id).
    Keys and values are ``code * scale``, not rounded to the query's type, so
    without a window the result is nearer to that definition than
    ``fp8_per_token_head_attention``'s, which attends to rounded rows.

    ``weights`` (fp32 ``[rows, KVH, positions]``, request ``b`` in row
    ``weight_rows[b]``, by default ``b``) are the running attention weights:
    every cached position gains the sum of its weights over the request's rows
    and the query heads of the kv head; the new rows' own positions start from
    nothing.  They are updated in place, or written to ``out_weights``.

    ``query`` may have rows behind the last request's (a padded batch), and its
    rows may lie apart (a view of a fused projection); rows of ``out`` behind
    the last request's stay as they were, zeros in a fresh one.  bf16, fp16 or
    fp32 queries, any head size of the cache.
    """
    _check_cache(k_data, k_scale, v_data, v_scale)
    nb, bs, kvh, d = k_data.shape
    if query.dim() != 3 or query.shape[2] != d:
        raise RuntimeError(
            f"{_ATTENTION}: query must be [tokens, heads, {d}], got {tuple(query.shape)}.")
    tokens, hq = query.shape[:2]
    dtype = _native.dtype_code(query.dtype)
    if kvh == 0 or hq == 0 or hq % kvh:
        raise RuntimeError(f"{_ATTENTION}: {hq} query heads over {kvh} kv heads.")
    if not scale > 0:
        raise RuntimeError(f"{_ATTENTION}: scale must be positive, got {scale}.")
    if window is not None and window < 1:
        raise RuntimeError(f"{_ATTENTION}: window must be at least 1, got {window}.")
    if sinks < 0:
        raise RuntimeError(f"{_ATTENTION}: sinks must not be negative, got {sinks}.")
    lens = _lengths(_ATTENTION, seq_lens, "seq_lens")
    news = _lengths(_ATTENTION, query_lens, "query_lens")
    batch = lens.shape[0]
    if news.shape[0] != batch:
        raise RuntimeError(f"{_ATTENTION}: {news.shape[0]} query_lens for {batch} seq_lens.")
    rows = int(news.sum())
    if rows > tokens:
        raise RuntimeError(f"{_ATTENTION}: query_lens sum to {rows}, the query has {tokens} rows.")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        if rows < tokens:
            out[rows:].zero_()
    elif out.shape != query.shape:
        raise RuntimeError(
            f"{_ATTENTION}: out {tuple(out.shape)} does not match query {tuple(query.shape)}.")
    longest = int(lens.max()) if batch else 0
    w_rows = target = None
    if weights is not None:
        target, w_rows = _weight_rows(_ATTENTION, weights, out_weights, weight_rows, batch, longest,
                                      kvh, k_data)
    elif out_weights is not None or weight_rows is not None:
        raise RuntimeError(f"{_ATTENTION}: out_weights and weight_rows need weights.")
    _check_same_device("query", query, k_data)
    _check_same_device("out", out, k_data)
    _check_same_device("block_table", block_table, k_data)
    table, host = _table(block_table, block_table_host, batch)
    lib = _native.lib()
    win = 0 if window is None else int(window)
    bad = int(lib.kvq_fp8_pth_window_check(
        host.ctypes.data, 1, table.shape[1], lens.ctypes.data, news.ctypes.data, batch, nb, bs, win,
        int(sinks)))
    if bad == _native.KVQ_ERR_CAPACITY:
        raise RuntimeError(
            "fp8_per_token_head block_table does not cover the longest sequence: "
            f"max_seq_len={longest}, max_blocks={table.shape[1]}, block_size={bs}."
        )
    if bad > 0:
        raise RuntimeError(
            f"fp8_per_token_head block_table has a block id outside the cache among the pages that "
            f"request {bad - 1} sees."
        )
    _native.check(bad, _ATTENTION)
    if rows == 0:
        return out
    _native.require_gpu_tensors(_ATTENTION, query, k_data, out)
    q = query
    if q.stride(2) != 1 or q.stride(1) != d or (tokens > 1 and q.stride(0) < hq * d):
        q = q.contiguous()
    # straight into `out` unless it is laid out otherwise or is the query's own memory
    direct = out.is_contiguous() and out.dtype == q.dtype and (
        out.untyped_storage().data_ptr() != q.untyped_storage().data_ptr())
    with _on_device(k_data):
        result = out if direct else torch.empty(query.shape, dtype=q.dtype, device=q.device)
        nbytes = int(lib.kvq_fp8_pth_window_attn_workspace_bytes(
            lens.ctypes.data, news.ctypes.data, batch, dtype, hq, kvh, d, bs, win, int(sinks),
            0 if target is None else 1))
        _native.check(nbytes if nbytes < 0 else 0, "kvq_fp8_pth_window_attn_workspace_bytes")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        rc = lib.kvq_fp8_pth_window_attn(
            q.data_ptr(), dtype, q.stride(0) if tokens > 1 else hq * d, lens.ctypes.data,
            news.ctypes.data, batch, hq, kvh, d, float(scale), win, int(sinks), k_data.data_ptr(),
            k_scale.data_ptr(), v_data.data_ptr(), v_scale.data_ptr(), nb, bs, table.data_ptr(),
            _native.index_code(table.dtype), table.shape[1],
            None if target is None else weights.data_ptr(), _native.ptr(target),
            None if w_rows is None else w_rows.ctypes.data,
            0 if target is None else weights.shape[2], _native.ptr(ws), nbytes, result.data_ptr(),
            _native.stream_of(k_data),
        )
    _native.check(rc, "kvq_fp8_pth_window_attn")
    if not direct:
        out[:rows].copy_(result[:rows])
    return out


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
    from with ``out_block_table``.
    """
    _check_cache(k_data, k_scale, v_data, v_scale)
    nb, bs, kvh, d = k_data.shape
    if kvh == 0 or d == 0:
        raise RuntimeError(f"{_EVICT}: an empty cache {tuple(k_data.shape)}.")
    if sinks < 0 or recent < 0:
        raise RuntimeError(f"{_EVICT}: sinks and recent must not be negative.")
    lens = _lengths(_EVICT, seq_lens, "seq_lens")
    batch = lens.shape[0]
    keeps = _lengths(_EVICT, [keep] * batch if isinstance(keep, (int, np.integer)) else keep, "keep")
    if keeps.shape[0] != batch:
        raise RuntimeError(f"{_EVICT}: {keeps.shape[0]} budgets for {batch} requests.")
    over = lens > keeps
    if batch and bool((over & (keeps < sinks + recent)).any()):
        raise RuntimeError(
            f"{_EVICT}: a budget under sinks + recent = {sinks + recent}: {keeps.tolist()}.")
    longest = int(lens.max()) if batch else 0
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
    bad = int(lib.kvq_fp8_pth_evict_check(
        host.ctypes.data, None if out_host is None else out_host.ctypes.data, 1, table.shape[1],
        0 if out_table is None else out_table.shape[1], lens.ctypes.data, keeps.ctypes.data, batch,
        nb, bs)) if batch else 0
    if bad == _native.KVQ_ERR_CAPACITY:
        raise RuntimeError(
            f"{_EVICT}: a block table does not cover its rows (block_size={bs}, longest={longest}).")
    if bad > 0:
        why = "outside the cache" if bad % 2 else "in use twice"
        raise RuntimeError(f"{_EVICT}: request {(bad - 1) // 2} has a page {why}.")
    _native.check(bad, _EVICT)
    new_lens = np.minimum(lens, keeps)
    width = int(new_lens.max()) if batch else 0
    _native.require_gpu_tensors(_EVICT, k_data, weights)
    with _on_device(k_data):
        kept = torch.empty((batch, kvh, width), dtype=torch.int32, device=k_data.device)
        rc = lib.kvq_fp8_pth_evict(
            k_data.data_ptr(), k_scale.data_ptr(), v_data.data_ptr(), v_scale.data_ptr(), nb, bs,
            kvh, d, table.data_ptr(), _native.ptr(out_table), _native.index_code(table.dtype),
            table.shape[1], 0 if out_table is None else out_table.shape[1], lens.ctypes.data,
            keeps.ctypes.data, batch, int(sinks), int(recent), weights.data_ptr(),
            target.data_ptr(), rows.ctypes.data, weights.shape[2], kept.data_ptr(), width,
            _native.stream_of(k_data),
        ) if width else 0
    _native.check(rc, "kvq_fp8_pth_evict")
    return new_lens.tolist(), kept


__all__ = ["fp8_per_token_head_evict", "fp8_per_token_head_window_attention"]
