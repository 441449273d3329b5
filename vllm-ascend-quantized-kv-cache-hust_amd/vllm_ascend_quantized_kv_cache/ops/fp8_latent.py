# SPDX-License-Identifier: Apache-2.0
"""A paged E4M3 cache of latent rows that all heads share (``kvq_fp8_latent_*``):
the store, with the position rotation applied on the way, and causal attention
straight over it, the up-projections absorbed.

A token keeps one latent row of ``R`` dims as E4M3 codes ``data [NB, Bs, R]`` (uint8)
with a scale ``scale [NB, Bs, 1]`` fp32, the quantization of
``pkg/methods/fp8_per_token_head/semantics.py:52-61``, and a rotated position part
``rope [NB, Bs, P]`` in the activation type.  The reference has no counterpart.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native
from .block8 import _checked_table
from .fp8_rotary import (
    _check_devices,
    _check_query,
    _check_rotation,
    _rows,
    _same_view,
    _storage,
)
from .fp8_window import _lengths, _on_device

_STORE = "fp8_latent_store"
_ATTENTION = "fp8_latent_attention"


def _check_cache(what: str, data, scale, rope):
    """(pages, positions a page, latent dims, dims of the position part)."""
    if data.dim() != 3 or data.dtype is not torch.uint8:
        raise RuntimeError(
            f"{what}: data must be uint8 [NB, Bs, R], got {tuple(data.shape)} / {data.dtype}.")
    nb, bs, rank = data.shape
    if scale.shape != (nb, bs, 1) or scale.dtype is not torch.float32:
        raise RuntimeError(
            f"{what}: scale must be float32 {(nb, bs, 1)}, got {tuple(scale.shape)} / {scale.dtype}.")
    if rope.dim() != 3 or rope.shape[:2] != (nb, bs):
        raise RuntimeError(f"{what}: rope must be [{nb}, {bs}, P], got {tuple(rope.shape)}.")
    _native.dtype_code(rope.dtype)
    for name, t in (("data", data), ("scale", scale), ("rope", rope)):
        if not t.is_contiguous():
            raise RuntimeError(f"{what}: {name} must be contiguous.")
        if t.device != data.device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, data on {data.device}.")
    return nb, bs, rank, rope.shape[2]


def _token_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [tokens, dims] with the dims of a row in one run, copied if need be."""
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        return t.contiguous()
    return t


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """(tokens', heads') of [tokens, heads, dims]."""
    return t.stride(0), t.stride(1)


def _apart(t: torch.Tensor) -> bool:
    """Whether the rows of [tokens, heads, dims] are runs that share no element."""
    (tokens, heads, dims), (token, head, dim) = t.shape, t.stride()
    if dim != 1 or min(token if tokens > 1 else dims, head if heads > 1 else dims) < dims:
        return False
    (n, near), (m, far) = sorted(((tokens, token), (heads, head)), key=lambda x: x[1])
    return n == 1 or m == 1 or far >= (n - 1) * near + dims


def fp8_latent_store(
    latent: torch.Tensor,
    part: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    slot_mapping: torch.Tensor,
    data: torch.Tensor,
    scale: torch.Tensor,
    rope: torch.Tensor,
    *,
    query: torch.Tensor | None = None,
    interleaved: bool = False,
    out_query: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write ``latent [T, R]`` rows as E4M3 codes, and their position part ``part
    [T, P]`` rotated to ``positions``, into the cache by slot; rotate ``query
    [T, H, P]``, the queries' position part, with them.

    ``cos_sin [N, P]`` holds the cosines, then the sines, of each position
    (``P / 2`` of either).  Pairs are dims ``i`` and ``i + P / 2``, or neighbours
    where ``interleaved``.  The rotation is fp32, rounded once to the rows' type,
    which is that of ``rope``.  Returns the rotated queries: ``out_query`` (the last
    dims of the absorbed queries, say; or ``query`` itself), or a fresh tensor;
    None without queries.

    Negative slots, and slots outside the cache, are padding and not stored, nor
    are rows whose position is outside the table (its rotated queries are NaN).
    A slot is given once.  A latent row that is not finite reads back as NaN.
    """
    nb, bs, rank, dims = _check_cache(_STORE, data, scale, rope)
    if latent.dim() != 2 or latent.shape[1] != rank or part.shape != (latent.shape[0], dims):
        raise RuntimeError(
            f"{_STORE}: latent and part must be [tokens, {rank}] and [tokens, {dims}], got "
            f"{tuple(latent.shape)} and {tuple(part.shape)}."
        )
    tokens, dtype = latent.shape[0], _native.dtype_code(latent.dtype)
    if part.dtype != latent.dtype or rope.dtype != latent.dtype:
        raise RuntimeError(
            f"{_STORE}: latent is {latent.dtype}, part {part.dtype}, rope {rope.dtype}.")
    if slot_mapping.shape != (tokens,):
        raise RuntimeError(
            f"{_STORE}: slot_mapping must be 1D of {tokens} slots, got {tuple(slot_mapping.shape)}.")
    slot_type = _native.index_code(slot_mapping.dtype)
    _check_devices(_STORE, latent, part=part, slot_mapping=slot_mapping, data=data)
    pos_type, table_type, table_rows, rot = _check_rotation(
        _STORE, positions, cos_sin, interleaved, tokens, dims, latent)
    if rot != dims:
        raise RuntimeError(f"{_STORE}: cos_sin rotates {rot} dims, the position part has {dims}.")
    if query is not None:
        _check_query(_STORE, query, out_query, tokens, dims, latent)
    elif out_query is not None:
        raise RuntimeError(f"{_STORE}: out_query needs query.")
    if tokens == 0:
        return query if out_query is None else out_query
    _native.require_gpu_tensors(_STORE, latent)
    rows, parts = _token_rows(latent), _token_rows(part)
    q = target = None
    if query is not None:
        q = query if query.stride(2) == 1 else query.contiguous()
        fits = out_query is not None and _apart(out_query) and (
            _same_view(out_query, query)
            or all(_storage(out_query) != _storage(t) for t in (query, latent, part)))
        target = out_query if fits else torch.empty(query.shape, dtype=query.dtype,
                                                    device=query.device)
    slots, places = slot_mapping.contiguous(), positions.contiguous()
    with _on_device(data):
        rc = _native.lib().kvq_fp8_latent_store(
            _native.ptr(q), *((0, 0) if q is None else _strides(q)), _native.ptr(target),
            *((0, 0) if q is None else _strides(target)), rows.data_ptr(),
            rows.stride(0) if tokens > 1 else rank, parts.data_ptr(),
            parts.stride(0) if tokens > 1 else dims, dtype, places.data_ptr(), pos_type,
            cos_sin.data_ptr(), table_type, table_rows, 1 if interleaved else 0, slots.data_ptr(),
            slot_type, tokens, 0 if q is None else q.shape[1], rank, dims, data.data_ptr(),
            scale.data_ptr(), rope.data_ptr(), nb, bs, _native.stream_of(data),
        )
    _native.check(rc, "kvq_fp8_latent_store")
    if out_query is not None and target is not out_query:
        out_query.copy_(target)
        return out_query
    return target


def fp8_latent_attention(
    query: torch.Tensor,
    data: torch.Tensor,
    scale: torch.Tensor,
    rope: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int],
    query_lens: Sequence[int],
    softmax_scale: float,
    *,
    out: torch.Tensor | None = None,
    block_table_host=None,
) -> torch.Tensor:
    """Causal attention of TND ``query [sum query_lens, H, R + P]`` over the latent
    rows, with the up-projections absorbed: ``[..., :R]`` is a head's query through
    its key up-projection, ``[..., R:]`` its rotated position part, and the result
    ``[.., H, R]`` is for the caller to take through the value up-projection.

    With ``c_j = code * scale`` of position ``j`` (not rounded to the query's type)
    and ``r_j`` its position part, a score is ``softmax_scale * (q[:R] . c_j + q[R:] .
    r_j)`` and a value is ``c_j``.  ``softmax_scale`` is that of the heads before
    absorption.  Each request's rows are its last ``query_lens[b]`` of
    ``seq_lens[b]`` cached positions (stored already); a row at position ``p`` sees
    ``j <= p``, one that sees nothing gives zeros.  Scales under 2^-90 may count as 0
    in the values; one that is not finite makes the rows that see it NaN.  Weights on
    the matrix units are rounded as in ``block8_attention``.

    ``block_table_host`` is the host's copy of the table, by which the pages are
    checked; without it the table is copied from the device and waited for.  The
    lengths are host values that travel with the launches: a call captured in a
    graph replays the lengths it was captured with.

    ``query`` may have rows behind the last request's (a padded batch), and its
    rows may lie apart; rows of ``out`` behind the last request's stay as they were,
    zeros in a fresh one.  Queries are of ``rope``'s type, ``R`` up to 512 and ``P`` up
    to 256; bf16 and fp16 with ``R`` 256 or 512, ``P`` 32 or 64 and pages of whole
    16-position groups run on the matrix units.
    """
    nb, bs, rank, dims = _check_cache(_ATTENTION, data, scale, rope)
    if query.dim() != 3 or query.shape[2] != rank + dims or query.shape[1] == 0:
        raise RuntimeError(
            f"{_ATTENTION}: query must be [tokens, heads, {rank + dims}], got "
            f"{tuple(query.shape)}.")
    tokens, heads = query.shape[:2]
    if query.dtype != rope.dtype:
        raise RuntimeError(f"{_ATTENTION}: query is {query.dtype}, rope {rope.dtype}.")
    dtype = _native.dtype_code(query.dtype)
    if not 0 < softmax_scale < float("inf"):
        raise RuntimeError(f"{_ATTENTION}: softmax_scale must be positive, got {softmax_scale}.")
    lens, totals = _lengths(_ATTENTION, seq_lens, "seq_lens")
    news, counts = _lengths(_ATTENTION, query_lens, "query_lens")
    batch = len(totals)
    if len(counts) != batch:
        raise RuntimeError(f"{_ATTENTION}: {len(counts)} query_lens for {batch} seq_lens.")
    rows = sum(counts)
    if rows > tokens:
        raise RuntimeError(f"{_ATTENTION}: query_lens sum to {rows}, the query has {tokens} rows.")
    _check_devices(_ATTENTION, data, query=query, block_table=block_table)
    shape = (tokens, heads, rank)
    if out is not None:
        if out.shape != shape:
            raise RuntimeError(f"{_ATTENTION}: out must be {shape}, got {tuple(out.shape)}.")
        _check_devices(_ATTENTION, data, out=out)
    table = _checked_table(_ATTENTION, block_table, block_table_host, totals, lens, news, nb, bs, 0, 0)
    # straight into `out` unless it is laid out otherwise or is the query's own memory
    direct = out is None or (out.is_contiguous() and out.dtype == query.dtype
                             and _storage(out) != _storage(query))
    if rows:
        _native.require_gpu_tensors(_ATTENTION, query, data)
    q, q_stride = _rows(query)
    result = out if out is not None and direct else torch.empty(
        shape, dtype=q.dtype, device=q.device)
    if rows < tokens and out is None:
        result[rows:].zero_()
    if rows == 0:
        return result if out is None else out
    lib = _native.lib()
    with _on_device(data):
        nbytes = lib.kvq_fp8_latent_attn_workspace_bytes(
            lens, news, batch, dtype, heads, rank, dims, bs)
        _native.check(nbytes if nbytes < 0 else 0, "kvq_fp8_latent_attn_workspace_bytes")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        rc = lib.kvq_fp8_latent_attn(
            q.data_ptr(), dtype, q_stride, lens, news, batch, heads, rank, dims,
            softmax_scale, data.data_ptr(), scale.data_ptr(), rope.data_ptr(), nb, bs,
            table.data_ptr(), _native.index_code(table.dtype), table.shape[1], _native.ptr(ws),
            nbytes, result.data_ptr(), _native.stream_of(data),
        )
    _native.check(rc, "kvq_fp8_latent_attn")
    if not direct:
        out[:rows].copy_(result[:rows])
        return out
    return result


__all__ = ["fp8_latent_attention", "fp8_latent_store"]
