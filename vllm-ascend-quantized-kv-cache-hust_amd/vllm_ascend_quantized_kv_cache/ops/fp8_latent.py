# SPDX-License-Identifier: Apache-2.0
"""A paged E4M3 cache of latent rows that all heads share (``kvq_fp8_latent_*``):
the store, with the position rotation applied on the way.

A token keeps one latent row of ``R`` dims as E4M3 codes ``data [NB, Bs, R]`` (uint8)
with a scale ``scale [NB, Bs, 1]`` fp32, the quantization of
``pkg/methods/fp8_per_token_head/semantics.py:52-61``, and a rotated position part
``rope [NB, Bs, P]`` in the activation type.  The reference has no counterpart.
"""

from __future__ import annotations

import torch

from . import _native
from .fp8_rotary import _check_devices, _check_query, _check_rotation, _same_view, _storage
from .fp8_window import _on_device

_STORE = "fp8_latent_store"


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
    tokens = latent.shape[0]
    if latent.dim() != 2 or latent.shape[1] != rank or part.shape != (tokens, dims):
        raise RuntimeError(
            f"{_STORE}: latent and part must be [tokens, {rank}] and [tokens, {dims}], got "
            f"{tuple(latent.shape)} and {tuple(part.shape)}."
        )
    dtype = _native.dtype_code(latent.dtype)
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
        fits = out_query is not None and out_query.stride(2) == 1 and (
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


__all__ = ["fp8_latent_store"]
