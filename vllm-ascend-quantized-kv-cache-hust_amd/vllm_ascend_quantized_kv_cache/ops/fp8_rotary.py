# SPDX-License-Identifier: Apache-2.0
"""The fp8_per_token_head store with the position rotation applied on the way
(``kvq_fp8_pth_rotary_store``): one launch takes a step's queries, keys and
values as the projection leaves them, rotates queries and keys, and stores keys
and values as ``fp8_per_token_head_store`` would store the rotated rows.

Beside ``fp8_ops``: the same pages, scales and slots, the quantization of
``pkg/methods/fp8_per_token_head/semantics.py:52-61`` of rows that were not
rounded to the activation type in between.  The reference rotates in the host's
own kernel.
"""

from __future__ import annotations

import torch

from . import _native
from .fp8_ops import validate_store_args
from .fp8_window import _on_device

_STORE = "fp8_per_token_head_rotary_store"


def _check_rotation(what: str, positions, cos_sin, interleaved, tokens: int, width: int, like):
    """(position type, table type, rows of the table, rotated dims) of a call."""
    if positions is None or cos_sin is None:
        raise RuntimeError(f"{what}: a rotation needs positions and cos_sin.")
    if positions.shape != (tokens,):
        raise RuntimeError(
            f"{what}: positions must be 1D of {tokens} tokens, got {tuple(positions.shape)}.")
    shape = cos_sin.shape
    if len(shape) != 2 or shape[0] == 0 or not cos_sin.is_contiguous():
        raise RuntimeError(
            f"{what}: cos_sin must be contiguous [positions, rotated dims], got {tuple(shape)}.")
    rot = shape[1]
    if rot == 0 or rot % 2 or rot > width:
        raise RuntimeError(f"{what}: cos_sin rotates {rot} dims of {width}; an even number of them.")
    _check_devices(what, like, positions=positions, cos_sin=cos_sin)
    return (_native.index_code(positions.dtype), _native.dtype_code(cos_sin.dtype),
            shape[0], rot)


def _check_devices(what: str, like, **tensors) -> None:
    device = like.device
    for name, t in tensors.items():
        if t.device != device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the rows on {device}.")


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` [tokens, heads, dims] with its heads and dims in one run, copied if need be, and the
    stride of its tokens."""
    tokens, heads, dims = t.shape
    token, head, dim = t.stride()
    run = heads * dims
    if dim != 1 or (heads > 1 and head != dims) or (tokens > 1 and token < run):
        return t.contiguous(), run
    return t, token if tokens > 1 else run


def _token_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def _storage(t: torch.Tensor) -> int:
    return t.untyped_storage().data_ptr()


def _check_query(what: str, query, out_query, tokens: int, width: int, like) -> None:
    dtype, device = like.dtype, like.device
    for name, t in (("query", query), ("out_query", out_query)):
        if t is None:
            continue
        shape = t.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != width or shape[1] == 0:
            raise RuntimeError(
                f"{what}: {name} must be [{tokens}, heads, {width}], got {tuple(shape)}.")
        if t.dtype != dtype:
            raise RuntimeError(f"{what}: {name} is {t.dtype}, the rows are {dtype}.")
        if t.device != device:
            raise RuntimeError(f"{what}: {name} is on {t.device}, the rows on {device}.")
    if out_query is not None and out_query.shape != query.shape:
        raise RuntimeError(
            f"{what}: out_query {tuple(out_query.shape)} does not match query {tuple(query.shape)}.")


def _target(query, out_query, others) -> torch.Tensor:
    """Where the launch writes rotated queries: ``out_query`` where its rows are laid out for it
    and it is the query itself or memory of its own, else a fresh tensor."""
    if out_query is not None:
        strides, (tokens, heads, dims) = out_query.stride(), out_query.shape
        plain = strides[2] == 1 and (heads == 1 or strides[1] == dims) and (
            tokens == 1 or strides[0] >= heads * dims)
        if plain and (_same_view(out_query, query)
                      or all(_storage(out_query) != _storage(t) for t in (query, *others))):
            return out_query
    return torch.empty(query.shape, dtype=query.dtype, device=query.device)


def fp8_per_token_head_rotary_store(
    query: torch.Tensor | None,
    key: torch.Tensor,
    value: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_data: torch.Tensor,
    k_scale: torch.Tensor,
    v_data: torch.Tensor,
    v_scale: torch.Tensor,
    *,
    interleaved: bool = False,
    out_query: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Rotate ``query [T, Hq, D]`` and ``key [T, KVH, D]`` to ``positions [T]`` and
    write the rotated keys and the values into the paged E4M3 cache by slot.

    ``cos_sin [P, rot]`` holds the cosines, then the sines, of each position
    (``rot / 2`` of either); ``rot <= D``, dims behind it stay.  Pairs are dims
    ``i`` and ``i + rot / 2``, or neighbours where ``interleaved``.  The rotation
    is fp32; keys are quantized without a rounding in between, queries rounded
    once.  Returns the rotated queries: ``out_query``, which may be ``query``
    itself, or a fresh tensor; None without queries.

    Caches and slots are those of ``fp8_per_token_head_store``: rows with
    negative slots, or slots outside the cache, are padding and not stored, nor
    are rows whose position is outside the table (its rotated queries are NaN).
    A slot is given once.  A row that is not finite reads back as NaN.  bf16,
    fp16 or fp32 rows, which may lie apart (views of a fused projection).
    """
    if key.dim() != 3 or value.dim() != 3:
        raise RuntimeError(
            f"{_STORE}: key and value must be [tokens, heads, dims], got {tuple(key.shape)} and "
            f"{tuple(value.shape)}.")
    validate_store_args(key, value, slot_mapping, k_data, k_scale, v_data, v_scale)
    tokens, kvh, d = key.shape
    dtype = _native.dtype_code(key.dtype)
    if value.dtype != key.dtype:
        raise RuntimeError(f"{_STORE}: value is {value.dtype}, key {key.dtype}.")
    pos_type, table_type, table_rows, rot = _check_rotation(
        _STORE, positions, cos_sin, interleaved, tokens, d, key)
    _check_devices(_STORE, key, value=value, slot_mapping=slot_mapping)
    if query is not None:
        _check_query(_STORE, query, out_query, tokens, d, key)
    elif out_query is not None:
        raise RuntimeError(f"{_STORE}: out_query needs query.")
    if tokens == 0 or kvh == 0:
        if query is None or tokens == 0:
            return query if out_query is None else out_query
        raise RuntimeError(f"{_STORE}: keys and values have no heads.")
    _native.require_gpu_tensors(_STORE, key)
    k, k_stride = _rows(key)
    v, v_stride = _rows(value)
    q, q_stride, target = None, 0, None
    if query is not None:
        q, q_stride = _rows(query)
        target = _target(query, out_query, (key, value))
    slots, places = slot_mapping.contiguous(), positions.contiguous()
    with _on_device(k_data):
        rc = _native.lib().kvq_fp8_pth_rotary_store(
            _native.ptr(q), q_stride, _native.ptr(target),
            0 if q is None else _token_stride(target), k.data_ptr(), k_stride, v.data_ptr(),
            v_stride, dtype, places.data_ptr(), pos_type, cos_sin.data_ptr(), table_type,
            table_rows, rot, 1 if interleaved else 0, slots.data_ptr(),
            _native.index_code(slots.dtype), tokens, 0 if q is None else q.shape[1], kvh, d,
            k_data.data_ptr(), k_scale.data_ptr(), v_data.data_ptr(), v_scale.data_ptr(),
            k_data.shape[0], k_data.shape[1], _native.stream_of(k_data),
        )
    _native.check(rc, "kvq_fp8_pth_rotary_store")
    if out_query is not None and target is not out_query:
        out_query.copy_(target)
        return out_query
    return target


__all__ = ["fp8_per_token_head_rotary_store"]
