# SPDX-License-Identifier: Apache-2.0
"""Inputs and 64-bit restatements for the tests of windowed attention, running
weights and eviction over the paged E4M3 cache."""

from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


class Cache:
    """Paged E4M3 rows behind a shuffled table, made from a seed."""

    def __init__(self, lens, kvh, d, bs, *, device="cpu", seed=0, index=torch.int32, spare=2,
                 value_spread=1.0, room=0):
        rng = np.random.default_rng(seed)
        width = max(1, max([-(-(n + room) // bs) for n in lens], default=1))
        nb = len(lens) * width + spare
        ids = rng.permutation(nb)[: len(lens) * width].reshape(len(lens), width)
        g = torch.Generator().manual_seed(seed)

        def side(x):
            scale = (x.abs().amax(-1, keepdim=True) / 448.0).clamp_min(1e-6)
            codes = (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            return (codes.view(nb, bs, kvh, d).to(device).contiguous(),
                    scale.view(nb, bs, kvh, 1).to(device).contiguous())

        k = torch.randn(nb * bs, kvh, d, generator=g) * torch.exp(
            0.5 * torch.randn(kvh, d, generator=g))
        v = torch.randn(nb * bs, kvh, d, generator=g) * torch.exp(
            value_spread * torch.randn(nb * bs, kvh, 1, generator=g))
        self.k, self.ks = side(k)
        self.v, self.vs = side(v)
        self.lens, self.kvh, self.d, self.bs, self.nb = list(lens), kvh, d, bs, nb
        self.host = ids.astype(np.int64)
        self.table = torch.from_numpy(self.host).to(device, index)

    def slots(self, b, positions):
        p = np.asarray(positions, dtype=np.int64)
        return self.host[b, p // self.bs] * self.bs + p % self.bs

    def rows(self, b, length):
        """64-bit ``[length, KVH, D]`` keys and values of request ``b``."""
        at = torch.from_numpy(self.slots(b, np.arange(length))).to(self.k.device)

        def side(codes, scales):
            x = codes.view(-1, self.kvh, self.d)[at].view(torch.float8_e4m3fn).double()
            return x * scales.view(-1, self.kvh, 1)[at].double()

        return side(self.k, self.ks), side(self.v, self.vs)

    def args(self):
        return (self.k, self.ks, self.v, self.vs, self.table)


def query(rows, hq, d, dtype, device, seed=1, size=1.5):
    g = torch.Generator().manual_seed(seed)
    return (size * torch.randn(rows, hq, d, generator=g)).to(dtype).to(device)


def attention64(q, cache, lens, news, scale, window=None, sinks=0):
    """(out, bound, weight sums ``[KVH, len]`` per request, and their bounds) in 64 bits.

    ``bound`` is what the kernels' arithmetic may be off per element beside the
    rounding of the result.  Scores: fp32 sums of D exact products, each step off by
    at most 2^-24 of the sum of magnitudes A, so a score by (D + 16) 2^-24 A, and a
    weight relatively by twice that (its own and the norm's).  exp2, the offset and
    the norm of n terms: (n + 200) 2^-24.  Probabilities times value scales go
    through the matrix units in 16 bits: 2^-11 relative, and 2^-24 of the row's
    largest where they are subnormal.
    """
    hq, d = q.shape[1:]
    kvh = cache.kvh
    rep = hq // kvh
    dev = q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    bound = torch.zeros_like(out)
    sums, sum_bounds = [], []
    row0 = 0
    for b, (length, n) in enumerate(zip(lens, news)):
        k, v = cache.rows(b, length)
        w = torch.zeros(kvh, length, dtype=torch.float64, device=dev)
        wb = torch.zeros_like(w)
        if n and length:
            pos = (length - n + torch.arange(n, device=dev))[:, None]
            j = torch.arange(length, device=dev)
            see = j <= pos
            if window is not None:
                see &= (j > pos - window) | (j < sinks)
            x = q[row0:row0 + n].double().view(n, kvh, rep, d).permute(1, 0, 2, 3)
            x = x.reshape(kvh, n * rep, d)
            kt = k.permute(1, 2, 0).contiguous()  # [KVH, D, L]
            s = torch.bmm(x, kt) * scale
            mask = see.repeat_interleave(rep, 0)[None]
            size = torch.bmm(x.abs(), kt.abs()) * scale
            a = torch.where(mask, size.nan_to_num(0.0, 0.0, 0.0), 0.0).amax(-1, keepdim=True)
            s = s.masked_fill(~mask, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
            p = torch.where(mask, p, torch.zeros_like(p))  # NaN only where it is seen
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l == 0, torch.ones_like(l), l)
            p = torch.where(mask, p, torch.zeros_like(p))  # (0 / NaN in a NaN row)
            vv = v.permute(1, 0, 2).contiguous()
            # a masked place adds nothing, whatever it holds
            seen_nan = torch.bmm(mask.expand(kvh, -1, -1).double(), vv.isnan().double()) > 0
            vz = torch.where(vv.isfinite(), vv, torch.zeros_like(vv))
            o = torch.bmm(p, vz)
            o = torch.where(seen_nan, torch.full_like(o, math.nan), o)
            off = 2 * (d + 16) * 2.0 ** -24 * a + (length + 200) * 2.0 ** -24
            peak = (p[..., None] * vz.abs().amax(-1)[:, None, :, None]).amax((2, 3))[..., None]
            ob = (off + 2.0 ** -11) * torch.bmm(p, vz.abs()) + length * 2.0 ** -24 * peak

            def rows(t):
                return t.view(kvh, n, rep, d).permute(1, 0, 2, 3).reshape(n, hq, d)

            out[row0:row0 + n], bound[row0:row0 + n] = rows(o), rows(ob)
            w, wb = p.sum(1), (p * off).sum(1)
        sums.append(w)
        # (and a weight under the smallest normal number of fp32 may come as zero)
        sum_bounds.append(wb + (n * rep + 8) * 2.0 ** -24 * w + n * rep * 2.0 ** -126)
        row0 += n
    return out, bound, sums, sum_bounds


def check_out(got, want, bound, dtype):
    """Every element within the result's half step and the arithmetic's bound."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    # the smallest steps of fp16 and fp32 are subnormal ones
    tiny = float(torch.finfo(dtype).smallest_normal) * HALF_STEP[dtype] * 2
    limit = HALF_STEP[dtype] * want.abs() + (1 + HALF_STEP[dtype]) * bound + tiny
    # past the type's range a result rounds to infinity: from half a step over its
    # largest value on (fp16: 65504 + 16), which the exact one is within `limit` of
    over = got.isinf()
    edge = float(torch.finfo(dtype).max) * (1 + HALF_STEP[dtype] / 2)
    assert bool((want.abs() + limit >= edge)[over].all())
    assert torch.equal(got[over].sign(), want[over].sign())
    ok &= ~over
    off = (got - want).abs()
    worst = (off - limit)[ok].max().item() if ok.any() else -1.0
    assert worst <= 0, f"{worst} past the bound, max off {off[ok].max().item()}"


def check_weights(before, after, sums, bounds, rows, lens, news):
    """Running weights: old positions gain, new ones start, the rest stay."""
    want = before.double().clone()
    limit = torch.zeros_like(want)
    for b, r in enumerate(rows):
        length, n = lens[b], news[b]
        if n == 0:
            continue
        first = max(length - n, 0)
        want[r, :, first:length] = 0.0
        want[r, :, :length] += sums[b]
        limit[r, :, :length] = bounds[b] + 2.0 ** -24 * want[r, :, :length].abs()
    off = (after.double() - want).abs()
    assert torch.equal(after.isnan(), want.isnan())
    ok = ~want.isnan()
    assert bool((off[ok] <= limit[ok]).all()), (off - limit)[ok].max().item()
    untouched = limit == 0
    assert torch.equal(after[untouched & ok], before[untouched & ok])


def kept_rows(weights, length, keep, sinks, recent):
    """Positions one kv head keeps of ``length`` with ``weights`` (numpy fp32)."""
    if length <= keep:
        return np.arange(length)
    middle = np.arange(sinks, length - recent)
    w = weights[middle].astype(np.float64) + 0.0
    w[np.isnan(w)] = np.inf
    nan_first = np.where(np.isnan(weights[middle]), 0, 1)
    order = middle[np.lexsort((middle, nan_first, -w))]
    chosen = order[: keep - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), chosen, np.arange(length - recent, length)]))
