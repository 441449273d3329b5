# SPDX-License-Identifier: Apache-2.0
"""Bounded-memory serving over the paged E4M3 cache, as measurable calls.

``attend``  attention of each request's new rows (one token to a whole chunk)
            over its paged codes, with a sliding window and sinks or without
``weigh``   the same, adding every cached position's attention weight to the
            request's running weights
``evict``   the heaviest rows of each request and kv head, compacted into fresh
            pages

A state is one layer's view at that moment: the E4M3 pages behind a shuffled
page table with the host's copy of it, the step's query rows, the running
weights.  With ``own`` the calls are the package's; without, plain torch.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PACKAGE = Path(__file__).resolve().parents[1] / "vllm-ascend-quantized-kv-cache-hust_amd"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one request's next token on one rank of a TP-4 split: latency alone
        dict(name="attend_one_token", kind="attend", batch=1, low=600, high=600, new_low=1,
             new_high=1, heads=10, kv_heads=2, head=128, block=128, window=0, sinks=0,
             dtype="bf16", lens=1),
        # a decode batch of long contexts read through a 4096-token window with 4
        # sinks (32 query / 8 kv heads)
        dict(name="attend_decode_window", kind="attend", batch=64, low=4096, high=16384,
             new_low=1, new_high=1, heads=32, kv_heads=8, head=128, block=128, window=4096,
             sinks=4, dtype="bf16", lens=2),
        # the headline decode batch (40 query / 8 kv heads), everything visible
        dict(name="attend_decode_full", kind="attend", batch=32, low=2048, high=16384,
             new_low=1, new_high=1, heads=40, kv_heads=8, head=128, block=128, window=0,
             sinks=0, dtype="bf16", lens=3),
        # a prefill chunk of 2048 tokens over a long prompt's pages, full causal
        dict(name="attend_chunk_full", kind="attend", batch=4, low=10240, high=10240,
             new_low=2048, new_high=2048, heads=40, kv_heads=8, head=128, block=128, window=0,
             sinks=0, dtype="bf16", lens=4),
        # the same step of a sliding-window layer at head size 256 (8 query heads on
        # one kv head per rank), ragged, fp16
        dict(name="attend_chunk_window_256", kind="attend", batch=6, low=3001, high=9000,
             new_low=200, new_high=1500, heads=8, kv_heads=1, head=256, block=128,
             window=2048, sinks=16, dtype="fp16", lens=5),
        # a mixed step: requests with anything from one to a few hundred new rows
        # over short histories, odd sizes, head size 64, small pages
        dict(name="attend_mixed_64", kind="attend", batch=23, low=333, high=3000, new_low=1,
             new_high=411, heads=14, kv_heads=2, head=64, block=16, window=1000, sinks=3,
             dtype="bf16", lens=6),
        # a decode batch that keeps its heavy-hitter weights up to date
        dict(name="weigh_decode", kind="weigh", batch=32, low=2048, high=16384, new_low=1,
             new_high=1, heads=32, kv_heads=8, head=128, block=128, window=0, sinks=0,
             dtype="bf16", lens=7),
        # whole prompts of moderate length with their weights: what a cache is
        # compressed by after prefill
        dict(name="weigh_prefill", kind="weigh", batch=3, low=1500, high=4100, new_low=4100,
             new_high=4100, heads=32, kv_heads=8, head=128, block=128, window=0, sinks=0,
             dtype="bf16", lens=8),
        # two short requests with a few new rows each (an observation window)
        dict(name="weigh_small", kind="weigh", batch=2, low=300, high=777, new_low=5,
             new_high=8, heads=14, kv_heads=2, head=128, block=32, window=0, sinks=0,
             dtype="fp16", lens=9),
        # one short request back to its budget
        dict(name="evict_one", kind="evict", batch=1, low=1100, high=1100, kv_heads=2, head=128,
             block=128, keep=600, sinks=4, recent=64, lens=10),
        # a batch of long contexts compressed to a quarter or less
        dict(name="evict_batch", kind="evict", batch=32, low=4096, high=16384, kv_heads=8,
             head=128, block=128, keep=2048, sinks=4, recent=256, lens=11),
        # one very long context, half of it kept
        dict(name="evict_long", kind="evict", batch=1, low=100001, high=100001, kv_heads=8,
             head=128, block=128, keep=50000, sinks=16, recent=1024, lens=12),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "weigh", "weigh", "evict", "evict"])
    head = rng.choice([64, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8]) if head < 256 else rng.choice([1, 2])
    case = dict(kind=kind, kv_heads=kv_heads, head=head, block=rng.choice([16, 32, 64, 128, 128]),
                lens=rng.randrange(1 << 30))
    if kind == "evict":
        high = _spread(rng, 40, 100000)
        most = max(1, min(32, 1500000 // (high * kv_heads)))
        case.update(batch=_spread(rng, 1, most), high=high, low=rng.randint(max(1, high // 4), high))
        case["sinks"] = min(rng.choice([0, 1, 4, 16]), high // 8)
        case["recent"] = rng.randint(0, high // 8)
        case["keep"] = rng.randint(case["sinks"] + case["recent"] + 1, max(2, high * 3 // 4))
        return case
    case["heads"] = kv_heads * rng.choice([1, 2, 4, 5, 7, 8])
    case["dtype"] = rng.choice(["bf16", "fp16"])
    case["window"] = rng.choice([0, _spread(rng, 1, 8192)])
    case["sinks"] = rng.choice([0, 1, 4, 100]) if case["window"] else 0
    case["high"] = _spread(rng, 1, 16384)
    case["low"] = rng.randint(max(1, case["high"] // 4), case["high"])
    if rng.random() < 0.5:  # decode, or a few rows for every request
        case["new_low"] = case["new_high"] = rng.choice([1, 1, 1, 2, 5])
    else:
        case["new_high"] = _spread(rng, 1, min(2048, case["high"]))
        case["new_low"] = rng.randint(1, case["new_high"])
    rows = case["new_high"] * case["heads"] * case["high"]  # scores of a request
    most = min(64, 2000000000 // rows, 2000000 // (case["high"] * kv_heads))
    case["batch"] = _spread(rng, 1, max(1, most))
    return case


def _lengths(case):
    """(cached rows, new rows) of every request."""
    rng = random.Random(case["lens"])
    total = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    if case["kind"] == "evict":
        return total, [0] * len(total)
    new = [min(n, rng.randint(case["new_low"], case["new_high"])) for n in total]
    return total, new


def _seen(total, new, window, sinks):
    """(positions that some row sees, visible (row, position) pairs) of a request."""
    first = total - new
    if not window:
        return total, new * first + new * (new + 1) // 2
    pos = np.arange(first, total, dtype=np.int64)
    low = np.maximum(pos - window + 1, 0)
    pairs = int((pos + 1 - low + np.minimum(low, sinks)).sum())
    low0 = max(first - window + 1, 0)
    return total - low0 + min(sinks, low0), pairs


def work(case):
    total, new = _lengths(case)
    kvh, d = case["kv_heads"], case["head"]
    row = 2 * d + 8  # codes and scales of a cached row
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in total)
        return {"bytes": 4 * kvh * sum(total) + kept * kvh * (2 * row + 8), "flops": 0}
    seen = [_seen(t, n, case["window"], case["sinks"]) for t, n in zip(total, new)]
    cols = sum(s[0] for s in seen)
    moved = cols * kvh * row + 4 * sum(new) * case["heads"] * d
    if case["kind"] == "weigh":
        moved += 4 * kvh * (sum(total) + sum(t - n for t, n in zip(total, new)))
    return {"bytes": moved, "flops": 4 * d * case["heads"] * sum(s[1] for s in seen)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _quantize(x):
    """fp32 ``[T, KVH, D]`` -> (E4M3 codes as bytes, fp32 scales ``[T, KVH, 1]``)."""
    scale = (x.abs().amax(-1, keepdim=True) / 448.0).clamp_min(1e-6)
    return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    total, new = _lengths(case)
    kvh, d, bs = case["kv_heads"], case["head"], case["block"]
    batch = len(total)
    width = -(-max(total) // bs)
    blocks = batch * width
    order = list(range(blocks))
    rng.shuffle(order)
    host = np.array(order, dtype=np.int64).reshape(batch, width)
    fresh = 0
    if case["kind"] == "evict":  # the pages behind the history's, for the rows that stay
        out_width = -(-min(max(total), case["keep"]) // bs)
        fresh = batch * out_width
    pages = blocks + fresh
    data = torch.empty((2, pages, bs, kvh, d), dtype=torch.uint8, device=dev)
    scale = torch.empty((2, pages, bs, kvh, 1), dtype=torch.float32, device=dev)
    # keys with outlier channels; values whose rows differ in size
    channel = torch.exp(0.5 * torch.randn((kvh, d), generator=gen, device=dev))
    step = max(1, (1 << 26) // (bs * kvh * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn((n * bs, kvh, d), generator=gen, device=dev)
        c, s = _quantize(x * channel)
        data[0, p:p + n], scale[0, p:p + n] = c.view(n, bs, kvh, d), s.view(n, bs, kvh, 1)
        x = torch.randn((n * bs, kvh, d), generator=gen, device=dev)
        x *= torch.exp(torch.randn((n * bs, kvh, 1), generator=gen, device=dev))
        c, s = _quantize(x)
        data[1, p:p + n], scale[1, p:p + n] = c.view(n, bs, kvh, d), s.view(n, bs, kvh, 1)
    state = dict(
        kind=case["kind"], k=data[0], v=data[1], ks=scale[0], vs=scale[1], total=total, new=new,
        host=host, table=torch.from_numpy(host.astype(np.int32)).to(dev),
        lens=torch.tensor(total, device=dev), news=torch.tensor(new, device=dev),
        window=case.get("window") or None, sinks=case["sinks"], scale=d ** -0.5,
    )
    if case["kind"] == "evict":
        out = np.arange(blocks, pages, dtype=np.int64)
        rng.shuffle(out)
        out = out.reshape(batch, out_width)
        longest = max(total)
        # a heavy tail with many rows that nothing looked at (equal weights)
        w = torch.randn((batch, kvh, longest), generator=gen, device=dev)
        w = torch.where(w < -1.0, torch.zeros_like(w), torch.exp(2.0 * w))
        state.update(keep=case["keep"], recent=case["recent"], weights=w, blocks=blocks,
                     out_weights=torch.zeros_like(w), out_host=out,
                     out_table=torch.from_numpy(out.astype(np.int32)).to(dev))
        return state
    rows, heads = sum(new), case["heads"]
    q = torch.randn((rows, heads, d), generator=gen, device=dev)
    state["q"] = (1.5 * q).to(DTYPES[case["dtype"]])
    if case["kind"] == "weigh":
        slots = list(range(batch + 1))
        rng.shuffle(slots)
        w = torch.rand((batch + 1, kvh, max(total) + 37), generator=gen, device=dev)
        state.update(rows=slots[:batch], weights=w, out_weights=w.clone(),
                     row_ids=torch.tensor(slots[:batch], device=dev))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _package():
    if str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    from vllm_ascend_quantized_kv_cache.ops import fp8_window

    return fp8_window


def run(s):
    if own:
        ops = _package()
        if s["kind"] == "evict":
            new_lens, kept = ops.fp8_per_token_head_evict(
                s["k"], s["ks"], s["v"], s["vs"], s["table"], s["total"], s["weights"], s["keep"],
                sinks=s["sinks"], recent=s["recent"], out_block_table=s["out_table"],
                out_weights=s["out_weights"], block_table_host=s["host"],
                out_block_table_host=s["out_host"])
            return _evicted(s, kept)
        more = {}
        if s["kind"] == "weigh":
            more = dict(weights=s["weights"], out_weights=s["out_weights"], weight_rows=s["rows"])
        out = ops.fp8_per_token_head_window_attention(
            s["q"], s["k"], s["ks"], s["v"], s["vs"], s["table"], s["total"], s["new"], s["scale"],
            window=s["window"], sinks=s["sinks"], block_table_host=s["host"], **more)
        return (out, s["out_weights"]) if more else out
    return _plain_evict(s) if s["kind"] == "evict" else _plain_attend(s)


def _evicted(s, kept):
    """The positions kept, the fresh pages (codes as the values they stand for) and weights."""
    fresh = slice(s["blocks"], None)
    e4m3 = torch.float8_e4m3fn
    return (kept, s["k"][fresh].view(e4m3), s["ks"][fresh], s["v"][fresh].view(e4m3),
            s["vs"][fresh], s["out_weights"])


def _slots(table, positions, bs):
    return table[:, positions // bs].long() * bs + positions % bs


def _plain_attend(s):
    q, total, new = s["q"], s["lens"], s["news"]
    nb, bs, kvh, d = s["k"].shape
    batch, hq = len(s["total"]), q.shape[1]
    rep, longest, most = hq // kvh, max(s["total"]), max(s["new"])
    dev = q.device
    pos = torch.arange(longest, device=dev)
    slot = _slots(s["table"], pos, bs)  # [B, L]
    def dense(codes, scales):
        x = codes.view(nb * bs, kvh, d)[slot].view(torch.float8_e4m3fn).float()
        x = x * scales.view(nb * bs, kvh, 1)[slot]
        return x.transpose(1, 2).reshape(batch * kvh, longest, d)
    k = dense(s["k"], s["ks"])
    # query rows padded to the longest chunk: row i of request b at cu[b] + i
    cu = torch.cumsum(new, 0) - new
    i = torch.arange(most, device=dev)
    at = (cu[:, None] + i).clamp_max(q.shape[0] - 1)
    qp = q.float()[at].view(batch, most, kvh, rep, d).permute(0, 2, 1, 3, 4)
    scores = torch.bmm(qp.reshape(batch * kvh, most * rep, d),
                       (k * s["scale"]).transpose(1, 2).contiguous())
    del k
    scores = scores.view(batch, kvh, most, rep, longest)
    qpos = (total - new)[:, None] + i  # [B, most]
    see = pos <= qpos[:, :, None]
    if s["window"]:
        see &= (pos > qpos[:, :, None] - s["window"]) | (pos < s["sinks"])
    see &= (i < new[:, None])[:, :, None]
    scores = scores.masked_fill_(~see[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    del scores
    norm = p.sum(-1, keepdim=True)
    p /= torch.where(norm == 0, torch.ones_like(norm), norm)
    v = dense(s["v"], s["vs"])
    out = torch.bmm(p.view(batch * kvh, most * rep, longest), v)
    out = out.view(batch, kvh, most, rep, d).permute(0, 2, 1, 3, 4).reshape(batch, most, hq, d)
    out = out[(i < new[:, None])].to(q.dtype)
    if s["kind"] == "attend":
        return out
    heavy = p.sum((2, 3))  # [B, KVH, L]
    rows, old, now = s["row_ids"], s["weights"], s["out_weights"]
    prior = old[rows][:, :, :longest]
    prior = prior * (pos < (total - new)[:, None])[:, None, :]
    keep = now[rows]
    keep[:, :, :longest] = torch.where((pos < total[:, None])[:, None, :], prior + heavy,
                                       keep[:, :, :longest])
    now[rows] = keep
    return out, now


def _plain_evict(s):
    total, w = s["lens"], s["weights"]
    nb, bs, kvh, d = s["k"].shape
    batch, longest = len(s["total"]), max(s["total"])
    dev = w.device
    width = min(longest, s["keep"])
    pos = torch.arange(longest, device=dev)
    live = (pos < total[:, None])[:, None, :]
    always = (pos < s["sinks"]) | (pos >= (total - s["recent"])[:, None])
    key = torch.where(always[:, None, :], torch.full_like(w, math.inf), w)
    key = torch.where(live, key, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    budget = total.clamp_max(s["keep"])
    r = torch.arange(width, device=dev)
    mine = (r < budget[:, None])[:, None, :].expand(batch, kvh, width)
    kept = order[:, :, :width].masked_fill(~mine, longest)
    kept = torch.sort(kept, dim=-1).values
    src_pos = kept.clamp_max(longest - 1)
    bi = torch.arange(batch, device=dev)[:, None, None]
    hi = torch.arange(kvh, device=dev)[None, :, None]
    src = s["table"][bi, src_pos // bs].long() * bs + src_pos % bs
    dst = _slots(s["out_table"], r, bs)[:, None, :].expand(batch, kvh, width)
    src, dst, head = src[mine], dst[mine], hi.expand(batch, kvh, width)[mine]
    kd, ks = s["k"].view(nb * bs, kvh, d), s["ks"].view(nb * bs, kvh)
    vd, vs = s["v"].view(nb * bs, kvh, d), s["vs"].view(nb * bs, kvh)
    kd[dst, head], ks[dst, head] = kd[src, head], ks[src, head]
    vd[dst, head], vs[dst, head] = vd[src, head], vs[src, head]
    moved = torch.gather(w, 2, src_pos)
    s["out_weights"][:, :, :width] = torch.where(mine, moved, s["out_weights"][:, :, :width])
    return _evicted(s, torch.where(mine, kept, torch.full_like(kept, -1)).int())


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "evict":
        return None  # rows move as they are: nothing is computed
    s = prepare(case, seed)
    q = s["q"].double()
    hq, d = q.shape[1:]
    kvh, bs = s["k"].shape[2], s["k"].shape[1]
    rep = hq // kvh
    out = torch.zeros_like(q)
    weights = s["weights"].double() if s["kind"] == "weigh" else None
    row0 = 0
    for b, (total, new) in enumerate(zip(s["total"], s["new"])):
        pages = s["table"][b, : -(-total // bs)].long()
        k = (s["k"][pages].view(torch.float8_e4m3fn).double() * s["ks"][pages]).flatten(0, 1)
        v = (s["v"][pages].view(torch.float8_e4m3fn).double() * s["vs"][pages]).flatten(0, 1)
        j = torch.arange(total, device=q.device)
        for h in range(kvh):
            kh, vh = k[:total, h].t().contiguous(), v[:total, h].contiguous()
            heavy = torch.zeros(total, dtype=torch.float64, device=q.device)
            for first in range(0, new, 512):
                n = min(512, new - first)
                at = slice(row0 + first, row0 + first + n)
                i = total - new + first + torch.arange(n, device=q.device)[:, None]
                hide = j > i
                if s["window"]:
                    hide |= (j <= i - s["window"]) & (j >= s["sinks"])
                x = q[at, h * rep:(h + 1) * rep].reshape(n * rep, d) @ kh * s["scale"]
                x = x.view(n, rep, total).masked_fill(hide[:, None], -math.inf)
                p = torch.softmax(x, -1)
                out[at, h * rep:(h + 1) * rep] = (p.view(n * rep, total) @ vh).view(n, rep, d)
                heavy += p.sum((0, 1))
            if weights is not None:
                r = s["rows"][b]
                weights[r, h, total - new:total] = 0.0
                weights[r, h, :total] += heavy
        row0 += new
    return out if weights is None else (out, weights)
