# SPDX-License-Identifier: Apache-2.0
"""Appending rotated rows to 8-bit pages, and attention over pages with a scale
for each block of positions and head and over pages of shared latent rows, as
measurable calls.

``rope``    a step's query, key and value rows, as the projection leaves them:
            queries and keys rotated to their positions, keys and values stored
            in the E4M3 pages with a scale for each token and head
``append``  the same into pages of E4M3 or INT8 codes with a scale for each
            block of positions and head, where a block may hold rows already
``attend``  attention of each request's new rows (one token to a whole chunk)
            over such pages, with a sliding window and sinks or without
``latent_append``  a step's latent rows (one a token, shared by all heads) as
            E4M3 codes, their position part rotated beside them, and the
            queries' position part rotated
``latent``  attention of new rows over those pages, the up-projections absorbed
            into the queries and the output: a score is over latent and position
            part, the values are the latent

A state is one layer's view at that moment.  With ``own`` the calls are the
package's; without, plain torch.
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
E4M3 = torch.float8_e4m3fn
PACKAGE = Path(__file__).resolve().parents[1] / "vllm-ascend-quantized-kv-cache-hust_amd"
POSITIONS = 32768  # rows of the rotation's table


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one request's next token on one rank of a TP-4 split: latency alone
        dict(name="rope_one_token", kind="rope", batch=1, low=600, high=600, new_low=1, new_high=1,
             heads=10, kv_heads=2, head=128, block=128, rot=128, interleaved=False, dtype="bf16",
             pad=0, lens=1),
        # the step of a prefill batch (40 query / 8 kv heads), everything new
        dict(name="rope_prefill", kind="rope", batch=8, low=0, high=0, new_low=1500, new_high=2048,
             heads=40, kv_heads=8, head=128, block=128, rot=128, interleaved=False, dtype="bf16",
             pad=0, lens=2),
        # a decode batch (32 query / 8 kv heads): one row into every request's last block,
        # padded to its graph's size
        dict(name="append_decode", kind="append", codes="e4m3", batch=59, low=1, high=16384,
             new_low=1, new_high=1, heads=32, kv_heads=8, head=128, block=128, group=128, rot=128,
             interleaved=False, dtype="bf16", pad=5, lens=4),
        # chunks of long prompts behind what is cached already, INT8
        dict(name="append_chunks", kind="append", codes="int8", batch=9, low=0, high=9000,
             new_low=700, new_high=2048, heads=40, kv_heads=8, head=128, block=128, group=128,
             rot=128, interleaved=False, dtype="bf16", pad=0, lens=5),
        # one request's next token on one rank of a TP-4 split, INT8: latency alone
        dict(name="attend_one_token", kind="attend", codes="int8", batch=1, low=600, high=600,
             new_low=1, new_high=1, heads=10, kv_heads=2, head=128, block=128, group=128, window=0,
             sinks=0, dtype="bf16", lens=7),
        # the headline decode batch (40 query / 8 kv heads)
        dict(name="attend_decode", kind="attend", codes="e4m3", batch=32, low=2048, high=16384,
             new_low=1, new_high=1, heads=40, kv_heads=8, head=128, block=128, group=128, window=0,
             sinks=0, dtype="bf16", lens=8),
        # a prefill chunk of 2048 tokens over a long prompt's pages, full causal
        dict(name="attend_chunk", kind="attend", codes="e4m3", batch=4, low=10240, high=10240,
             new_low=2048, new_high=2048, heads=40, kv_heads=8, head=128, block=128, group=128,
             window=0, sinks=0, dtype="bf16", lens=10),
        # a decode batch's next rows, 16 heads a rank
        dict(name="latent_append_decode", kind="latent_append", batch=64, low=600, high=16384,
             new_low=1, new_high=1, heads=16, rank=512, block=128, rot=64, interleaved=True,
             dtype="bf16", pad=0, lens=13),
        # the step of a prefill batch with all of 128 heads
        dict(name="latent_append_prefill", kind="latent_append", batch=8, low=0, high=3000,
             new_low=900, new_high=2048, heads=128, rank=512, block=128, rot=64, interleaved=True,
             dtype="bf16", pad=0, lens=14),
        # a decode batch of long contexts, 16 heads a rank: the cache streams through once
        dict(name="latent_decode_16", kind="latent", batch=32, low=2048, high=16384, new_low=1,
             new_high=1, heads=16, rank=512, block=128, rot=64, dtype="bf16", lens=15),
        # all of 128 heads on one card, two rows a request (one speculated)
        dict(name="latent_decode_128", kind="latent", batch=64, low=1000, high=8192, new_low=2,
             new_high=2, heads=128, rank=512, block=128, rot=64, dtype="bf16", lens=16),
        # ragged chunks over what is cached, 16 heads a rank, small pages
        dict(name="latent_chunk", kind="latent", batch=5, low=1111, high=6000, new_low=100,
             new_high=1024, heads=16, rank=512, block=64, rot=64, dtype="bf16", lens=17),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "latent_append",
                       "latent", "latent"])
    case = dict(kind=kind, block=rng.choice([16, 32, 64, 128, 128]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]), lens=rng.randrange(1 << 30))
    if kind.startswith("latent"):
        head, kv_heads = 64, 1
        case.update(heads=rng.choice([8, 16, 16, 32, 64, 128]), rank=rng.choice([256, 512, 512, 512]),
                    rot=rng.choice([32, 64, 64, 64]))
    else:
        head = rng.choice([64, 128, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8, 8]) if head < 256 else rng.choice([1, 2])
        case.update(kv_heads=kv_heads, head=head, heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8]))
    if kind in ("append", "attend"):
        case["codes"] = rng.choice(["e4m3", "int8"])
        case["group"] = rng.choice([g for g in (16, 32, 64, 128) if g <= case["block"]])
    if kind in ("rope", "append", "latent_append"):
        if kind != "latent_append":
            case["rot"] = rng.choice([head, head, head // 2])
        case["interleaved"] = rng.random() < (0.7 if kind == "latent_append" else 0.3)
        case["pad"] = rng.choice([0, 0, rng.randint(1, 40)])
        case["high"] = _spread(rng, 1, 16384)
        case["low"] = rng.randint(0, case["high"])
        if rng.random() < 0.5:
            case["new_low"] = case["new_high"] = rng.choice([1, 1, 2, 5])
        else:
            case["new_high"] = _spread(rng, 1, 2048)
            case["new_low"] = rng.randint(1, case["new_high"])
        tokens = 14000000 // (head * (case["heads"] + 2 * kv_heads))
        case["batch"] = _spread(rng, 1, max(1, min(200, tokens // case["new_high"])))
        return case
    if kind == "attend":
        case["window"] = rng.choice([0, _spread(rng, 1, 8192)])
        case["sinks"] = rng.choice([0, 1, 4, 100]) if case["window"] else 0
    longest = 16384 if kind == "attend" else 8192
    case["high"] = _spread(rng, 1, longest)
    case["low"] = rng.randint(max(1, case["high"] // 4), case["high"])
    if rng.random() < 0.5:  # decode, or a few rows for every request
        case["new_low"] = case["new_high"] = rng.choice([1, 1, 1, 2, 5])
    else:
        case["new_high"] = _spread(rng, 1, min(2048, case["high"]))
        case["new_low"] = rng.randint(1, case["new_high"])
    rows = case["new_high"] * case["heads"] * case["high"]  # scores of a request
    most = min(64, (2000000000 if kind == "attend" else 500000000) // rows,
               2000000 // (case["high"] * kv_heads))
    case["batch"] = _spread(rng, 1, max(1, most))
    return case


def _lengths(case):
    """(rows after the step, new rows) of every request."""
    rng = random.Random(case["lens"])
    total = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
    new = [rng.randint(case["new_low"], case["new_high"]) for _ in total]
    if case["kind"] in ("attend", "latent"):
        return total, [min(t, n) for t, n in zip(total, new)]
    return [t + n for t, n in zip(total, new)], new  # low .. high rows are there before it


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
    hq = case["heads"]
    if case["kind"] in ("attend", "latent"):
        seen = [_seen(t, n, case.get("window"), case.get("sinks")) for t, n in zip(total, new)]
        cols, pairs = sum(s[0] for s in seen), sum(s[1] for s in seen)
        if case["kind"] == "latent":
            r, p = case["rank"], case["rot"]
            return {"bytes": cols * (r + 4 + 2 * p) + 2 * sum(new) * hq * (2 * r + p),
                    "flops": 2 * hq * pairs * (2 * r + p)}
        kvh, d = case["kv_heads"], case["head"]
        moved = 2 * cols * kvh * d + 8 * kvh * (cols // case["group"]) + 4 * sum(new) * hq * d
        return {"bytes": moved, "flops": 4 * d * hq * pairs}
    rows, live = sum(new) + case["pad"], sum(new)
    table = rows * (4 * case["rot"] + 16)
    if case["kind"] == "latent_append":
        r, p = case["rank"], case["rot"]
        return {"bytes": 4 * rows * hq * p + live * (3 * r + 4 + 4 * p) + table,
                "flops": 3 * rows * (hq + 1) * p}
    kvh, d = case["kv_heads"], case["head"]
    scales = live
    if case["kind"] == "append":
        g = case["group"]
        scales = sum(-(-t // g) - (t - n) // g for t, n in zip(total, new))
    moved = 4 * rows * hq * d + 6 * live * kvh * d + 8 * kvh * scales + table
    return {"bytes": moved, "flops": 3 * rows * (hq + kvh) * case["rot"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _pages(gen, dev, pages, bs, kvh, d, group, codes, sides=2):
    """Keys and values as such a cache holds them: (codes, scales) of each.  Keys have
    outlier channels, values rows of different size.  group 0: a scale for each row."""
    e4m3 = codes == "e4m3"
    data = torch.empty((sides, pages, bs, kvh, d), dtype=torch.uint8 if e4m3 else torch.int8, device=dev)
    shape = (sides, pages, bs // group, kvh) if group else (sides, pages, bs, kvh, 1)
    scale = torch.empty(shape, dtype=torch.float32, device=dev)
    channel = torch.exp(0.5 * torch.randn((kvh, d), generator=gen, device=dev))
    step = max(1, (1 << 26) // (bs * kvh * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        for side in range(sides):
            x = torch.randn((n, bs, kvh, d), generator=gen, device=dev)
            if side == 0:
                x *= channel
            else:
                x *= torch.exp(0.7 * torch.randn((n, bs, kvh, 1), generator=gen, device=dev))
            g = group or 1
            x = x.view(n, bs // g, g, kvh, d)
            top = x.abs().amax((2, 4), keepdim=True)
            if not group:
                s = (top / 448.0).clamp_min(1e-6)
            elif e4m3:
                s = torch.exp2(torch.ceil(torch.log2(top.double() / 448.0))).float()
                s = s.clamp_min(2.0 ** -20)
            else:
                s = (top / 127.0).clamp_min(1e-6)
            x = x / s
            x = x.clamp_(-448.0, 448.0).to(E4M3).view(torch.uint8) if e4m3 else x.round_().to(torch.int8)
            data[side, p:p + n] = x.view(n, bs, kvh, d)
            scale[side, p:p + n] = s.view(scale[side, p:p + n].shape)
    return data, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    if case["kind"] in ("attend", "latent"):
        return _prepare_attend(case, dev, gen, rng)
    total, new = _lengths(case)
    hq, bs, rot = case["heads"], case["block"], case["rot"]
    dtype, pad = DTYPES[case["dtype"]], case["pad"]
    latent = case["kind"] == "latent_append"
    kvh, d = (1, case["rank"]) if latent else (case["kv_heads"], case["head"])
    # the pages that the step writes to, anywhere in a cache
    spans = [((t - n) // bs, (t - 1) // bs) for t, n in zip(total, new)]
    ids = list(range(sum(b - a + 1 for a, b in spans) + 3))
    rng.shuffle(ids)
    pages = len(ids)
    data, scale = _pages(gen, dev, pages, bs, kvh, d, case.get("group", 0), case.get("codes", "e4m3"),
                         sides=1 if latent else 2)
    slots, positions = [], []
    for (a, b), t, n in zip(spans, total, new):
        own_pages = np.array([ids.pop() for _ in range(b - a + 1)], dtype=np.int64)
        pos = np.arange(t - n, t, dtype=np.int64)
        slots.append(own_pages[pos // bs - a] * bs + pos % bs)
        positions.append(pos)
    slots = np.concatenate([*slots, np.full(pad, -1)])
    positions = np.concatenate([*positions, np.zeros(pad, dtype=np.int64)])
    rows = len(slots)
    angle = torch.arange(POSITIONS, dtype=torch.float64, device=dev)[:, None] * torch.pow(
        10000.0, -torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    state = dict(
        kind=case["kind"], interleaved=case["interleaved"], rot=rot, live=rows - pad,
        cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float(),
        positions=torch.from_numpy(positions).to(dev), slots=torch.from_numpy(slots).to(dev),
    )
    def projection(*shape):
        x = torch.randn((rows, *shape), generator=gen, device=dev)
        x *= torch.exp(0.5 * torch.randn(shape, generator=gen, device=dev))
        return x
    if latent:
        # two projections' outputs: [latent | position part] a token, and the queries,
        # each [128 dims | position part]
        down, up = projection(d + rot), projection(hq, 128 + rot).to(dtype)
        down[:, :d] *= torch.exp(0.3 * torch.randn((rows, 1), generator=gen, device=dev))
        down = down.to(dtype)
        state.update(
            q=up[..., 128:], latent=down[:, :d], part=down[:, d:], data=data[0].view(pages, bs, d),
            scale=scale[0].view(pages, bs, 1),
            rope=torch.randn((pages, bs, rot), generator=gen, device=dev).to(dtype))
        return state
    # the fused projection's output, of which queries, keys and values are views
    qkv = projection(hq + 2 * kvh, d)
    qkv[:, hq:] *= torch.exp(0.3 * torch.randn((rows, 2 * kvh, 1), generator=gen, device=dev))
    qkv = qkv.to(dtype)
    state.update(
        q=qkv[:, :hq], key=qkv[:, hq:hq + kvh], value=qkv[:, hq + kvh:], k=data[0], v=data[1],
        ks=scale[0], vs=scale[1], group=case.get("group", 0), codes=case.get("codes", "e4m3"))
    return state


def _prepare_attend(case, dev, gen, rng):
    total, new = _lengths(case)
    bs, dtype = case["block"], DTYPES[case["dtype"]]
    latent = case["kind"] == "latent"
    kvh, d = (1, case["rank"]) if latent else (case["kv_heads"], case["head"])
    batch = len(total)
    width = -(-max(total) // bs)
    pages = batch * width
    order = list(range(pages))
    rng.shuffle(order)
    host = np.array(order, dtype=np.int64).reshape(batch, width)
    data, scale = _pages(gen, dev, pages, bs, kvh, d, case.get("group", 0), case.get("codes", "e4m3"),
                         sides=1 if latent else 2)
    state = dict(
        kind=case["kind"], total=total, new=new, host=host,
        table=torch.from_numpy(host.astype(np.int32)).to(dev), lens=torch.tensor(total, device=dev),
        news=torch.tensor(new, device=dev), window=case.get("window") or None,
        sinks=case.get("sinks", 0))
    wide = d + case["rot"] if latent else d
    q = torch.randn((sum(new), case["heads"], wide), generator=gen, device=dev)
    if latent:  # (the scale is that of a head before its up-projection was absorbed)
        q[..., :d] *= 0.5
        state.update(q=q.to(dtype), data=data[0].view(pages, bs, d), scale_=scale[0].view(pages, bs, 1),
                     rope=torch.randn((pages, bs, case["rot"]), generator=gen, device=dev).to(dtype),
                     scale=(128 + case["rot"]) ** -0.5)
    else:
        state.update(q=(1.5 * q).to(dtype), k=data[0], v=data[1], ks=scale[0], vs=scale[1],
                     group=case["group"], codes=case["codes"], scale=d ** -0.5)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _package():
    if str(PACKAGE) not in sys.path:
        sys.path.insert(0, str(PACKAGE))
    from vllm_ascend_quantized_kv_cache.ops import block8, fp8_latent, fp8_rotary

    return block8, fp8_latent, fp8_rotary


def run(s):
    if own:
        block8, fp8_latent, fp8_rotary = _package()
        if s["kind"] == "attend":
            return block8.block8_attention(
                s["q"], s["k"], s["ks"], s["v"], s["vs"], s["table"], s["total"], s["new"],
                s["scale"], window=s["window"], sinks=s["sinks"], block_table_host=s["host"])
        if s["kind"] == "latent":
            return fp8_latent.fp8_latent_attention(
                s["q"], s["data"], s["scale_"], s["rope"], s["table"], s["total"], s["new"],
                s["scale"], block_table_host=s["host"])
        if s["kind"] == "latent_append":
            q = fp8_latent.fp8_latent_store(
                s["latent"], s["part"], s["positions"], s["cos_sin"], s["slots"], s["data"],
                s["scale"], s["rope"], query=s["q"], interleaved=s["interleaved"])
        elif s["kind"] == "rope":
            q = fp8_rotary.fp8_per_token_head_rotary_store(
                s["q"], s["key"], s["value"], s["positions"], s["cos_sin"], s["slots"], s["k"],
                s["ks"], s["v"], s["vs"], interleaved=s["interleaved"])
        else:
            q = block8.block8_store(
                s["key"], s["value"], s["slots"], s["k"], s["ks"], s["v"], s["vs"], query=s["q"],
                positions=s["positions"], cos_sin=s["cos_sin"], interleaved=s["interleaved"])
        return _stored(s, q)
    if s["kind"] in ("attend", "latent"):
        return _plain_attend(s)
    if s["kind"] == "latent_append":
        return _stored(s, _plain_latent_append(s))
    return _stored(s, _plain_rope(s) if s["kind"] == "rope" else _plain_append(s))


def _stored(s, q):
    """The rotated queries and what the pages hold: E4M3 codes as the values they stand for,
    of INT8 codes the rows just written."""
    if s["kind"] == "latent_append":
        return q, s["data"].view(E4M3), s["scale"], s["rope"]
    if s["codes"] == "e4m3":
        return q, s["k"].view(E4M3), s["ks"], s["v"].view(E4M3), s["vs"]
    slots, (kvh, d) = s["slots"][:s["live"]], s["k"].shape[2:]
    def rows(codes, scales):
        x = codes.view(-1, kvh, d)[slots] * scales.view(-1, kvh, 1)[slots // s["group"]]
        return x.to(q.dtype)
    return q, rows(s["k"], s["ks"]), s["ks"], rows(s["v"], s["vs"]), s["vs"]


def _rotate(x, s):
    """fp32 rows rotated to their positions."""
    half = s["rot"] // 2
    row = s["cos_sin"][s["positions"]]
    cos, sin = row[:, None, :half], row[:, None, half:]
    y = x.float()
    if s["interleaved"]:
        a, b = y[..., 0:s["rot"]:2], y[..., 1:s["rot"]:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:s["rot"]]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., s["rot"]:]], -1)


def _plain_rope(s):
    slots, (kvh, d) = s["slots"][:s["live"]], s["k"].shape[2:]
    for x, codes, scales in ((_rotate(s["key"], s), s["k"], s["ks"]),
                             (s["value"].float(), s["v"], s["vs"])):
        x = x[:s["live"]]
        scale = (x.abs().amax(-1, keepdim=True) / 448.0).clamp_min(1e-6)
        codes.view(-1, kvh, d)[slots] = (x / scale).clamp(-448.0, 448.0).to(E4M3).view(torch.uint8)
        scales.view(-1, kvh, 1)[slots] = scale
    return _rotate(s["q"], s).to(s["q"].dtype)


def _plain_latent_append(s):
    slots, d, p = s["slots"][:s["live"]], s["data"].shape[2], s["rot"]
    x = s["latent"][:s["live"]].float()
    scale = (x.abs().amax(-1, keepdim=True) / 448.0).clamp_min(1e-6)
    s["data"].view(-1, d)[slots] = (x / scale).clamp(-448.0, 448.0).to(E4M3).view(torch.uint8)
    s["scale"].view(-1, 1)[slots] = scale
    part = _rotate(s["part"][:, None], s)[:s["live"], 0]
    s["rope"].view(-1, p)[slots] = part.to(s["rope"].dtype)
    return _rotate(s["q"], s).to(s["q"].dtype)


def _block_scale(top, e4m3):
    if not e4m3:
        return (top / 127.0).clamp_min(1e-6)
    mant, exp = torch.frexp(top.clamp_min(448.0 * 2.0 ** -20))
    return torch.ldexp(torch.ones_like(top), exp - 9 + (mant > 0.875))


def _plain_append(s):
    slots, (kvh, d), g = s["slots"][:s["live"]], s["k"].shape[2:], s["group"]
    e4m3 = s["codes"] == "e4m3"
    blocks, of = torch.unique(slots // g, return_inverse=True)
    first = torch.full_like(blocks, g).scatter_reduce(0, of, slots % g, "amin")
    before = (torch.arange(g, device=slots.device) < first[:, None])[:, :, None, None]
    for x, codes, scales in ((_rotate(s["key"], s), s["k"], s["ks"]),
                             (s["value"].float(), s["v"], s["vs"])):
        x = x[:s["live"]]
        top = torch.zeros((len(blocks), kvh), device=x.device)
        top = top.scatter_reduce(0, of[:, None].expand(-1, kvh), x.abs().amax(-1), "amax")
        scale = _block_scale(top, e4m3)
        old = scales.view(-1, kvh)[blocks]
        scale = torch.where(first[:, None] > 0, torch.maximum(scale, old), scale)
        there = codes.view(-1, g, kvh, d)[blocks]
        was = there.view(E4M3).float() if e4m3 else there.float()
        grown = was * old[:, None, :, None] / scale[:, None, :, None]
        new = x / scale[of][..., None]
        if e4m3:
            grown = grown.to(E4M3).view(torch.uint8)
            new = new.clamp(-448.0, 448.0).to(E4M3).view(torch.uint8)
        else:
            grown = grown.round().to(torch.int8)
            new = new.round().clamp(-127.0, 127.0).to(torch.int8)
        codes.view(-1, g, kvh, d)[blocks] = torch.where(
            before & (scale > old)[:, None, :, None], grown, there)
        codes.view(-1, kvh, d)[slots] = new
        scales.view(-1, kvh)[blocks] = scale
    return _rotate(s["q"], s).to(s["q"].dtype)


def _plain_attend(s):
    q, total, new = s["q"], s["lens"], s["news"]
    batch, (hq, wide), longest, most = len(s["total"]), q.shape[1:], max(s["total"]), max(s["new"])
    latent = s["kind"] == "latent"
    bs, kvh = s["data" if latent else "k"].shape[1], 1 if latent else s["k"].shape[2]
    rep = hq // kvh
    pos = torch.arange(longest, device=q.device)
    slot = s["table"][:, pos // bs].long() * bs + pos % bs  # [B, L]
    if latent:
        d = s["data"].shape[2]
        v = s["data"].view(-1, d)[slot].view(E4M3).float() * s["scale_"].view(-1, 1)[slot]
        k = torch.cat([v, s["rope"].view(-1, wide - d)[slot].float()], -1)
    else:
        d = wide
        def dense(codes, scales):
            x = codes.view(-1, kvh, d)[slot]
            x = x.view(E4M3).float() if s["codes"] == "e4m3" else x.float()
            x = x * scales.view(-1, kvh, 1)[slot // s["group"]]
            return x.transpose(1, 2).reshape(batch * kvh, longest, d)
        k = dense(s["k"], s["ks"])
    # query rows padded to the longest chunk: row i of request b at cu[b] + i
    cu = torch.cumsum(new, 0) - new
    i = torch.arange(most, device=q.device)
    at = (cu[:, None] + i).clamp_max(q.shape[0] - 1)
    qp = q.float()[at].view(batch, most, kvh, rep, wide).permute(0, 2, 1, 3, 4)
    scores = torch.bmm(qp.reshape(batch * kvh, most * rep, wide),
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
    out = torch.bmm(p.view(batch * kvh, most * rep, longest), v if latent else dense(s["v"], s["vs"]))
    out = out.view(batch, kvh, most, rep, d).permute(0, 2, 1, 3, 4).reshape(batch, most, hq, d)
    return out[(i < new[:, None])].to(q.dtype)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(s) if s["kind"] in ("attend", "latent") else _exact_store(s)


def _round_e4m3(x):
    """The nearest E4M3 number, ties to even, past 448 that."""
    size = x.abs()
    step = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(x) * (torch.round(size / step) * step).clamp_max(448.0)


def _exact_store(s):
    e4m3, g, rot = s.get("codes") != "int8", s.get("group"), s["rot"]
    angle = s["cos_sin"].double()[s["positions"]][:, None]
    def rotate(x):
        x = x.double().clone()
        turn = x[..., :rot].clone()
        pairs = turn.unflatten(-1, (rot // 2, 2)) if s["interleaved"] else (
            turn.unflatten(-1, (2, rot // 2)).transpose(-1, -2))
        z = torch.view_as_complex(pairs.contiguous()) * torch.complex(
            angle[..., :rot // 2].contiguous(), angle[..., rot // 2:].contiguous())
        z = torch.view_as_real(z)
        x[..., :rot] = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return x
    def levels(x):
        return _round_e4m3(x) if e4m3 else torch.round(x).clamp(-127, 127)
    if s["kind"] == "latent_append":
        slots, d = s["slots"][:s["live"]], s["data"].shape[2]
        rows = s["latent"][:s["live"]].double()
        data, size = s["data"].view(E4M3).double(), s["scale"].double()
        rope = s["rope"].double()
        size.view(-1)[slots] = (rows.abs().amax(-1) / 448.0).clamp_min(1e-6)
        data.view(-1, d)[slots] = levels(rows / size.view(-1, 1)[slots])
        rope.view(-1, rot)[slots] = rotate(s["part"][:, None])[:s["live"], 0]
        return rotate(s["q"]), data, size, rope
    kvh, d = s["k"].shape[2:]
    slots = s["slots"][:s["live"]]
    host = slots.cpu().numpy()
    result = [rotate(s["q"])]
    for x, codes, scales in ((rotate(s["key"]), s["k"], s["ks"]), (s["value"].double(), s["v"], s["vs"])):
        held = (codes.view(E4M3) if e4m3 else codes).double().view(-1, kvh, d)
        size = scales.double().view(-1, kvh)
        if not g:
            rows = x[:s["live"]]
            size[slots] = (rows.abs().amax(-1) / 448.0).clamp_min(1e-6)
            held[slots] = levels(rows / size[slots][..., None])
        else:
            cuts = [0, *(np.flatnonzero(np.diff(host // g)) + 1).tolist(), len(host)]
            for a, b in zip(cuts, cuts[1:]):
                block, at = int(host[a]) // g, int(host[a]) % g
                top = x[a:b].abs().amax((0, 2))
                if e4m3:
                    want = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp_min(-20.0))
                else:
                    want = (top / 127.0).clamp_min(1e-6)
                if at:
                    old = size[block].clone()
                    want = torch.maximum(want, old)
                    there = held[block * g:block * g + at]
                    there[:] = torch.where((want > old)[:, None],
                                           levels(there * (old / want)[:, None]), there)
                size[block] = want
                held[block * g + at:block * g + at + b - a] = levels(x[a:b] / want[:, None])
        if not e4m3:
            held = held[slots] * size[slots // g][..., None]
        result += [held.view(codes.shape) if e4m3 else held, size.view(scales.shape)]
    return tuple(result)


def _exact_attend(s):
    q = s["q"].double()
    hq = q.shape[1]
    latent = s["kind"] == "latent"
    kvh = 1 if latent else s["k"].shape[2]
    rep = hq // kvh
    out = q.new_zeros((*q.shape[:2], s["data"].shape[2] if latent else q.shape[2]))
    row0 = 0
    for b, (total, new) in enumerate(zip(s["total"], s["new"])):
        bs = s["data" if latent else "k"].shape[1]
        pages = s["table"][b, : -(-total // bs)].long()
        if latent:
            v = s["data"][pages].view(E4M3).double() * s["scale_"][pages]
            k = torch.cat([v, s["rope"][pages].double()], -1).flatten(0, 1)[:, None]
            v = v.flatten(0, 1)[:, None]
        else:
            def values(codes, scales):
                x = codes[pages].view(E4M3) if s["codes"] == "e4m3" else codes[pages]
                x = x.double().unflatten(1, (-1, s["group"]))
                return (x * scales[pages].double()[:, :, None, :, None]).flatten(0, 2)
            k, v = values(s["k"], s["ks"]), values(s["v"], s["vs"])
        j = torch.arange(total, device=q.device)
        for h in range(kvh):
            kh, vh = k[:total, h].t().contiguous(), v[:total, h].contiguous()
            for first in range(0, new, 512):
                n = min(512, new - first)
                at = slice(row0 + first, row0 + first + n)
                i = total - new + first + torch.arange(n, device=q.device)[:, None]
                hide = j > i
                if s["window"]:
                    hide |= (j <= i - s["window"]) & (j >= s["sinks"])
                x = q[at, h * rep:(h + 1) * rep].reshape(n * rep, -1) @ kh * s["scale"]
                x = x.view(n, rep, total).masked_fill(hide[:, None], -math.inf)
                p = torch.softmax(x, -1)
                out[at, h * rep:(h + 1) * rep] = (p.view(n * rep, total) @ vh).view(n, rep, -1)
        row0 += new
    return out
