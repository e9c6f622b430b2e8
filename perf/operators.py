"""The paged-cache operators, measured: cases, their plain forms in elementary
torch operations, and the calls a serving step makes of the framework.

Four kinds of pass (``case["op"]``):

``append``   one layer's new tokens: K rotated to its position and written
             into the paged cache with V, the query rotated beside it
``store4``   the same rows quantised into a cache held in 4 bits, then read
             back as donor rows (what a later request injects)
``attend``   attention from the paged cache, causal, with an optional sliding
             window and a few first tokens that stay visible (sinks)
``attend4``  the same attention over a cache held in 4 bits

Lengths, new tokens and positions of a case follow from the case alone
(``lens`` seeds them); values, page order and queries follow from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: where block, kv, head, position and dim stand in each per-layer cache layout
AXES = {"canonical": (0, 1, 2, 3, 4), "vllm": (1, 0, 3, 2, 4), "trtllm": (0, 1, 3, 2, 4)}
DEV = "cuda"


def _case(name, op, **kw):
    c = {
        "name": name, "op": op, "dtype": "bf16", "q_heads": 28, "kv_heads": 4, "head_dim": 128, "block": 16,
        "layout": "canonical", "style": "neox", "base": 1e6, "group": 64, "requests": 1, "ctx_min": 1,
        "ctx_max": 1, "new_min": 1, "new_max": 1, "idle": 0, "rows": "tail", "window": 0, "sinks": 0, "lens": 1,
    }
    c.update(kw)
    return c


def listed():
    llama = {"q_heads": 64, "kv_heads": 8, "base": 5e5}
    return [
        # a decode step of one tensor-parallel rank: 64 requests of 4K-32K tokens, one new token each
        _case("append step", "append", q_heads=8, kv_heads=1, base=5e5, requests=64, ctx_min=4096, ctx_max=32768),
        # prefill of a 16K request: every row of a layer's K, V and query
        _case("append chunk", "append", ctx_min=16384, ctx_max=16384, new_min=16384, new_max=16384),
        # a ragged mixed batch: short fp16 heads, interleaved pairs, the position-major layout, idle slots
        _case("append ragged", "append", dtype="fp16", q_heads=12, kv_heads=3, head_dim=64, style="interleaved",
              layout="vllm", base=1e4, block=32, requests=9, ctx_min=700, ctx_max=3000, new_min=1, new_max=700, idle=2),
        # one decoded token of each of 64 requests into a 4-bit cache of every KV head
        _case("store4 step", "store4", requests=64, ctx_min=4096, ctx_max=8192, **llama),
        # a 16K request's rows into a 4-bit cache
        _case("store4 chunk", "store4", ctx_min=16384, ctx_max=16384, new_min=16384, new_max=16384),
        # the smallest call: one request's next token over a short prompt
        _case("attend one", "attend", ctx_min=517, ctx_max=517, window=4096, sinks=4),
        # a decode step of 64 long requests under a sliding window with sinks
        _case("attend step", "attend", requests=64, ctx_min=4096, ctx_max=32768, window=4096, sinks=4, **llama),
        # a decode step of a few 32K requests that see every key, fp16, trtllm pages of 64
        _case("attend long", "attend", dtype="fp16", requests=8, ctx_min=20000, ctx_max=32768, layout="trtllm", block=64),
        # partial prefill: a tenth of 32K positions recomputed (spans and the tail), the rest reused
        _case("attend partial", "attend", ctx_min=32768, ctx_max=32768, new_min=3277, new_max=3277, rows="spans",
              window=4096, sinks=4),
        # the next token of one 32K request from a 4-bit cache
        _case("attend4 one", "attend4", ctx_min=32768, ctx_max=32768),
        # a decode step of 64 long requests from a 4-bit cache
        _case("attend4 step", "attend4", requests=64, ctx_min=4096, ctx_max=32768, **llama),
        # a prefill chunk that attends to a 16K prompt held in 4 bits
        _case("attend4 chunk", "attend4", ctx_min=16384, ctx_max=16384, new_min=2048, new_max=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "store4", "attend", "attend4"])
    kv = rng.choice([1, 2, 3, 4, 8])
    c = _case("", op, dtype=rng.choice(["bf16", "bf16", "fp16"]), kv_heads=kv,
              q_heads=kv * rng.choice([1, 2, 4, 5, 7, 8, 8]), head_dim=rng.choice([64, 128, 128]),
              block=rng.choice([16, 16, 16, 32, 64]), layout=rng.choice(["canonical", "canonical", "vllm", "trtllm"]),
              style=rng.choice(["neox", "interleaved"]), base=rng.choice([1e4, 5e5, 1e6]), lens=rng.randrange(1 << 30))
    c["group"] = rng.choice([32, 64, 64, 128]) if c["head_dim"] == 128 else rng.choice([32, 64])
    c["requests"] = _log(rng, 1, 64)
    if op in ("append", "store4"):
        if op == "append":
            c["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
        row = (2 * kv + (c["q_heads"] if op == "append" else 0)) * c["head_dim"] * (2 if c["dtype"] == "fp32" else 1)
        most = 16384 * 128 * (36 if op == "append" else 8) // row  # new tokens of the listed chunks' bytes
        total = _log(rng, c["requests"], max(c["requests"], min(16384, most // 2)))
        c["new_max"] = max(1, 2 * total // c["requests"] - 1)
        c["ctx_min"], c["ctx_max"] = c["new_max"], c["new_max"] + _log(rng, 1, 4096)
        c["idle"] = rng.choice([0, 0, c["requests"] // 4])
    else:
        c["window"] = rng.choice([0, _log(rng, 64, 8192)])
        c["sinks"] = rng.choice([0, 4, _log(rng, 1, 200)])
        if rng.random() < 0.6:  # decode, or a few tokens verified at once
            c["new_max"] = rng.choice([1, 1, 1, 2, 5])
            c["ctx_min"] = _log(rng, 5, 8192)
            c["ctx_max"] = max(c["ctx_min"], _log(rng, 64, 32768))
            if op == "attend" and c["requests"] * c["ctx_max"] <= 1 << 18 and rng.random() < 0.2:
                c["dtype"] = "fp32"
        else:  # prefill chunks, whole or the recomputed rows of partial ones
            c["requests"] = min(c["requests"], 4)
            past = _log(rng, 1, 16384)
            most = 4e11 / (4 * c["head_dim"] * c["q_heads"] * (past + 1500))  # no more than the largest listed case
            n = _log(rng, 64, max(65, min(3000, most)))
            c["new_max"] = max(1, n // c["requests"])
            c["new_min"] = max(1, c["new_max"] // 2)
            c["ctx_min"], c["ctx_max"] = c["new_max"], c["new_max"] + past
            c["rows"] = rng.choice(["tail", "tail", "spans"])
            c["idle"] = rng.choice([0, 1]) if c["requests"] > 1 else 0
    del c["name"]
    return c


def _plan(case):
    """(context length, ascending positions of the new tokens) of each request."""
    rng = random.Random(case["lens"])
    got = []
    for b in range(case["requests"]):
        lo, hi = case["ctx_min"], case["ctx_max"]
        ctx = lo if lo == hi else int(min(hi, max(lo, round(rng.lognormvariate(math.log(math.sqrt(lo * hi)), 0.7)))))
        new = 0 if b < case["idle"] else min(ctx, rng.randint(case["new_min"], case["new_max"]))
        if case["rows"] == "spans" and new < ctx:
            # contiguous recomputed spans over the context, and the tail
            tail = max(1, new // 6)
            rest, n_spans = new - tail, max(1, (new - tail) // 43)
            cuts = sorted(rng.sample(range(rest + n_spans), n_spans - 1)) if n_spans > 1 else []
            sizes = np.diff([-1] + cuts + [rest + n_spans - 1]) - 1
            free = ctx - tail - rest
            gaps = np.sort([rng.randint(0, free) for _ in range(n_spans)])
            starts = gaps + np.concatenate([[0], np.cumsum(sizes)[:-1]])
            pos = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, sizes)] + [np.arange(ctx - tail, ctx)])
        else:
            pos = np.arange(ctx - new, ctx)
        got.append((ctx, pos.astype(np.int64)))
    return got


def _visible(case, ctx, pos):
    """(sum over the tokens of keys seen, keys that some token sees)."""
    w = case["window"] or ctx + 1
    inside = np.minimum(pos + 1, w)
    total = int((inside + np.minimum(case["sinks"], pos + 1 - inside)).sum())
    edge = np.zeros(ctx + 1, np.int64)
    np.add.at(edge, np.maximum(0, pos + 1 - w), 1)
    np.add.at(edge, pos + 1, -1)
    seen = np.cumsum(edge)[:ctx] > 0
    if len(pos):
        seen[: min(case["sinks"], int(pos.max()) + 1)] = True
    return total, int(seen.sum())


def work(case):
    plan = _plan(case)
    hq, h, d, es = case["q_heads"], case["kv_heads"], case["head_dim"], 4 if case["dtype"] == "fp32" else 2
    t = sum(len(p) for _, p in plan)
    four = 2 * h * (d // 2 + 4 * d // case["group"])  # one token's row of a 4-bit cache
    meta = 12 * t + 4 * len(plan)
    if case["op"] == "append":
        return {"bytes": 2 * t * (2 * h + hq) * d * es + meta, "flops": 3 * t * (h + hq) * d}
    if case["op"] == "store4":
        return {"bytes": 2 * t * 2 * h * d * es + 2 * t * four + meta, "flops": t * h * d * (3 + 2 * 8)}
    seen = [_visible(case, ctx, pos) for ctx, pos in plan]
    row = four if case["op"] == "attend4" else 2 * h * d * es
    keys = sum(s[1] for s in seen)
    return {"bytes": keys * row + 2 * t * hq * d * es + meta + 4 * keys / case["block"],
            "flops": 4 * d * hq * sum(s[0] for s in seen)}


def _quantise(x, group):
    """4-bit codes [..., D] and (step, zero) [..., D / group, 2] of fp32 rows:
    zero = fp16(min), step = fp16((max - min) / 15), codes to the nearest."""
    g = x.unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    zero = lo.clamp(-65504, 65504).half()
    step = ((hi - lo) / 15).clamp(max=65504).half()
    inv = torch.where(step > 0, 1.0 / step.float(), 0.0)
    codes = ((g - zero.float()[..., None]) * inv[..., None]).round().clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), torch.stack([step, zero], -1)


def _values(codes, scales, group):
    """What the codes stand for, in fp32."""
    s = scales.float()
    return (codes.float().unflatten(-1, (-1, group)) * s[..., 0:1] + s[..., 1:2]).flatten(-2)


def _ordered(t, layout):
    """[blocks, 2, heads, block, last dims] view of a cache tensor in `layout`."""
    return t.permute(*AXES[layout], *range(5, t.dim()))


def _stored(t, layout):
    """A canonical tensor laid out in memory as `layout` has it."""
    inverse = [AXES[layout].index(i) for i in range(5)]
    return t.permute(*inverse, *range(5, t.dim())).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    plan = _plan(case)
    dt, d, h, bs = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"], case["block"]
    t = sum(len(p) for _, p in plan)
    pages = [-(-ctx // bs) for ctx, _ in plan]
    blocks = sum(pages) + max(1, sum(pages) // 16)
    order = torch.randperm(blocks, generator=g, device=DEV)
    owner = torch.tensor(np.repeat(np.arange(len(plan)), pages), device=DEV)
    slot = torch.tensor(np.concatenate([np.arange(n) for n in pages]), device=DEV)
    table = torch.full((len(plan), max(pages)), -1, dtype=torch.int32, device=DEV)
    table[owner, slot] = order[: sum(pages)].int()
    counts = [len(p) for _, p in plan]
    s = {
        "case": case,
        "longest": max(ctx for ctx, _ in plan),
        "most": max(counts),
        "tables": table,
        "cu": torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEV),
        "positions": torch.tensor(np.concatenate([p for _, p in plan]), dtype=torch.int32, device=DEV),
        "request": torch.tensor(np.repeat(np.arange(len(plan)), counts), device=DEV),
        "query": torch.randn(t, case["q_heads"], d, generator=g, device=DEV).to(dt),
        "inv_freq": case["base"] ** (-torch.arange(0, d, 2, dtype=torch.float64) / d),
    }
    s["inv_freq"] = s["inv_freq"].to(DEV)
    # keys with a gain of their own per channel, values of unit variance
    gain = torch.exp(0.25 * torch.randn(d, generator=g, device=DEV))
    shape = (blocks, 1, h, bs, d)
    four = case["op"] in ("store4", "attend4")
    parts = []
    for scale in (gain, torch.ones_like(gain)):
        rows = torch.randn(shape, generator=g, device=DEV).mul_(scale)
        parts.append(_quantise(rows, case["group"]) if four else (rows.to(dt),))
        del rows
    if four:
        codes = torch.cat([parts[0][0], parts[1][0]], 1)
        s["codes"] = _stored(codes[..., 0::2] | (codes[..., 1::2] << 4), case["layout"])
        s["scales"] = _stored(torch.cat([parts[0][1], parts[1][1]], 1), case["layout"])
    else:
        s["cache"] = _stored(torch.cat([parts[0][0], parts[1][0]], 1), case["layout"])
    if case["op"] in ("append", "store4"):
        s["key"] = (torch.randn(t, h, d, generator=g, device=DEV) * gain).to(dt)
        s["value"] = torch.randn(t, h, d, generator=g, device=DEV).to(dt)
    s["out"] = torch.zeros(2, h, t, d, dtype=dt, device=DEV) if case["op"] == "store4" else torch.zeros_like(s["query"])
    return s


def _rotated(x, angles, style):
    """Rows [T, heads, D] rotated by angles [T, D / 2] (both in 64 bits)."""
    c, n = torch.cos(angles)[:, None], torch.sin(angles)[:, None]
    x = x.double()
    if style == "neox":
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * n, b * c + a * n], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)


def _places(s):
    """Physical block and offset of each new token."""
    bs = s["case"]["block"]
    pos = s["positions"].long()
    return s["tables"].long()[s["request"], pos // bs], pos % bs


def _plain_append(s):
    c = s["case"]
    angles = s["positions"].double()[:, None] * s["inv_freq"]
    block, off = _places(s)
    cache = _ordered(s["cache"], c["layout"])
    cache[block, 0, :, off] = _rotated(s["key"], angles, c["style"]).to(cache.dtype)
    cache[block, 1, :, off] = s["value"]
    s["out"].copy_(_rotated(s["query"], angles, c["style"]))
    return s["cache"], s["out"]


def _plain_store4(s):
    c = s["case"]
    angles = s["positions"].double()[:, None] * s["inv_freq"]
    block, off = _places(s)
    codes, scales = _ordered(s["codes"], c["layout"]), _ordered(s["scales"], c["layout"])
    k = _quantise(_rotated(s["key"], angles, c["style"]).float(), c["group"])
    v = _quantise(s["value"].float(), c["group"])
    q = torch.stack([k[0], v[0]], 1)
    codes[block, :, :, off] = q[..., 0::2] | (q[..., 1::2] << 4)
    scales[block, :, :, off] = torch.stack([k[1], v[1]], 1)
    back = codes[block, :, :, off]
    back = torch.stack([back & 15, back >> 4], -1).flatten(-2)
    rows = _values(back, scales[block, :, :, off], c["group"])
    s["out"].copy_(rows.permute(1, 2, 0, 3))
    return s["out"]


def _plain_attend(s):
    c = s["case"]
    hq, h, d, n = c["q_heads"], c["kv_heads"], c["head_dim"], s["most"]
    b, length = c["requests"], s["longest"]
    j = torch.arange(length, device=DEV)
    block = s["tables"].long()[:, j // c["block"]]
    mapped, block, off = block >= 0, block.clamp(min=0), (j % c["block"]).expand(b, -1)
    if c["op"] == "attend4":
        codes, scales = _ordered(s["codes"], c["layout"]), _ordered(s["scales"], c["layout"])

        def rows(kv):
            q = codes[block, kv, :, off]
            return _values(torch.stack([q & 15, q >> 4], -1).flatten(-2), scales[block, kv, :, off], c["group"])
    else:
        cache = _ordered(s["cache"], c["layout"])

        def rows(kv):
            return cache[block, kv, :, off].float()
    place = torch.arange(len(s["request"]), device=DEV) - s["cu"].long()[s["request"]]
    q = torch.zeros(b, n, hq, d, device=DEV)
    q[s["request"], place] = s["query"].float()
    p = torch.full((b, n), -1, dtype=torch.long, device=DEV)
    p[s["request"], place] = s["positions"].long()
    q = q.unflatten(2, (h, hq // h)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, H, G * n, D]
    see = (j <= p[..., None]) & mapped[:, None]
    if c["window"]:
        see &= (j > p[..., None] - c["window"]) | (j < c["sinks"])
    score = (q @ rows(0).permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    score = score.unflatten(2, (hq // h, n)).masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.flatten(2, 3) @ rows(1).permute(0, 2, 1, 3)).unflatten(2, (hq // h, n))
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
    s["out"].copy_(out[s["request"], place])
    return s["out"]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "store4": _plain_store4}.get(c["op"], _plain_attend)(s)
    from semblend_b200.paged_attention import Int4KVCache, PagedBatch, append_paged_kv, gather_paged_kv, paged_attention

    batch = PagedBatch(s["tables"], s["cu"], s["positions"])
    four = c["op"] in ("store4", "attend4")
    cache = Int4KVCache(s["codes"], s["scales"], layout=c["layout"]) if four else s["cache"]
    layout = "auto" if four else c["layout"]
    if c["op"] == "append":
        append_paged_kv(cache, s["key"], s["value"], batch, rope_base=c["base"], rotary_style=c["style"],
                        layout=layout, query=s["query"], query_out=s["out"])
        return cache, s["out"]
    if c["op"] == "store4":
        append_paged_kv(cache, s["key"], s["value"], batch, rope_base=c["base"], rotary_style=c["style"])
        return gather_paged_kv(cache, batch, out=s["out"])
    return paged_attention(s["query"], cache, batch, window=c["window"] or None, sinks=c["sinks"], layout=layout,
                           out=s["out"])


def exact(case, seed):
    """The definitions in 64 bits, request by request."""
    s, plan = prepare(case, seed), _plan(case)
    bs, d, h, hq = case["block"], case["head_dim"], case["kv_heads"], case["q_heads"]
    cu = s["cu"].tolist()
    half = torch.arange(d // 2, device=DEV)
    first, second = (half, half + d // 2) if case["style"] == "neox" else (2 * half, 2 * half + 1)

    def turn(x, pos):
        """Each RoPE pair as a complex number times exp(i * position * frequency)."""
        z = torch.complex(x[..., first].double(), x[..., second].double())
        freq = torch.tensor([case["base"] ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device=DEV)
        z = z * torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos.double()[:, None, None] * freq)
        y = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if case["op"] == "append":
        cache = s["cache"].double()
        view = _ordered(cache, case["layout"])
        k = turn(s["key"], s["positions"])
        for r in range(len(plan)):
            a, e = cu[r], cu[r + 1]
            pos = s["positions"][a:e].long()
            at = s["tables"][r].long()[pos // bs]
            view[at, 0, :, pos % bs] = k[a:e]
            view[at, 1, :, pos % bs] = s["value"][a:e].double()
        return cache, turn(s["query"], s["positions"])
    if case["op"] == "store4":
        def kept(x):
            rows = x.double().reshape(-1, case["group"])
            lo, hi = rows.min(1, keepdim=True).values, rows.max(1, keepdim=True).values
            zero, step = lo.float().half().double(), ((hi - lo) / 15).float().half().double()
            code = torch.nan_to_num((rows - zero) / step, nan=0.0, posinf=0.0, neginf=0.0).round().clamp(0, 15)
            return (zero + code * step).reshape(x.shape)

        k, v = kept(turn(s["key"], s["positions"]).float()), kept(s["value"])
        return torch.stack([k, v]).transpose(1, 2)
    out = torch.zeros(cu[-1], hq, d, dtype=torch.float64, device=DEV)
    for r, (ctx, _) in enumerate(plan):
        a, e = cu[r], cu[r + 1]
        pages = s["tables"][r, : -(-ctx // bs)].long()
        if case["op"] == "attend4":
            codes = _ordered(s["codes"], case["layout"])[pages].transpose(0, 1)
            low, high = (codes % 16).double(), (codes // 16).double()
            sc = _ordered(s["scales"], case["layout"])[pages].transpose(0, 1).double()
            kv = torch.empty(*codes.shape[:-1], d, dtype=torch.float64, device=DEV)
            kv[..., 0::2], kv[..., 1::2] = low, high
            kv = kv * sc[..., 0].repeat_interleave(case["group"], -1) + sc[..., 1].repeat_interleave(case["group"], -1)
        else:
            kv = _ordered(s["cache"], case["layout"])[pages].transpose(0, 1).double()
        k, v = kv.transpose(1, 2).flatten(2, 3)[:, :, :ctx]  # each [H, ctx, D]
        j = torch.arange(ctx, device=DEV)
        for i in range(a, e, 256):
            p = s["positions"][i : min(i + 256, e)].long()[:, None]
            q = s["query"][i : min(i + 256, e)].double().reshape(len(p), h, hq // h, d)
            see = (p >= j) if not case["window"] else (p >= j) & ((p - j < case["window"]) | (j < case["sinks"]))
            logit = torch.einsum("nhgd,hjd->nhgj", q, k) / math.sqrt(d)
            weight = torch.softmax(logit.masked_fill(~see[:, None, None], -math.inf), -1)
            out[i : i + len(p)] = torch.einsum("nhgj,hjd->nhgd", weight, v).reshape(len(p), hq, d)
    return out
