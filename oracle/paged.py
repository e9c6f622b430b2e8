"""Plain 64-bit restatement of the paged-cache operators on the CPU: append
with rotation, the 4-bit rows, gather, and attention with a window and sinks.

Caches are canonical per-layer tensors ``[num_blocks, 2, H, block_size, D]``;
a 4-bit cache is a pair of unpacked codes (same shape) and ``(step, zero)``
pairs ``[num_blocks, 2, H, block_size, D / group, 2]``.
"""

from __future__ import annotations

import math

import torch

AXES = {"canonical": (0, 1, 2, 3, 4), "vllm": (1, 0, 3, 2, 4), "trtllm": (0, 1, 3, 2, 4)}


def to_layout(t: torch.Tensor, layout: str) -> torch.Tensor:
    """A canonical cache tensor as a contiguous tensor of ``layout``."""
    inverse = [AXES[layout].index(i) for i in range(5)]
    return t.permute(*inverse, *range(5, t.ndim)).contiguous()


def from_layout(t: torch.Tensor, layout: str) -> torch.Tensor:
    return t.permute(*AXES[layout], *range(5, t.ndim))


def pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpack(packed: torch.Tensor) -> torch.Tensor:
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def rotate(x: torch.Tensor, positions: torch.Tensor, base: float | None, style: str) -> torch.Tensor:
    """``[T, H, D]`` rows turned by their positions, in float64."""
    x = x.double()
    if base is None:
        return x
    d = x.shape[-1]
    freq = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    ang = (positions.double()[:, None] * freq)[:, None]
    c, s = torch.cos(ang), torch.sin(ang)
    out = torch.empty_like(x)
    if style == "neox":
        a, b = x[..., : d // 2], x[..., d // 2 :]
        out[..., : d // 2], out[..., d // 2 :] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        out[..., 0::2], out[..., 1::2] = a * c - b * s, b * c + a * s
    return out


def quantise(x: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and (step, zero) of rows rounded to fp32, each operation rounded to fp32."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).clamp(-60000, 60000), g.amax(-1).clamp(-60000, 60000)
    zero, step = lo.half(), ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).half()
    inv = torch.where(step.float() > 0, 1.0 / step.float(), torch.zeros(()))
    codes = ((g - zero.float()[..., None]) * inv[..., None]).round().clamp(0, 15).nan_to_num(0.0)
    return codes.flatten(-2).to(torch.uint8), torch.stack([step, zero], -1)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    group = codes.shape[-1] // scales.shape[-2]
    s = scales.double()
    return (codes.double().unflatten(-1, (-1, group)) * s[..., 0:1] + s[..., 1:2]).flatten(-2)


def rows_of(tables, cu, positions, block_size: int, num_blocks: int):
    """Per token: (request, block, offset), block -1 where the position addresses no row; None for padding."""
    got = []
    for t, p in enumerate(positions.tolist()):
        owner = [b for b in range(len(cu) - 1) if cu[b] <= t < cu[b + 1]]
        if not owner:
            got.append(None)
            continue
        lb = p // block_size
        e = int(tables[owner[0], lb]) if 0 <= p and lb < tables.shape[1] else -1
        got.append((owner[0], e if 0 <= e < num_blocks else -1, p % block_size))
    return got


def append(cache, key, value, tables, cu, positions, base, style) -> int:
    """Into a 16- or 32-bit canonical cache, in place; returns the tokens skipped."""
    k = rotate(key, positions, base, style).to(cache.dtype)
    skipped = 0
    for t, at in enumerate(rows_of(tables, cu, positions, cache.shape[3], cache.shape[0])):
        if at is None:
            continue
        if at[1] < 0:
            skipped += 1
            continue
        cache[at[1], 0, :, at[2]] = k[t]
        cache[at[1], 1, :, at[2]] = value[t]
    return skipped


def append4(codes, scales, key, value, tables, cu, positions, base, style) -> int:
    group = codes.shape[-1] // scales.shape[-2]
    rows = [quantise(rotate(key, positions, base, style), group), quantise(value.double(), group)]
    skipped = 0
    for t, at in enumerate(rows_of(tables, cu, positions, codes.shape[3], codes.shape[0])):
        if at is None:
            continue
        if at[1] < 0:
            skipped += 1
            continue
        for kv in (0, 1):
            codes[at[1], kv, :, at[2]] = rows[kv][0][t]
            scales[at[1], kv, :, at[2]] = rows[kv][1][t]
    return skipped


def attention(query, cache, tables, cu, positions, window=None, sinks=0, scale=None):
    """``query [T, Hq, D]`` over a canonical cache of float64 values.

    Returns ``(out, spread, reach)``: the result, ``sum_j w_j |v_j|`` (the
    weight a relative error of a probability has) and, per row,
    ``max_j sum_d |q_d| |k_jd| * scale`` (the size of what a score sums).
    Padding rows are zero.  Only visible rows are looked at.
    """
    T, Hq, D = query.shape
    H, bs = cache.shape[2], cache.shape[3]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros(T, Hq, dtype=torch.float64)
    for t, at in enumerate(rows_of(tables, cu, positions, bs, cache.shape[0])):
        if at is None:
            continue
        b, p = at[0], int(positions[t])
        j = torch.arange(0, max(0, min(p + 1, tables.shape[1] * bs)))
        if window is not None:
            j = j[(j > p - window) | (j < sinks)]
        page = tables[b, j // bs].long()
        j = j[(page >= 0) & (page < cache.shape[0])]
        if j.numel() == 0:
            continue
        page = tables[b, j // bs].long()
        kv = cache[page, :, :, j % bs].double()  # [J, 2, H, D]
        q, k, v = query[t].double().unflatten(0, (H, -1)), kv[:, 0].transpose(0, 1), kv[:, 1].transpose(0, 1)
        x = (q @ k.mT) * scale  # [H, Hq / H, J]
        w = torch.exp(x - x.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        out[t], spread[t] = (w @ v).flatten(0, 1), (w @ v.abs()).flatten(0, 1)
        reach[t] = (q.abs() @ k.abs().mT).amax(-1).flatten() * abs(scale)
    return out, spread, reach
