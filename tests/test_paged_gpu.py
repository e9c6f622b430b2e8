"""GPU tests of the paged-cache operators against the 64-bit restatement
(``oracle/paged.py``).

Tolerances count roundings (u = half a step of a type, relative):

* a rotated element: the fp32 rotation is within 6 u32 of the pair's norm (cos
  and sin to 2 u32 each after the 64-bit reduction, two products, one sum),
  then one rounding to the cache's type;
* 4-bit rows: none; codes, steps and zeros are functions of the fp32 values,
  which the 64-bit rotation pins;
* attention: one rounding of the result, u * |out|; one rounding of each
  probability to the type the products take, u_p * sum_j w_j |v_j|, or, over a
  4-bit cache and a bf16 result, of each probability times its key's step to
  fp16, which multiplies the code alone (the zero's part is summed in fp32):
  2^-11 * sum_j w_j step_j code_j; the fp32 sums, and the scores: a sum of D products in steps of 16 loses at most
  2^-23 per step of the largest partial sum, and moves the result by twice that
  times sum_j w_j |v_j|.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as op
from semblend_b200 import _lib
from semblend_b200 import rope_correction as rc
from semblend_b200.paged_attention import (
    Int4KVCache,
    PagedBatch,
    append_paged_kv,
    gather_paged_kv,
    paged_attention,
)
from semblend_b200.triton_kernels import partial_prefill_attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


class Case:
    """A seeded ragged batch over a shuffled pool; host tensors, canonical layout."""

    def __init__(self, *, ctx, new, dtype=BF, hq=8, h=2, d=128, bs=16, group=None, seed=0, spread=False, pad=0,
                 table=torch.int32, pos=torch.int32, stale=None):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.dtype, self.hq, self.h, self.d, self.bs, self.group = dtype, hq, h, d, bs, group
        pages = [-(-c // bs) for c in ctx]
        self.nb = sum(pages) + 3
        order = torch.randperm(self.nb, generator=g).tolist()
        width = max(max(pages), 1)
        self.tables = torch.full((len(ctx), width), -1, dtype=table)
        at = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = torch.tensor(order[at : at + n], dtype=table)
            at += n
        self.cu = [0] + np.cumsum(new).tolist()
        positions = []
        for c, n in zip(ctx, new):
            positions += sorted(rng.choice(c, n, replace=False).tolist()) if spread else list(range(c - n, c))
        self.positions = torch.tensor(positions + [0] * pad, dtype=pos)
        T = len(positions) + pad
        self.T, self.pad = T, pad
        self.q = torch.randn(T, hq, d, generator=g).to(dtype)
        self.k = torch.randn(T, h, d, generator=g).to(dtype)
        self.v = torch.randn(T, h, d, generator=g).to(dtype)
        shape = (self.nb, 2, h, bs, d)
        full = torch.randn(shape, generator=g) * torch.exp(0.3 * torch.randn(d, generator=g))
        if group is None:
            self.cache = full.to(dtype)
        else:
            self.codes, self.scales = op.quantise(full, group)
        self.ctx = ctx
        if stale is not None:
            self._spoil(stale)

    def _spoil(self, what):
        """Every row no request holds: `what`."""
        held = torch.zeros(self.nb, self.bs, dtype=torch.bool)
        for b, c in enumerate(self.ctx):
            for j in range(c):
                held[int(self.tables[b, j // self.bs]), j % self.bs] = True
        lost = (~held)[:, None, None, :]
        if self.group is None:
            self.cache = torch.where(lost[..., None], torch.tensor(what, dtype=self.dtype), self.cache)
        else:
            self.scales = torch.where(lost[..., None, None], torch.tensor(what, dtype=torch.float16), self.scales)

    def value_cache(self):
        return self.cache if self.group is None else op.values(self.codes, self.scales)

    def device_cache(self, layout="canonical"):
        if self.group is None:
            return op.to_layout(self.cache, layout).to(DEV)
        return Int4KVCache(op.to_layout(op.pack(self.codes), layout).to(DEV), op.to_layout(self.scales, layout).to(DEV),
                           layout=layout)

    def batch(self):
        return PagedBatch(self.tables.to(DEV), torch.tensor(self.cu, dtype=torch.int32, device=DEV),
                          self.positions.to(DEV))


def check_attention(c: Case, got, *, window=None, sinks=0, scale=None):
    want, spread, reach = op.attention(c.q, c.value_cache(), c.tables, c.cu, c.positions, window, sinks, scale)
    n = c.cu[-1]
    got = got.cpu().double()
    u = U[c.dtype]
    # scores over codes sum q * (1024 + code): up to 1039 / 15 times what q * code sums
    partial = reach * (1.0 if c.group is None else 1039.0 / 7.5)
    delta = (c.d / 16 + 2) * 2.0**-23 * partial + 2.0**-21
    tol = u * want.abs() + (u + 2.0**-20 + 2 * delta[..., None]) * spread + 2.0**-25
    if c.group is not None and c.dtype == BF:
        coded = c.value_cache()
        coded[:, 1] -= c.scales[:, 1, ..., 1].double().repeat_interleave(c.group, -1)  # step * code
        tol += 2.0**-11 * op.attention(c.q, coded, c.tables, c.cu, c.positions, window, sinks, scale)[0]
    if c.dtype == FP:  # a plain chain of D products
        tol = u * want.abs() + (2.0**-19 + 2 * (c.d * 2.0**-24 * partial[..., None])) * spread + 2.0**-30
    bad = ~((got[:n] - want[:n]).abs() <= tol[:n])
    assert not bad.any(), (int(bad.sum()), float((got[:n] - want[:n]).abs().max()),
                           float(((got[:n] - want[:n]).abs() / tol[:n]).max()), bad.nonzero()[:4].tolist())


def attend(c: Case, layout="canonical", **kw):
    out = torch.full((c.T, c.hq, c.d), 7.0, dtype=c.dtype, device=DEV)
    got = paged_attention(c.q.to(DEV), c.device_cache(layout), c.batch(), out=out, layout=layout, **kw)
    assert got is out
    if c.pad:
        assert torch.all(out[c.cu[-1] :] == 7.0)  # rows behind the last sequence are left as they were
    kw.pop("status", None)
    check_attention(c, out, **kw)
    return out


# --------------------------------------------------------------------------- append


def rope_tolerance(x, want, style, u):
    n = x.double()
    d = n.shape[-1]
    if style == "neox":
        norm = torch.sqrt(n[..., : d // 2] ** 2 + n[..., d // 2 :] ** 2)
        norm = torch.cat([norm, norm], -1)
    else:
        norm = torch.sqrt(n[..., 0::2] ** 2 + n[..., 1::2] ** 2).repeat_interleave(2, -1)
    return 6 * U[FP] * norm + u * (want.abs() + 6 * U[FP] * norm) + 2.0**-26


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("style", ["neox", "interleaved"])
@pytest.mark.parametrize(
    "layout,hq,h,d,bs,pad,pos",
    [("canonical", 8, 2, 128, 16, 3, torch.int32), ("vllm", 6, 3, 64, 8, 0, torch.int64),
     ("trtllm", 5, 5, 80, 7, 1, torch.int32), ("canonical", 1, 1, 2, 1, 2, torch.int64),
     ("canonical", 3, 1, 18, 24, 0, torch.int32), ("canonical", 2, 1, 512, 4, 0, torch.int32)],
)
def test_append_rows(dtype, style, layout, hq, h, d, bs, pad, pos):
    c = Case(ctx=[40, 9, 1, 33], new=[17, 0, 1, 33], dtype=dtype, hq=hq, h=h, d=d, bs=bs, pad=pad, pos=pos, seed=d)
    cache = c.device_cache(layout)
    before = _lib.skipped_pairs(DEV)
    q = c.q.to(DEV)
    q_out = torch.full_like(q, 5.0)
    got = append_paged_kv(cache, c.k.to(DEV), c.v.to(DEV), c.batch(), 1e4, query=q, query_out=q_out,
                          rotary_style=style, layout=layout)
    assert got is cache and _lib.skipped_pairs(DEV) == before
    want = c.cache.double()
    exact = op.rotate(c.k, c.positions, 1e4, style)
    places = op.rows_of(c.tables, c.cu, c.positions, bs, c.nb)
    tol = torch.zeros_like(want)
    k_tol = rope_tolerance(c.k, exact, style, U[dtype])
    for t, at in enumerate(places):
        if at is not None:
            want[at[1], 0, :, at[2]], want[at[1], 1, :, at[2]] = exact[t], c.v[t].double()
            tol[at[1], 0, :, at[2]] = k_tol[t]
    diff = (op.from_layout(cache.cpu(), layout).double() - want).abs()
    assert torch.all(diff <= tol), float((diff - tol).max())  # V and every other row bit for bit
    n = c.cu[-1]
    exact = op.rotate(c.q, c.positions, 1e4, style)
    diff = (q_out.cpu().double() - exact).abs()[:n]
    assert torch.all(diff <= rope_tolerance(c.q, exact, style, U[dtype])[:n])
    assert torch.all(q_out[n:] == 5.0) and torch.equal(q.cpu(), c.q)


def test_append_without_rotation_in_place_query_and_strided_rows():
    c = Case(ctx=[50, 20], new=[9, 20], dtype=HF, hq=4, h=2, d=64, seed=3)
    fused = torch.randn(c.T, 8, 64, generator=torch.Generator().manual_seed(4)).to(HF)
    dev = fused.to(DEV)
    cache = c.device_cache()
    append_paged_kv(cache, dev[:, 4:6], dev[:, 6:], c.batch(), None)
    want = c.cache.clone()
    op.append(want, fused[:, 4:6], fused[:, 6:], c.tables, c.cu, c.positions, None, "neox")
    assert torch.equal(cache.cpu(), want)
    append_paged_kv(cache, dev[:, 4:6], dev[:, 6:], c.batch(), 1e6, query=dev[:, :4], query_out=dev[:, :4],
                    rotary_style="neox")
    exact = op.rotate(fused[:, :4], c.positions, 1e6, "neox")
    diff = (dev[:, :4].cpu().double() - exact).abs()
    assert torch.all(diff <= rope_tolerance(fused[:, :4], exact, "neox", U[HF]))
    assert torch.equal(dev[:, 4:].cpu(), fused[:, 4:])


def test_append_unaligned_rows():
    """Rows that start at odd element offsets take the narrow path."""
    c = Case(ctx=[20], new=[20], dtype=BF, hq=2, h=1, d=64, seed=5)
    wide = torch.randn(c.T, 1, 67, generator=torch.Generator().manual_seed(5)).to(BF)
    cache = c.device_cache()
    append_paged_kv(cache, wide.to(DEV)[..., 3:], wide.to(DEV)[..., 1:65], c.batch(), None)
    want = c.cache.clone()
    op.append(want, wide[..., 3:], wide[..., 1:65], c.tables, c.cu, c.positions, None, "neox")
    assert torch.equal(cache.cpu(), want)


@pytest.mark.parametrize("position", [5, 131071, 3_000_000, (1 << 31) + 12345])
def test_far_positions_keep_their_angle(position):
    """fp32 angles are off by 2^-24 * position radians; the 64-bit ones are not."""
    q = torch.randn(1, 3, 128, generator=torch.Generator().manual_seed(1))
    k = torch.randn(1, 1, 128, generator=torch.Generator().manual_seed(2))
    cache = torch.zeros(2, 2, 1, 16, 128, device=DEV)
    batch = PagedBatch(torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                       torch.tensor([position], device=DEV))
    out = torch.empty_like(q, device=DEV)
    before = _lib.skipped_pairs(DEV)
    append_paged_kv(cache, k.to(DEV), k.to(DEV), batch, 1e6, query=q.to(DEV), query_out=out, rotary_style="neox")
    exact = op.rotate(q, torch.tensor([position]), 1e6, "neox")
    # the 64-bit angle itself is within 2^-52 of its size
    tol = rope_tolerance(q, exact, "neox", U[FP]) + 2.0**-50 * position * q.abs().max()
    assert torch.all((out.cpu().double() - exact).abs() <= tol)
    assert _lib.skipped_pairs(DEV) - before == (0 if position < 16 else 1)
    assert bool((cache != 0).any()) == (position < 16)


def test_bad_pages_are_skipped_and_counted():
    c = Case(ctx=[64, 64], new=[40, 40], dtype=BF, h=2, d=64, seed=7, pad=2, table=torch.int64)
    c.tables[0, 2] = -1
    c.tables[1, 1] = c.nb  # one past the pool
    c.tables[1, 3] = 1 << 40
    c.positions = c.positions.clone()
    c.positions[3] = -5
    c.positions[50] = 64  # behind the table
    for four in (False, True):
        before = _lib.skipped_pairs(DEV)
        if four:
            c.group = 32
            c.codes, c.scales = op.quantise(c.cache.double(), 32)
            cache = c.device_cache()
            append_paged_kv(cache, c.k.to(DEV), c.v.to(DEV), c.batch(), 1e4)
            skipped = op.append4(c.codes, c.scales, c.k, c.v, c.tables, c.cu, c.positions, 1e4, "interleaved")
            assert torch.equal(op.unpack(cache.codes.cpu()), c.codes) and torch.equal(cache.scales.cpu(), c.scales)
        else:
            cache = c.device_cache()
            append_paged_kv(cache, c.k.to(DEV), c.v.to(DEV), c.batch(), None)
            skipped = op.append(c.cache, c.k, c.v, c.tables, c.cu, c.positions, None, "neox")
            assert torch.equal(cache.cpu(), c.cache)
        assert skipped > 10 and _lib.skipped_pairs(DEV) - before == skipped
        out = torch.full((2, c.h, c.T, c.d), 3.0, dtype=BF, device=DEV)
        gather_paged_kv(cache, c.batch(), out=out)
        assert _lib.skipped_pairs(DEV) - before == 2 * skipped
        src = c.value_cache()
        for t, at in enumerate(op.rows_of(c.tables, c.cu, c.positions, c.bs, c.nb)):
            if at is None or at[1] < 0:
                assert torch.all(out[:, :, t] == 3.0)
            else:
                assert torch.equal(out[:, :, t].cpu(), src[at[1], :, :, at[2]].float().to(BF))


# --------------------------------------------------------------------------- 4-bit rows


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("d,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("style,layout", [("neox", "canonical"), ("interleaved", "vllm"), ("neox", "trtllm")])
def test_append4_codes(dtype, d, group, style, layout):
    """Codes, steps and zeros equal the definition's bit for bit; other rows stay."""
    c = Case(ctx=[300, 5, 70], new=[120, 0, 70], dtype=dtype, hq=4, h=3, d=d, bs=8, group=group, seed=group, pad=2)
    cache = c.device_cache(layout)
    q_out = torch.full((c.T, 4, d), 2.0, dtype=dtype, device=DEV)
    append_paged_kv(cache, c.k.to(DEV), c.v.to(DEV), c.batch(), 5e5, query=c.q.to(DEV), query_out=q_out,
                    rotary_style=style, layout=layout)
    op.append4(c.codes, c.scales, c.k, c.v, c.tables, c.cu, c.positions, 5e5, style)
    assert torch.equal(op.from_layout(cache.scales.cpu(), layout), c.scales)
    assert torch.equal(op.unpack(op.from_layout(cache.codes.cpu(), layout)), c.codes)
    n = c.cu[-1]
    exact = op.rotate(c.q, c.positions, 5e5, style)
    assert torch.all((q_out.cpu().double() - exact).abs()[:n] <= rope_tolerance(c.q, exact, style, U[dtype])[:n])
    assert torch.all(q_out[n:] == 2.0)
    for out_dtype in (BF, HF, FP):
        back = gather_paged_kv(cache, c.batch(), dtype=out_dtype)
        assert back.dtype == out_dtype and torch.all(back[:, :, n:] == 0)
        vals = op.values(c.codes, c.scales)
        want = torch.stack([vals[b, :, :, o] for _, b, o in op.rows_of(c.tables, c.cu, c.positions, c.bs, c.nb)[:n]])
        # code * step is exact in fp32, so there is one rounding to fp32 and one to the type
        assert torch.equal(back[:, :, :n].cpu().permute(2, 0, 1, 3), want.float().to(out_dtype))


def test_append4_odd_groups():
    """Equal values, steps that vanish, values beyond fp16, infinities and NaN."""
    d, group = 64, 32
    rows = torch.randn(8, 1, d, generator=torch.Generator().manual_seed(0))
    rows[0] = 0.0
    rows[1] = -3.25
    rows[2, 0, 5] = 1e6  # saturates
    rows[3] *= 1e-9  # the step is below fp16's smallest
    rows[4, 0, 40] = float("nan")
    rows[5, 0, 2] = -1e30
    rows[6] = torch.linspace(0, 15, 32).repeat(2)  # step 1, zero 0
    rows[7] = rows[6] + 0.5  # step 1, zero 0.5
    cache = Int4KVCache.allocate(1, 1, 8, d, group=group)
    batch = PagedBatch(torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 8], dtype=torch.int32, device=DEV),
                       torch.arange(8, device=DEV))
    append_paged_kv(cache, rows.to(DEV), rows.to(DEV), batch, None)
    codes, scales = op.quantise(rows, group)
    got = gather_paged_kv(cache, batch, dtype=FP).cpu()
    want = op.values(codes, scales).float()
    for kv in (0, 1):
        assert torch.equal(op.unpack(cache.codes.cpu())[0, kv, 0], codes[:, 0])
        assert torch.equal(cache.scales.cpu()[0, kv, 0].nan_to_num(9.0), scales[:, 0].nan_to_num(9.0))
        assert torch.equal(got[kv, 0].nan_to_num(9.0), want[:, 0].nan_to_num(9.0))
    assert torch.equal(got[0, 0, 1], rows[1, 0]) and torch.equal(got[0, 0, 6], rows[6, 0].round())
    assert got[0, 0, 4, 32:].isnan().all() and not got[0, 0, 4, :32].isnan().any()


# --------------------------------------------------------------------------- attention

SHAPES = [  # hq, h, d, bs, layout
    (8, 2, 128, 16, "canonical"),
    (7, 1, 128, 16, "vllm"),
    (6, 6, 64, 32, "trtllm"),
    (16, 1, 64, 8, "canonical"),
    (40, 2, 128, 64, "canonical"),
]
ODD = [(3, 3, 80, 16, "canonical"), (4, 2, 256, 16, "trtllm"), (2, 1, 17, 5, "vllm"), (4, 2, 128, 7, "canonical"),
       (2, 1, 64, 1, "canonical")]
MASKS = [(None, 0), (1, 0), (33, 4), (100, 130), (4096, 4)]


@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("dtype,group", [(BF, None), (HF, None), (FP, None), (BF, 64), (HF, 32), (FP, 64), (BF, "D")])
@pytest.mark.parametrize("hq,h,d,bs,layout", SHAPES)
def test_attention_decode(hq, h, d, bs, layout, dtype, group, window, sinks):
    """One new token each over contexts around page, tile and window borders."""
    ctx = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 517]
    c = Case(ctx=ctx, new=[1] * len(ctx), dtype=dtype, hq=hq, h=h, d=d, bs=bs, group=d if group == "D" else group, seed=hq)
    attend(c, layout, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("dtype,group", [(BF, None), (HF, None), (BF, 64), (HF, 32)])
@pytest.mark.parametrize("hq,h,d,bs,layout", SHAPES)
def test_attention_chunks(hq, h, d, bs, layout, dtype, group, window, sinks):
    """Chunks of several tokens, idle requests, whole prompts and padding."""
    c = Case(ctx=[200, 30, 1, 64, 333], new=[37, 0, 1, 64, 100], dtype=dtype, hq=hq, h=h, d=d, bs=bs, group=group,
             seed=d + hq, pad=3, pos=torch.int64, table=torch.int64)
    attend(c, layout, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,h,d,bs,layout", ODD)
def test_attention_odd_shapes(hq, h, d, bs, layout, dtype, window, sinks):
    c = Case(ctx=[90, 3, 41], new=[20, 1, 2], dtype=dtype, hq=hq, h=h, d=d, bs=bs, seed=bs)
    attend(c, layout, window=window, sinks=sinks)


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("hq,h", [(28, 4), (4, 4)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 4), (64, 300)])
def test_attention_scattered_rows(hq, h, group, window, sinks):
    """The rows of a partial prefill: scattered positions, many tiles."""
    c = Case(ctx=[900, 400], new=[230, 90], hq=hq, h=h, d=128, group=group, seed=11, spread=True)
    attend(c, window=window, sinks=sinks)


@pytest.mark.parametrize("group", [None, 64])
def test_attention_unordered_positions(group):
    c = Case(ctx=[500, 300], new=[130, 40], hq=8, h=2, group=group, seed=12, spread=True)
    order = torch.cat([torch.randperm(130), 130 + torch.randperm(40)])
    c.positions = c.positions[order]
    attend(c, window=70, sinks=2)


@pytest.mark.parametrize("group", [None, 32, 64, 128])
@pytest.mark.parametrize("new", [1, 4, 300])
@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -float("inf")])
def test_unseen_rows_do_not_matter(group, new, stale):
    """Rows no request holds (freed pages, the rest of a last page) hold NaN or infinities."""
    c = Case(ctx=[1 + 16 * 20 + 5, 301, 311], new=[min(new, 326), min(new, 301), 1], hq=8, h=2, group=group, seed=13,
             stale=stale)
    attend(c, window=None)
    attend(c, window=50, sinks=4)


@pytest.mark.parametrize("new", [1, 2, 16, 200])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_rows_another_token_sees_do_not_leak(new, dtype):
    """A NaN or infinite V (or K) row inside the context reaches exactly the tokens that see it."""
    c = Case(ctx=[400], new=[new], hq=4, h=1, dtype=dtype, seed=14)
    bad = [400 - new - 30, 400 - new // 2 - 1, 399]
    for j, what, kv in zip(bad, (float("nan"), float("inf"), float("nan")), (1, 1, 0)):
        c.cache[int(c.tables[0, j // 16]), kv, 0, j % 16, 3] = what
    out = paged_attention(c.q.to(DEV), c.device_cache(), c.batch(), window=20, out=None).cpu()
    keep = [t for t in range(new) if not any(int(c.positions[t]) - 20 < j <= int(c.positions[t]) for j in bad)]
    hit = [t for t in range(new) if t not in keep]
    assert all(not torch.isfinite(out[t].float()).all() for t in hit)
    if keep:
        want, spread, reach = op.attention(c.q[keep], c.cache, c.tables, [0, len(keep)], c.positions[keep], 20)
        tol = U[dtype] * want.abs() + (U[dtype] + 2.0**-12) * spread
        assert torch.all((out[keep].double() - want).abs() <= tol)


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("new", [1, 40])
def test_tokens_that_see_nothing_are_zero(group, new):
    """Positions below zero, unmapped windows and empty tables."""
    c = Case(ctx=[200, 100], new=[new, new], hq=4, h=2, group=group, seed=15, table=torch.int64)
    c.positions[0] = -1
    c.tables[1, :] = -1  # every page of the second request
    attend(c, window=10)
    batch = PagedBatch(torch.zeros(2, 0, dtype=torch.int32, device=DEV), c.batch().cu_seqlens, c.positions.to(DEV))
    out = paged_attention(c.q.to(DEV), c.device_cache(), batch)
    assert torch.all(out == 0)


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("new", [1, 70])
def test_unmapped_pages_inside_the_context(group, new):
    c = Case(ctx=[300, 300], new=[new, new], hq=8, h=2, group=group, seed=16, table=torch.int64)
    c.tables[0, 3] = -1
    c.tables[0, 17] = c.nb + 5
    c.tables[1, 0] = 1 << 40
    attend(c)
    attend(c, window=200, sinks=5)


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("scale", [0.0, -0.1, 2.5])
def test_scales(group, scale):
    c = Case(ctx=[260, 90], new=[1, 33], hq=8, h=2, group=group, seed=17)
    attend(c, scale=scale)


@pytest.mark.parametrize("group", [None, 64])
def test_large_scores(group):
    """Scores in the hundreds, growing along the context: the running maximum moves at every tile."""
    c = Case(ctx=[700, 650], new=[1, 200], hq=8, h=2, group=None, seed=18)
    ramp = torch.zeros(c.nb, c.bs)
    for b, n in enumerate(c.ctx):
        for j in range(n):
            ramp[int(c.tables[b, j // c.bs]), j % c.bs] = j / 700
    q = c.q.float()
    c.cache[:, 0] = (c.cache[:, 0].float() + 2 * ramp[:, None, :, None] * q[0, 0]).to(BF)
    if group is not None:
        c.group = group
        c.codes, c.scales = op.quantise(c.cache.double(), group)
    attend(c, scale=0.7)


def test_strided_query_out_and_table():
    c = Case(ctx=[150, 80], new=[30, 1], hq=4, h=2, d=128, seed=19)
    big = torch.zeros(c.T, 12, 128, dtype=BF, device=DEV)
    big[:, 2:6] = c.q.to(DEV)
    out = torch.full((c.T, 4, 300), 7.0, dtype=BF, device=DEV)[..., 100:228]
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    wide[:, 3 : 3 + c.tables.shape[1]] = c.tables.to(DEV)
    cache = torch.zeros(c.nb, 2, 2, 16, 136, dtype=BF, device=DEV)[..., :128]  # rows with a gap between them
    cache.copy_(c.cache)
    batch = PagedBatch(wide[:, 3 : 3 + c.tables.shape[1]], c.batch().cu_seqlens, c.positions.to(DEV))
    paged_attention(big[:, 2:6], cache, batch, window=60, out=out)
    check_attention(c, out, window=60)


def test_unaligned_rows_take_the_plain_path():
    c = Case(ctx=[150, 80], new=[5, 1], hq=4, h=2, d=64, seed=20)
    q = torch.zeros(c.T, 4, 67, dtype=BF, device=DEV)
    q[..., 3:] = c.q.to(DEV)
    check_attention(c, paged_attention(q[..., 3:], c.device_cache(), c.batch()))
    cache = torch.zeros(c.nb, 2, 2, 16, 65, dtype=BF, device=DEV)
    cache[..., 1:] = c.cache.to(DEV)
    check_attention(c, paged_attention(c.q.to(DEV), cache[..., 1:], c.batch()))


@pytest.mark.parametrize("group", [None, 64])
def test_many_requests(group):
    """More requests than fit one pass over the batch, most of them idle."""
    B = 3000
    new = [1 if b % 7 == 0 else 0 for b in range(B)]
    ctx = [1 + (b * 13) % 90 if n else 1 for b, n in enumerate(new)]
    c = Case(ctx=ctx, new=new, hq=4, h=2, d=64, bs=16, group=group, seed=21)
    attend(c)


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("new", [1, 3, 200])
def test_long_context(group, new):
    """A context of many splits, checked on sampled rows."""
    c = Case(ctx=[9000, 40], new=[new, 1], hq=8, h=2, group=group, seed=22)
    attend(c) if new < 10 else attend(c, window=1000, sinks=64)


TILED = [(28, 4, 128, 16, "canonical"), (64, 8, 64, 32, "vllm"), (16, 16, 128, 128, "trtllm"),
         (32, 4, 128, 256, "canonical"), (40, 1, 64, 8, "canonical")]


@pytest.mark.parametrize("window,sinks", [(None, 0), (33, 4), (300, 130)])
@pytest.mark.parametrize("dtype,group", [(BF, None), (HF, None), (BF, 64), (HF, 32), (BF, "D")])
@pytest.mark.parametrize("hq,h,d,bs,layout", TILED)
def test_attention_many_rows(hq, h, d, bs, layout, dtype, group, window, sinks):
    """Enough rows for tiles of 128; pages below, at and above a block of 128 keys."""
    c = Case(ctx=[700, 513, 640, 1], new=[150, 97, 160, 0], dtype=dtype, hq=hq, h=h, d=d, bs=bs,
             group=d if group == "D" else group, seed=23, pad=2)
    attend(c, layout, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 4), (1500, 300)])
@pytest.mark.parametrize("dtype,group", [(BF, None), (HF, None), (BF, 64), (HF, 32)])
@pytest.mark.parametrize("hq,h,d,spread", [(28, 4, 128, False), (28, 4, 128, True), (16, 16, 64, False)])
def test_attention_cut_along_the_keys(hq, h, d, spread, dtype, group, window, sinks):
    """Few tiles over long contexts: each is cut into pieces, some without a key for a row."""
    c = Case(ctx=[2600, 1900, 1281], new=[150, 97, 130], dtype=dtype, hq=hq, h=h, d=d, group=group, seed=24,
             spread=spread)
    attend(c, window=window, sinks=sinks)


@pytest.mark.parametrize("group", [None, 64])
def test_cut_along_the_keys_with_holes(group):
    """Unmapped pages, a whole piece without any page, tokens that see nothing, positions in any order."""
    c = Case(ctx=[2600, 1900], new=[150, 97], hq=28, h=4, group=group, seed=25, spread=True, table=torch.int64)
    c.tables[0, 3] = -1
    c.tables[0, 40] = c.nb + 9
    c.tables[0, 64:130] = -1
    c.tables[1, :70] = -1
    c.positions[3] = -1
    c.positions[:150] = c.positions[torch.randperm(150)]
    attend(c)
    attend(c, window=900, sinks=70)
    c.tables[1, :] = -1
    attend(c)


@pytest.mark.parametrize("new", [200, 400])
def test_cut_along_the_keys_keeps_odd_values_apart(new):
    """Infinities and NaN of V and K reach exactly the tokens that see them."""
    c = Case(ctx=[2600], new=[new], hq=28, h=4, seed=26)
    clean = c.cache.clone()
    for j, what, kv in ((2450, float("inf"), 0), (2520, float("nan"), 0), (2580, float("nan"), 1)):
        at = int(c.tables[0, j // 16]), 1 - kv, 2, j % 16, 3
        c.cache[at], clean[at] = what, 0.0
    out = paged_attention(c.q.to(DEV), c.device_cache(), c.batch()).cpu().double()
    c.cache = clean
    want, spread, _ = op.attention(c.q, clean, c.tables, c.cu, c.positions)
    pos = c.positions
    heads = slice(14, 21)  # of KV head 2
    assert torch.all(out[(pos >= 2450) & (pos < 2520), heads, 3] == float("inf"))
    assert torch.all(out[(pos >= 2520) & (pos < 2580), heads, 3].isnan())
    assert torch.all(out[pos >= 2580, heads].isnan())
    ok = torch.ones_like(out, dtype=torch.bool)
    ok[pos >= 2450, heads, 3] = False
    ok[pos >= 2580, heads] = False
    tol = U[BF] * want.abs() + (U[BF] + 2.0**-12) * spread
    assert torch.all(((out - want).abs() <= tol)[ok])


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("new,d", [(1, 128), (3, 128), (180, 128), (40, 80)])
def test_out_may_be_the_query(new, d, group):
    """One token, a few, tiles cut along the keys, and the path of other head dims."""
    if d == 80 and group:
        pytest.skip("4-bit rows have 64 or 128 elements")
    c = Case(ctx=[1700, 1300], new=[new, new], hq=28, h=4, d=d, group=group, seed=27)
    q = c.q.to(DEV)
    assert paged_attention(q, c.device_cache(), c.batch(), window=1500, sinks=4, out=q) is q
    check_attention(c, q, window=1500, sinks=4)


def test_many_tiles_with_odd_values():
    """More tiles with a NaN in V than a CTA keeps a list of."""
    B, n, h, hq, d = 2600, 20, 8, 64, 64
    g = torch.Generator(device=DEV).manual_seed(28)
    cache = torch.randn(B, 2, h, 32, d, generator=g, device=DEV).to(BF)
    cache[:, 1, :, 5, 3] = float("nan")
    cache[:, :, :, n:] = float("inf")  # behind the last token
    q = torch.randn(B * n, hq, d, generator=g, device=DEV).to(BF)
    batch = PagedBatch(torch.randperm(B, generator=g, device=DEV).int()[:, None],
                       torch.arange(B + 1, dtype=torch.int32, device=DEV) * n,
                       torch.arange(n, dtype=torch.int32, device=DEV).repeat(B))
    out = paged_attention(q, cache, batch).view(B, n, hq, d)
    assert torch.all(out[:, :5].isfinite()) and torch.all(out[:, 5:, :, 3].isnan())
    out[..., 3] = 0
    assert torch.all(out.isfinite())
    assert torch.equal(out[:, 0, :, 4:], cache[batch.block_tables[:, 0].long(), 1, :, 0, 4:].repeat_interleave(8, 1))


@pytest.mark.parametrize("group", [None, 32])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_gather_into_rows_of_any_stride(group, offset):
    c = Case(ctx=[60, 33], new=[23, 33], hq=2, h=2, d=64, group=group, seed=29)
    wide = torch.full((2, c.h, c.T, 70), 5.0, dtype=BF, device=DEV)
    out = wide[..., offset : offset + 64]
    gather_paged_kv(c.device_cache(), c.batch(), out=out)
    src = c.value_cache()
    for t, (_, page, row) in enumerate(op.rows_of(c.tables, c.cu, c.positions, c.bs, c.nb)):
        assert torch.equal(out[:, :, t].cpu(), src[page, :, :, row].float().to(BF))
    rest = torch.cat([wide[..., :offset], wide[..., offset + 64 :]], -1)
    assert torch.all(rest == 5.0)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_append4_unaligned_rows_and_query_in_place(dtype):
    c = Case(ctx=[70, 20], new=[33, 20], dtype=dtype, hq=3, h=1, d=64, group=32, seed=30)
    fused = torch.randn(c.T, 5, 67, generator=torch.Generator().manual_seed(31)).to(dtype)
    dev = fused.to(DEV)
    cache = c.device_cache()
    append_paged_kv(cache, dev[:, 3:4, 3:], dev[:, 4:, 1:65], c.batch(), 1e5, query=dev[:, :3, 2:66],
                    query_out=dev[:, :3, 2:66], rotary_style="neox")
    assert op.append4(c.codes, c.scales, fused[:, 3:4, 3:], fused[:, 4:, 1:65], c.tables, c.cu, c.positions, 1e5,
                      "neox") == 0
    assert torch.equal(op.unpack(cache.codes.cpu()), c.codes) and torch.equal(cache.scales.cpu(), c.scales)
    exact = op.rotate(fused[:, :3, 2:66], c.positions, 1e5, "neox")
    diff = (dev[:, :3, 2:66].cpu().double() - exact).abs()
    assert torch.all(diff <= rope_tolerance(fused[:, :3, 2:66], exact, "neox", U[dtype]))
    dev[:, :3, 2:66] = fused[:, :3, 2:66].to(DEV)
    assert torch.equal(dev.cpu(), fused)


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("new", [1, 2, 180])
def test_wide_table_and_short_window(new, group):
    """A table far wider than the contexts, a window of a few tiles: what is cut follows the window."""
    c = Case(ctx=[1500, 900], new=[new, new], hq=28, h=4, group=group, seed=32)
    c.tables = torch.cat([c.tables, torch.full((2, 2500), -1, dtype=c.tables.dtype)], 1)
    for window, sinks in ((None, 0), (200, 4), (1100, 200)):
        attend(c, window=window, sinks=sinks)


def test_rows_past_32_bits():
    """A pool whose rows lie more than 2^31 elements from its start."""
    h, d, bs = 1, 128, 16
    nb = (1 << 31) // (2 * h * bs * d) + 40
    cache = torch.zeros(nb, 2, h, bs, d, dtype=BF, device=DEV)
    c = Case(ctx=[64], new=[64], hq=2, h=h, d=d, seed=23)
    far = torch.tensor([[nb - 1, nb - 3, 0, nb - 20]], dtype=torch.int32, device=DEV)
    batch = PagedBatch(far, c.batch().cu_seqlens, c.positions.to(DEV))
    append_paged_kv(cache, c.k.to(DEV), c.v.to(DEV), batch, None)
    back = gather_paged_kv(cache, batch).cpu()
    assert torch.equal(back[0].transpose(0, 1), c.k) and torch.equal(back[1].transpose(0, 1), c.v)
    out = paged_attention(c.q.to(DEV), cache, batch)
    c.tables = torch.arange(4)[None]
    c.nb = 4
    c.cache = torch.stack([c.k, c.v]).view(2, 4, 16, h, d).permute(1, 0, 3, 2, 4)
    check_attention(c, out)


# --------------------------------------------------------------------------- together


@pytest.mark.parametrize("four", [False, True])
def test_inject_append_attend(four):
    """A partial prefill on one cache: donor rows injected (or gathered, moved
    and injected from 4 bits), recomputed rows appended, attention from the
    pages; against attention over the same K and V held densely."""
    g = torch.Generator().manual_seed(31)
    S, h, hq, d, bs, base = 256, 2, 8, 128, 16, 1e4
    rows = torch.randn(2, S, h, d, generator=g).to(BF)
    q = torch.randn(S, hq, d, generator=g).to(BF)
    mask = torch.zeros(S, dtype=torch.bool)
    mask[40:70] = True
    mask[-20:] = True
    reuse, fresh = torch.where(~mask)[0], torch.where(mask)[0]
    table = torch.randperm(32, generator=g)[:16].to(torch.int32)[None].to(DEV)
    shift = 64  # the donor held the reused rows 64 positions later
    donor_pos = reuse + shift
    donor = torch.zeros(2, h, S + shift, d, dtype=BF)
    donor[0][:, donor_pos] = op.rotate(rows[0, reuse], donor_pos, base, "neox").to(BF).transpose(0, 1)
    donor[1][:, donor_pos] = rows[1, reuse].transpose(0, 1)
    cache = torch.zeros(32, 2, h, bs, d, dtype=BF, device=DEV)
    rc.rope_correct_scatter_paged(cache, donor.to(DEV), table[0], donor_pos.to(DEV), reuse.to(DEV), base,
                                  rotary_style="neox")
    batch = PagedBatch(table, torch.tensor([0, len(fresh)], dtype=torch.int32, device=DEV), fresh.to(DEV))
    k, v, qd = rows[0, fresh].to(DEV), rows[1, fresh].to(DEV), q[fresh].to(DEV)
    q_rot = torch.empty_like(qd)
    append_paged_kv(cache, k, v, batch, base, query=qd, query_out=q_rot, rotary_style="neox")
    every = PagedBatch(table, torch.tensor([0, S], dtype=torch.int32, device=DEV), torch.arange(S, device=DEV))
    dense = gather_paged_kv(cache, every)
    if four:
        held = Int4KVCache.allocate(32, h, bs, d, group=64)
        append_paged_kv(held, dense[0].transpose(0, 1), dense[1].transpose(0, 1), every, None)
        dense = gather_paged_kv(held, every)
        out = paged_attention(q_rot, held, batch)
    else:
        out = paged_attention(q_rot, cache, batch)
        want_k = op.rotate(rows[0], torch.arange(S), base, "neox")
        # two rotations and roundings of a reused row (fp32 angles in the inject), one of a fresh row
        assert (dense[0].cpu().transpose(0, 1).double() - want_k).abs().max() <= 3 * U[BF] * want_k.abs().max()
    full = torch.zeros(hq, S, d, dtype=BF, device=DEV)
    full[:, fresh.to(DEV)] = q_rot.transpose(0, 1)
    want = partial_prefill_attention(full, dense[0], dense[1], mask.to(DEV))[:, fresh.to(DEV)].transpose(0, 1)
    # each side rounds its probabilities and its result once; the dense values of 4-bit rows are rounded too
    spread = dense[1].abs().float().max().item()
    assert (out.float() - want.float()).abs().max().item() <= (6 if four else 4) * U[BF] * spread


@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("new", [1, 150])
def test_captured_and_replayed(group, new):
    """A captured step follows what its tensors hold at replay, beside eager calls."""
    c = Case(ctx=[400, 300], new=[new, new], hq=8, h=2, group=group, seed=41)
    cache, q, k, v = c.device_cache(), c.q.to(DEV), c.k.to(DEV), c.v.to(DEV)
    tables, cu, pos = c.tables.to(DEV), torch.tensor(c.cu, dtype=torch.int32, device=DEV), c.positions.to(DEV)
    batch = PagedBatch(tables, cu, pos)
    out, q_rot = torch.zeros_like(q), torch.zeros_like(q)

    def step():
        append_paged_kv(cache, k, v, batch, 1e4, query=q, query_out=q_rot)
        paged_attention(q_rot, cache, batch, window=90, sinks=4, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    eager = out.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for g in graphs:
        out.zero_()
        g.replay()
        assert torch.equal(out, eager)
    # other positions and values through the same graph
    pos.sub_(17)
    q.copy_(torch.flip(q, [0]))
    graphs[0].replay()
    got = out.clone()
    step()
    assert torch.equal(out, got) and not torch.equal(got, eager)


@pytest.mark.parametrize("group", [None, 64])
def test_two_streams_at_once(group):
    """Calls that overlap on two streams keep their own workspaces."""
    cases = [Case(ctx=[3000, 900], new=[n, 1], hq=8, h=2, group=group, seed=50 + n) for n in (1, 160)]
    state = [(c.q.to(DEV), c.device_cache(), c.batch(), torch.zeros_like(c.q, device=DEV)) for c in cases]
    want = [paged_attention(q, cache, b, out=o).clone() for q, cache, b, o in state]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (q, cache, b, o) in zip(streams, state):
            with torch.cuda.stream(s):
                paged_attention(q, cache, b, out=o)
    torch.cuda.synchronize()
    for w, (_, _, _, o) in zip(want, state):
        assert torch.equal(w, o)


def test_same_call_gives_the_same_bits():
    c = Case(ctx=[2500, 700, 64], new=[1, 1, 1], hq=8, h=2, seed=60)
    q, cache, b = c.q.to(DEV), c.device_cache(), c.batch()
    first = paged_attention(q, cache, b)
    for _ in range(5):
        assert torch.equal(paged_attention(q, cache, b), first)


# --------------------------------------------------------------------------- refusals


def test_refusals():
    c = Case(ctx=[20, 10], new=[2, 1], hq=4, h=2, d=64)
    q, cache, b, k = c.q.to(DEV), c.device_cache(), c.batch(), c.k.to(DEV)
    tables, cu, pos = b.block_tables, b.cu_seqlens, b.positions
    ok = torch.zeros_like(q)
    with pytest.raises(ValueError):
        PagedBatch(tables[0], cu, pos)
    with pytest.raises(ValueError):
        PagedBatch(tables, cu[:-1], pos)
    with pytest.raises(ValueError):
        PagedBatch(tables, cu, pos[None])
    with pytest.raises(ValueError):
        PagedBatch(tables[:1].expand(2, -1), cu, pos)
    with pytest.raises(TypeError):
        PagedBatch(tables, cu.long(), pos)
    with pytest.raises(TypeError):
        PagedBatch(tables.float(), cu, pos)
    with pytest.raises(_lib.NativeLibraryError):
        PagedBatch(tables.cpu(), cu, pos)
    for bad in (dict(window=0), dict(window=-3), dict(sinks=-1), dict(scale=float("nan")), dict(out=ok[:2]),
                dict(layout="trtllm"), dict(out=ok[:1].expand(3, -1, -1)), dict(out=ok[..., :32])):
        with pytest.raises(ValueError):
            paged_attention(q, cache, b, **bad)
    with pytest.raises(ValueError):
        paged_attention(q[:, :3], cache, b)  # 3 heads over 2
    with pytest.raises(ValueError):
        paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache, b)
    for bad in (q.half(), q.float()):
        with pytest.raises(TypeError):
            paged_attention(bad, cache, b)
    with pytest.raises(TypeError):
        paged_attention(q, cache, b, out=ok.half())
    with pytest.raises(TypeError):
        paged_attention(q, cache.double(), b)
    with pytest.raises(TypeError):
        paged_attention(q, cache, b, status=torch.zeros(1, device=DEV))
    with pytest.raises(_lib.NativeLibraryError):
        paged_attention(c.q, cache, b)
    with pytest.raises(ValueError):
        append_paged_kv(cache, k[:2], k, b)
    with pytest.raises(TypeError):
        append_paged_kv(cache, k, k.half(), b)
    with pytest.raises(ValueError):
        append_paged_kv(cache, k, k, b, query=q)
    with pytest.raises(ValueError):
        append_paged_kv(cache, k, k, b, rotary_style="gptj")
    with pytest.raises(TypeError):
        gather_paged_kv(cache, b, dtype=HF)
    with pytest.raises(ValueError):
        gather_paged_kv(cache, b, out=torch.zeros(2, 2, 3, 32, dtype=BF, device=DEV))
    held = Int4KVCache.allocate(4, 2, 16, 64, group=32, layout="vllm")
    with pytest.raises(ValueError):
        paged_attention(q, held, b, layout="trtllm")
    for dim, group in ((96, 32), (64, 128), (128, 16)):
        with pytest.raises(ValueError):
            Int4KVCache.allocate(4, 2, 16, dim, group=group)
    with pytest.raises(TypeError):
        Int4KVCache(held.codes.int(), held.scales, layout="vllm")
    with pytest.raises(ValueError):
        Int4KVCache(held.codes, held.scales[..., :1, :], layout="canonical")
    with pytest.raises(ValueError):
        Int4KVCache(held.codes.transpose(2, 4), held.scales, layout="vllm")
    with pytest.raises(_lib.NativeLibraryError):
        Int4KVCache.allocate(4, 2, 16, 64, device="cpu")


def test_empty_batches():
    cache = torch.ones(4, 2, 2, 16, 64, dtype=BF, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    rows = torch.zeros(0, 2, 64, dtype=BF, device=DEV)
    for tables, cu in ((torch.zeros(0, 3), [0]), (torch.zeros(2, 3), [0, 0, 0])):
        b = PagedBatch(tables.int().to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), none)
        append_paged_kv(cache, rows, rows, b)
        assert gather_paged_kv(cache, b).shape == (2, 2, 0, 64)
        assert paged_attention(rows, cache, b).shape == (0, 2, 64)
    assert torch.all(cache == 1)
    # tokens, but no sequence that holds them
    b = PagedBatch(torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV),
                   torch.zeros(5, dtype=torch.int32, device=DEV))
    q = torch.ones(5, 2, 64, dtype=BF, device=DEV)
    append_paged_kv(cache, q, q, b)
    assert torch.all(cache == 1) and torch.all(paged_attention(q, cache, b) == 0)
    out = torch.full_like(q, 4.0)
    assert torch.all(paged_attention(q, cache, b, out=out) == 4.0)
