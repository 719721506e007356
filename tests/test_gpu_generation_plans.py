"""Attention over a paged cache at sizes that fill the chip: every choice of
blocks, wave groups and parts that the planner makes, each named by its test so
that other thresholds cannot leave one untested."""
from __future__ import annotations

import math

import pytest
import torch

from lzhip import _lib, ops
from test_gpu_generation import BF16, DEV, F16, F32, MUCH, U32, Case, _u

pytestmark = pytest.mark.gpu
CODE = {F32: 0, BF16: 1, F16: 2}
TYPES = [(BF16, False), (F16, False), (BF16, True), (F16, True)]


def _plan(c, H):
    """(packed rows of a block, wave groups, parts)"""
    s, code = c.step, CODE[c.dtype]
    p = _lib.query("lz_paged_attn_plan", code, 8 if c.e4m3 else code, c.rows, len(c.seqs), H, c.KV, c.hd, s.max_new, s.max_len)
    return p & 255, p >> 8 & 255, p >> 16


def _reference(c, q, H, scale, hidden=()):
    """(o, bound) in float64, a kv head at a time; hidden: pages of the
    sequences' tables that hold nothing.  Bound as in Case.attention, with the
    weights in two terms (u^2 of them) or, in fp32, as they are."""
    G = H // c.KV
    q = q.double().view(-1, c.KV, G, c.hd)
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    weights = _u(c.dtype) ** 2 if c.dtype != F32 else 0.0
    for b, (n, l) in enumerate(c.seqs):
        if n == 0 or l == 0:
            continue
        k, v = c.tokens(0, b), c.tokens(1, b)
        pos = torch.arange(l)
        seen = pos[None] <= torch.arange(l - n, l)[:, None]
        for page in hidden:
            seen = seen & (pos // c.page != page)
        count = seen.sum(1)
        for g in range(c.KV):
            x = q[c.starts[b] : c.starts[b] + n, g]
            s = (x.reshape(n * G, c.hd) @ k[:, g].T).view(n, G, l) * scale
            p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1).nan_to_num(0.0).view(n * G, l)
            size = (x.abs().reshape(n * G, c.hd) @ k[:, g].abs().T).view(n, G, l).masked_fill(~seen[:, None], 0.0).amax(-1) * scale
            y, a = (p @ t for t in (v[:, g], v[:, g].abs()))
            fp32 = (2 * (c.hd + 4) * size + 8 + 3 * count[:, None]) * U32
            rows = slice(c.starts[b], c.starts[b] + n)
            o[rows, g] = y.view(n, G, c.hd)
            tol[rows, g] = _u(c.dtype) * o[rows, g].abs() + (weights + fp32[..., None]) * a.view(n, G, c.hd)
    return o.view(-1, H * c.hd), tol.view(-1, H * c.hd)


CHUNKS = [(400, 500), (333, 333), (300, 1100), (257, 260), (129, 700)]
MIXED = [(1, 1 + 41 * b % 700) for b in range(30)] + [(700, 900)] + [(b % 3, 200 + b) for b in range(33)]  # 64 sequences
MANY = [(b % 37, b % 37 + 11 * b % 50) for b in range(70)]
PLANS = {
    # name: (sequences, query heads, kv heads, page, bound on the lengths, plan)
    "one group": (CHUNKS, 32, 8, 32, 0, (128, 1, 1)),
    "one group, equal": ([(352, 1500)] * 3, 32, 8, 64, 0, (128, 1, 1)),
    "one group, many sequences": (MANY, 16, 4, 16, MUCH, (128, 1, 1)),
    "one group, a chunk beside 63 others": (MIXED, 16, 8, 32, 0, (128, 1, 1)),
    "one group, a chunk beside 64 others": ([(1, 77)] + MIXED, 16, 8, 32, 0, (128, 1, 1)),
    "three parts": ([(600, 4200)], 32, 8, 64, 0, (128, 1, 3)),
    "two groups, a few more blocks than CUs": ([(1056, 1056)], 32, 8, 32, 0, (128, 2, 1)),
    "two groups": ([(600, 800)], 32, 8, 16, 0, (128, 2, 1)),
    "two groups, in parts": ([(200, 3000), (64, 100)], 16, 4, 32, 0, (128, 2, 6)),
}


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("dtype,e4m3", TYPES)
@pytest.mark.parametrize("name", sorted(PLANS))
def test_tiles(name, dtype, e4m3, hd):
    seqs, H, KV, page, most, plan = PLANS[name]
    c = Case(seqs, KV, hd, page, dtype, e4m3, seed=hd, most=most, fill=None if e4m3 else math.nan)
    assert _plan(c, H) == plan
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, hd**-0.5).cpu().double()
    want, tol = _reference(c, q, H, hd**-0.5)
    assert float(((got - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("dtype,e4m3", TYPES)
@pytest.mark.parametrize("name", ["one group", "three parts", "two groups, a few more blocks than CUs"])
def test_tiles_with_pages_that_are_not_there(name, dtype, e4m3):
    """Page ids outside the pool in every table: their tokens are left out."""
    seqs, H, KV, page, most, plan = PLANS[name]
    c = Case(seqs, KV, 64, page, dtype, e4m3, seed=5, most=most, fill=None if e4m3 else math.inf)
    hidden = (0, 5, 6)
    table = c.table.clone()
    for i, bad in zip(hidden, (-1, 10**7, -(2**31))):
        table[:, i] = bad
    assert _plan(c, H) == plan
    q = torch.randn(c.rows, H * 64, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.step._replace(page_table=table.to(DEV)), H, 0.125).cpu().double()
    want, tol = _reference(c, q, H, 0.125, hidden)
    assert float(((got - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("dtype,e4m3", TYPES)
@pytest.mark.parametrize("name", sorted(PLANS))
def test_tiles_nonfinite_reaches_only_who_sees_it(name, dtype, e4m3):
    """An infinity or NaN among the last new token's keys and values: the rows
    before it and the other sequences keep their bits."""
    seqs, H, KV, page, most, plan = PLANS[name]
    c = Case(seqs, KV, 64, page, dtype, e4m3, seed=6, most=most)
    q = torch.randn(c.rows, H * 64, generator=c.g).to(dtype).to(DEV)
    before = ops.paged_attention(q, c.layer, c.step, H, 0.125)
    b = max(range(len(seqs)), key=lambda i: seqs[i][0])
    p, last = seqs[b][1] - 1, c.starts[b + 1] - 1
    where, slot = int(c.table[b, p // page]), p % page
    c.layer.v[where, :, slot, 3:5] = torch.tensor(math.nan if e4m3 else math.inf, device=DEV).to(c.layer.v.dtype)
    c.layer.k[where, 1, slot, 2] = torch.tensor(math.nan, device=DEV).to(c.layer.k.dtype)
    after = ops.paged_attention(q, c.layer, c.step, H, 0.125)
    keep = torch.arange(c.rows, device=DEV) != last
    assert torch.equal(after[keep], before[keep])
    assert not torch.isfinite(after[last].view(H, 64)[:, 3:5]).any()


WAVES = {
    "whole, a block a CU and more": ([(1, 1 + 61 * b % 1500) for b in range(64)], 8, 8, 16, (16, 1, 1)),
    "four parts, a few more blocks than CUs": ([(1, 1 + 237 * b % 2048) for b in range(36)], 16, 8, 64, (16, 1, 4)),
    "many parts": ([(1, 9000), (1, 70)], 8, 4, 64, (16, 1, 29)),
    "short, whole": ([(1, 500), (3, 77)], 8, 4, 32, (16, 1, 1)),
    "blocks of 32": ([(40, 300), (7, 500)], 4, 4, 16, (32, 1, 1)),
}


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("dtype,e4m3", TYPES)
@pytest.mark.parametrize("name", sorted(WAVES))
def test_waves(name, dtype, e4m3, hd):
    seqs, H, KV, page, plan = WAVES[name]
    c = Case(seqs, KV, hd, page, dtype, e4m3, seed=hd, fill=None if e4m3 else math.nan)
    assert _plan(c, H) == plan
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, hd**-0.5).cpu().double()
    want, tol = _reference(c, q, H, hd**-0.5)
    assert float(((got - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("seqs,H,KV,plan", [
    ([(150, 300), (90, 700)], 12, 4, (32, 1, 2)),
    ([(200, 200), (77, 701)] * 4, 10, 10, (32, 1, 1)),
    ([(188, 2500), (20, 100)], 10, 2, (32, 1, 5)),
])
def test_fp32_chunks(seqs, H, KV, plan, e4m3, hd):
    c = Case(seqs, KV, hd, 16, F32, e4m3, seed=hd, fill=None if e4m3 else math.nan)
    assert _plan(c, H) == plan
    q = torch.randn(c.rows, H * hd, generator=c.g)
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, hd**-0.5).cpu().double()
    want, tol = _reference(c, q, H, hd**-0.5)
    assert float(((got - want).abs() - tol).max()) <= 0
