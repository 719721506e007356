"""Drafted tokens over a paged key/value cache: a step's tables made on the
device, attention of trees, verification and the move of kept branches, against
plain restatements on the CPU (float64 where numbers are computed).

Tolerances count roundings: u = finfo.eps / 2 of a type is the most that one
rounding to it changes a value, relative to it; u32 = 2^-24.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from lzhip import _lib, ops
from lzhip.cache import CacheStep, DraftStep, LayerCache, PageTables
from test_gpu_generation import BF16, DEV, E4M3, F16, F32, MUCH, U32, Case, _u

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def _closure(parents):
    """Ancestors (and itself) of each node, as sets; depths."""
    sets, depth = [], []
    for i, p in enumerate(parents):
        up = 0 <= p < i
        sets.append((sets[p] if up else set()) | {i})
        depth.append(depth[p] + 1 if up else 0)
    return sets, depth


def _pack(bits):
    """[rows, n] truth values -> int32 words, lowest bit first."""
    rows, n = bits.shape
    out = torch.zeros(rows, -(-n // 32), dtype=torch.int64)
    for j in range(n):
        out[:, j // 32] |= bits[:, j].long() << (j % 32)
    return out.to(torch.int32)


# ---------------------------------------------------------------------------
# attention of trees
# ---------------------------------------------------------------------------

def _seen(c, bases, bits):
    """[n, l] for each sequence: what its rows see."""
    out = []
    for b, (n, l) in enumerate(c.seqs):
        base = min(max(bases[b], 0), l)
        seen = torch.zeros(n, l, dtype=torch.bool)
        seen[:, :base] = True
        own = bits[c.starts[b] : c.starts[b + 1]]
        w = min(l - base, own.shape[1])
        seen[:, base : base + w] = own[:, :w]
        out.append(seen)
    return out


def _reference(c, q, H, scale, seen):
    """(o, bound) in float64.  Bound: one rounding of the output; the weights in
    two terms of the type (u^2 of them; none in fp32); and in fp32 the scores
    (their products' sum over hd, and the exponent's scaling), the sum of the
    weights and the second product's over the keys."""
    G = H // c.KV
    q = q.double().cpu().view(-1, c.KV, G, c.hd)
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    weights = _u(c.dtype) ** 2 if c.dtype != F32 else 0.0
    for b, (n, l) in enumerate(c.seqs):
        if n == 0 or l == 0:
            continue
        k, v, vis = c.tokens(0, b), c.tokens(1, b), seen[b]
        there = c.table[b, torch.arange(l) // c.page] >= 0
        vis = vis & there
        k, v = torch.where(there[:, None, None], k, 0.0), torch.where(there[:, None, None], v, 0.0)
        k, v = (torch.where(vis.any(0)[:, None, None], x, 0.0) for x in (k, v))  # what nobody sees may be NaN
        count = vis.sum(1)
        rows = slice(c.starts[b], c.starts[b] + n)
        for g in range(c.KV):
            x = q[rows, g].reshape(n * G, c.hd)
            s = (x @ k[:, g].T).view(n, G, l) * scale
            p = torch.softmax(s.masked_fill(~vis[:, None], -math.inf), -1).nan_to_num(0.0).view(n * G, l)
            size = (x.abs() @ k[:, g].abs().T).view(n, G, l).masked_fill(~vis[:, None], 0.0).amax(-1) * scale
            y, a = (p @ t for t in (v[:, g], v[:, g].abs()))
            fp32 = (2 * (c.hd + 4) * size + 8 + 3 * count[:, None]) * U32
            o[rows, g] = y.view(n, G, c.hd)
            tol[rows, g] = _u(c.dtype) * o[rows, g].abs() + (weights + fp32[..., None]) * a.view(n, G, c.hd)
    return o.view(-1, H * c.hd), tol.view(-1, H * c.hd)


def _tree_case(seqs, bases, KV, hd, page, dtype, e4m3=False, seed=0, words=None, fill=math.nan, most=0, density=0.4):
    """A Case whose rows see random bits of the places from the base on (no
    trees: any mask has to be right); the first row of a sequence sees none of
    them and its last one all."""
    c = Case(seqs, KV, hd, page, dtype, e4m3, seed=seed, fill=None if e4m3 else fill, most=most)
    span = max([1] + [l - min(max(a, 0), l) for (_, l), a in zip(seqs, bases)])
    words = -(-span // 32) if words is None else words
    bits = torch.rand(c.rows, 32 * words, generator=c.g) < density
    for b, (n, _) in enumerate(seqs):
        if n:
            bits[c.starts[b]] = False
            bits[c.starts[b + 1] - 1] = True
    s = c.step
    c.draft = DraftStep(s.row_start, s.kv_len, s.page_table, s.rows, s.max_new, s.max_len, _i32(bases),
                        torch.zeros(c.rows, dtype=torch.int32, device=DEV), torch.zeros(c.rows, dtype=torch.int64, device=DEV),
                        _pack(bits).to(DEV))
    return c, bits


TREES = {
    # sequences of (new, all) tokens, and the places that all rows see
    "one node": ([(1, 1)], [0]),
    "one node and a text": ([(1, 130)], [129]),
    "a few": ([(5, 17), (8, 8), (1, 33), (3, 64)], [12, 0, 32, 61]),
    "empty ones": ([(0, 0), (4, 20), (0, 50), (7, 7)], [0, 16, 50, 0]),
    "a word and more": ([(33, 40), (32, 300), (31, 31), (65, 129)], [7, 268, 0, 64]),
    "bases inside tiles": ([(12, 75), (12, 76), (12, 93), (20, 150)], [63, 60, 81, 97]),
    "levels of a tree": ([(6, 400), (9, 37)], [383, 5]),  # more places than rows behind the base
    "bases that are none": ([(6, 40), (6, 40), (6, 70)], [-3, 40, 1000]),
    "wide": ([(150, 700), (97, 97), (128, 260)], [550, 0, 132]),
}
TYPES = [(BF16, False), (F16, False), (F32, False), (BF16, True), (F16, True), (F32, True)]


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("dtype,e4m3", TYPES)
@pytest.mark.parametrize("name", sorted(TREES))
def test_tree_attention(name, dtype, e4m3, hd):
    seqs, bases = TREES[name]
    for (H, KV), page, most in (((4, 2), 16, 0), ((3, 3), 64, 0), ((8, 1), 32, MUCH), ((8, 2), 32, MUCH)):
        c, bits = _tree_case(seqs, bases, KV, hd, page, dtype, e4m3, seed=hd + page, most=most)
        q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
        scale = 1.3 / math.sqrt(hd)
        got = ops.paged_attention(q.to(DEV), c.layer, c.draft, H, scale).double().cpu()
        want, tol = _reference(c, q, H, scale, _seen(c, bases, bits))
        assert bool(((got - want).abs() <= tol).all()), (name, H, KV, page, float(((got - want).abs() - tol).max()))


LONG = {
    # sequences, bases, heads, bound on the lengths
    "two texts": ([(8, 5000), (3, 700)], [4990, 690], (16, 8), 0),
    "one text": ([(13, 3000)], [2950], (4, 2), 0),
    "wide trees": ([(160, 400)] * 9, [240] * 9, (32, 8), MUCH),
    "wide trees over long texts": ([(64, 3000), (20, 100)], [2930, 77], (16, 4), 0),
}


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True)])
@pytest.mark.parametrize("name", sorted(LONG))
def test_tree_attention_over_long_texts(name, dtype, e4m3, hd):
    """Texts that go in parts: the mask lies in the last of them, or over two."""
    seqs, bases, (H, KV), most = LONG[name]
    c, bits = _tree_case(seqs, bases, KV, hd, 64, dtype, e4m3, seed=hd, most=most)
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.draft, H, hd**-0.5).double().cpu()
    want, tol = _reference(c, q, H, hd**-0.5, _seen(c, bases, bits))
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("most", [0, MUCH])
def test_a_chain_as_a_tree_is_causal(dtype, most):
    """The mask of a chain leaves the bits of causal attention."""
    H, KV, hd = 8, 2, 64
    seqs = [(20, 90), (33, 33), (1, 5), (70, 300)]
    c = Case(seqs, KV, hd, 32, dtype, seed=3, most=most)
    bits = torch.zeros(c.rows, 96, dtype=torch.bool)
    for b, (n, _) in enumerate(seqs):
        bits[c.starts[b] : c.starts[b + 1], :n] = torch.ones(n, n).tril().bool()
    s = c.step
    draft = DraftStep(s.row_start, s.kv_len, s.page_table, s.rows, s.max_new, s.max_len, _i32([l - n for n, l in seqs]),
                      torch.zeros(c.rows, dtype=torch.int32, device=DEV), torch.zeros(c.rows, dtype=torch.int64, device=DEV),
                      _pack(bits).to(DEV))
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype).to(DEV)
    want = ops.paged_attention(q, c.layer, s, H, hd**-0.5)
    got = ops.paged_attention(q, c.layer, draft, H, hd**-0.5)
    reference, tol = _reference(c, q, H, hd**-0.5, _seen(c, [l - n for n, l in seqs], bits))
    assert bool(((got.double().cpu() - reference).abs() <= tol).all())
    assert bool(((got.double() - want.double()).abs().cpu() <= 2 * tol).all())
    none = draft._replace(mask=None)  # without a mask it is the causal call itself
    assert torch.equal(ops.paged_attention(q, c.layer, none, H, hd**-0.5), want)


@pytest.mark.parametrize("most", [0, MUCH])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_that_see_nothing_and_missing_pages(dtype, most):
    """Nothing seen: zeros, whatever lies in the places; scores that are all
    -inf: NaN; pages that are not there are not seen."""
    H, KV, hd = 8, 2, 64
    seqs, bases = [(34, 34), (40, 200)], [0, 160]
    c, bits = _tree_case(seqs, bases, KV, hd, 16, dtype, seed=11, most=most, fill=math.nan)
    bits[:34] = False
    bits[5, 3] = bits[9, 7] = True
    c.table[0, 0] = -1          # the page of places 0 .. 15 of sequence 0
    c.table[1, 10] = 10**6      # and of 160 .. 175 of sequence 1
    draft = c.draft._replace(mask=_pack(bits).to(DEV), page_table=c.table.to(DEV))
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    c.table[1, 10] = -1
    got = ops.paged_attention(q.to(DEV), c.layer, draft, H, hd**-0.5).double().cpu()
    want, tol = _reference(c, q, H, hd**-0.5, _seen(c, bases, bits))
    assert bool((got[:34] == 0).all())
    assert bool(((got - want).abs() <= tol).all())
    c.table[0, 0] = 0
    k = c.layer.k.clone()
    k[0] = -math.inf
    layer = LayerCache(k, torch.nan_to_num(c.layer.v))
    q = torch.rand(c.rows, H * hd, generator=c.g).to(dtype) + 0.5
    got = ops.paged_attention(q.to(DEV), layer, draft._replace(page_table=c.table.to(DEV)), H, hd**-0.5).float().cpu()
    assert bool(got[[5, 9]].isnan().all())  # they see one place each, whose score is -inf
    assert bool((got[[0, 1, 2, 3, 4, 6, 7, 8]] == 0).all())


@pytest.mark.parametrize("most", [0, MUCH])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("odd", [math.inf, math.nan])
def test_an_infinity_reaches_those_that_see_it(dtype, most, odd):
    H, KV, hd = 8, 2, 64
    seqs, bases = [(40, 90)], [50]
    c, bits = _tree_case(seqs, bases, KV, hd, 16, dtype, seed=5, most=most, fill=0.0)
    bits[:, 13] = torch.arange(40) % 3 == 0
    draft = c.draft._replace(mask=_pack(bits).to(DEV))
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype).to(DEV)
    clean = ops.paged_attention(q, c.layer, draft, H, hd**-0.5)
    v = c.layer.v.clone()
    page, place = int(c.table[0, 63 // 16]), 63 % 16
    v[page, 1, place, 7] = odd
    got = ops.paged_attention(q, LayerCache(c.layer.k, v), draft, H, hd**-0.5)
    hit = torch.zeros(40, H, hd, dtype=torch.bool)
    hit[torch.arange(40) % 3 == 0, H // 2 :, 7] = True
    hit = hit.view(40, -1).to(DEV)
    assert torch.equal(got[~hit], clean[~hit])
    assert bool((got[hit].isnan() if math.isnan(odd) else got[hit] == odd).all())


NANS = {
    # sequence of (new, all) tokens, base, heads, bound on the length, (rows of a block, 1: shared out, 2: eight
    # waves), keys that are NaN
    "alone in a wave's tile": ((1, 33), 32, (4, 2), 0, (32, 0), lambda k: k == 32),
    "every tile of a wave": ((9, 250), 241, (4, 2), 0, (32, 0), lambda k: k // 32 % 4 == 2),
    "every tile of one wave in eight": ((9, 500), 480, (4, 2), 0, (32, 2), lambda k: k // 32 % 8 == 1),
    "one node": ((9, 500), 480, (4, 2), 0, (32, 2), lambda k: k == 485),
    "a whole share": ((16, 8192), 8100, (32, 8), 0, (32, 1), lambda k: k // 512 == 3),
    "half of the tiles of shared stages": ((160, 6000), 5840, (32, 8), 0, (64, 1), lambda k: k // 32 % 2 == 1),
}


@pytest.mark.parametrize("dtype,e4m3,odd", [(BF16, False, math.nan), (F16, False, math.nan), (F16, False, math.inf),
                                            (F32, False, math.nan), (BF16, True, math.nan)])
@pytest.mark.parametrize("name", sorted(NANS))
def test_a_score_of_nan_reaches_the_rows_that_see_it(name, dtype, e4m3, odd):
    """However the keys fall to waves and shares.  (A key of infinities gives it
    too: its products with a query of both signs do not add up.)"""
    (n, l), base, (H, KV), most, plan, which = NANS[name]
    hd = 64
    c, bits = _tree_case([(n, l)], [base], KV, hd, 64, dtype, e4m3, seed=13, most=most, fill=0.0)
    code = {F32: 0, BF16: 1, F16: 2}[dtype]
    p = _lib.query("lz_tree_attn_plan", code, 8 if e4m3 else code, c.rows, 1, H, KV, hd, c.step.max_new, c.step.max_len)
    assert dtype == F32 or (p & 255, p >> 8 & 255) == plan
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype).to(DEV)
    clean = ops.paged_attention(q, c.layer, c.draft, H, hd**-0.5)
    keys = torch.tensor([k for k in range(l) if which(k)])
    k = c.layer.k.clone()
    stored = k.view(torch.uint8) if e4m3 else k
    stored[c.table[0, keys // 64].long().to(DEV), KV - 1, (keys % 64).to(DEV)] = 0x7F if e4m3 else odd
    got = ops.paged_attention(q, c.layer._replace(k=k), c.draft, H, hd**-0.5).view(n, H, hd)
    hit = torch.zeros(n, H, dtype=torch.bool)
    hit[:, H - H // KV :] = _seen(c, [base], bits)[0][:, keys].any(1)[:, None]
    assert bool(hit.any())
    hit = hit.to(DEV)
    assert bool(got[hit].isnan().all())
    assert torch.equal(got[~hit], clean.view(n, H, hd)[~hit])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_scores_of_nan_in_a_chain_are_the_causal_calls(dtype):
    H, KV, hd, n, l = 8, 2, 64, 20, 500
    c = Case([(n, l)], KV, hd, 64, dtype, seed=3)
    bits = torch.ones(n, n).tril().bool()
    s = c.step
    draft = DraftStep(*s, _i32([l - n]), torch.zeros(n, dtype=torch.int32, device=DEV),
                      torch.zeros(n, dtype=torch.int64, device=DEV), _pack(bits).to(DEV))
    q = torch.randn(n, H * hd, generator=c.g).to(dtype).to(DEV)
    for keys in ([l - n + 7], [0], [k for k in range(l) if k // 32 % 8 == 3]):
        k = c.layer.k.clone()
        for key in keys:
            k[int(c.table[0, key // 64]), :, key % 64] = math.nan
        layer = LayerCache(k, c.layer.v)
        got, want = ops.paged_attention(q, layer, draft, H, hd**-0.5), ops.paged_attention(q, layer, s, H, hd**-0.5)
        assert torch.equal(got.isnan(), want.isnan())
        assert bool(got.view(n, -1).isnan().all(1)[max(0, keys[0] - (l - n)) :].all())


def test_rows_of_no_sequence_and_past_the_bounds_are_left():
    H, KV, hd = 4, 2, 32
    c, bits = _tree_case([(6, 20), (9, 40)], [14, 31], KV, hd, 16, BF16, seed=2)
    q = torch.randn(c.rows + 3, H * hd, generator=c.g).to(BF16).to(DEV)
    draft = c.draft
    whole = ops.paged_attention(q, c.layer, draft, H, 0.2)
    assert bool((whole[c.rows :] == 0).all())
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, c.layer, draft._replace(max_new=8), H, 0.2, out)  # 9 rows, 8 of them are computed
    assert torch.equal(out[: c.rows - 1], whole[: c.rows - 1]) and bool((out[c.rows - 1 :] == 7).all())
    # what the device tables say: starts past the rows, lengths past the table
    odd = draft._replace(row_start=_i32([0, 6, 2**31 - 1]), kv_len=_i32([20, 2**31 - 1]), base=_i32([14, -(2**31)]))
    got = ops.paged_attention(q, c.layer, odd, H, 0.2)
    assert torch.equal(got[:6], whole[:6])


def test_sequences_of_one_step_do_not_change_each_other():
    """Each sequence alone gives the bits that it gives among others of the same plan."""
    H, KV, hd = 8, 4, 64
    seqs, bases = [(9, 70), (12, 200), (4, 31), (12, 12)], [60, 188, 20, 0]
    c, bits = _tree_case(seqs, bases, KV, hd, 32, BF16, seed=8)
    q = torch.randn(c.rows, H * hd, generator=c.g).to(BF16).to(DEV)
    whole = ops.paged_attention(q, c.layer, c.draft, H, 0.1)
    for b, (n, l) in enumerate(seqs):
        rows = slice(c.starts[b], c.starts[b + 1])
        one = c.draft._replace(row_start=_i32([0, n]), kv_len=_i32([l]), page_table=c.draft.page_table[b : b + 1].contiguous(),
                               rows=n, base=_i32([bases[b]]), positions=c.draft.positions[rows],
                               mask=c.draft.mask[rows].contiguous())
        assert torch.equal(ops.paged_attention(q[rows].contiguous(), c.layer, one, H, 0.1), whole[rows])


def test_drafts_are_refused():
    H, KV, hd = 4, 2, 32
    c, _ = _tree_case([(6, 20), (9, 40)], [14, 31], KV, hd, 16, BF16, seed=2)
    q = torch.zeros(c.rows, H * hd, dtype=BF16, device=DEV)
    d = c.draft
    for bad in (d._replace(mask=d.mask[:-1]), d._replace(mask=d.mask.long()), d._replace(mask=d.mask[:, :0]),
                d._replace(base=d.base[:1]), d._replace(positions=d.positions[:-1]), d._replace(base=d.base.cpu()),
                d._replace(mask=d.mask.t().contiguous().t() if d.mask.shape[1] > 1 else d.mask[:, 0])):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_attention(q, c.layer, bad, H, 0.2)
    with pytest.raises(TypeError, match="CacheStep"):
        ops.paged_attention(q, c.layer, tuple(d[:9]), H, 0.2)


# ---------------------------------------------------------------------------
# writing drafted tokens, keeping a branch
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,e4m3", TYPES)
def test_rows_are_rotated_to_their_positions(dtype, e4m3):
    """A row at position p has the bits of a row that is cached in place p, and
    is cached in its own place."""
    H, KV, hd, page = 4, 2, 64, 16
    seqs = [(7, 40), (0, 3), (12, 12)]
    c = Case(seqs, KV, hd, page, dtype, e4m3, seed=4)
    qkv = torch.randn(c.rows, (H + 2 * KV) * hd, generator=c.g).to(dtype).to(DEV)
    angle = torch.rand(64, hd, generator=c.g) * 6
    cos, sin = angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV)
    at = torch.randint(0, 64, (c.rows,), generator=c.g).tolist()
    at[3], at[9] = -1, 64  # outside the tables: zeros, nothing cached
    before = [t.clone() for t in c.layer[:2]]
    slots = [int(c.table[b, p // page]) * page + p % page for b, (n, l) in enumerate(seqs) for p in range(l - n, l)]
    draft = DraftStep(*c.step[:5], 64, _i32([0] * 3), _i32(at), torch.tensor(slots, device=DEV))
    q = ops.kv_cache_write(qkv, c.layer, draft, H, cos, sin)
    written = set()
    for r, (p, slot) in enumerate(zip(at, slots)):
        where = (slot // page, slice(None), slot % page)
        if not 0 <= p < 64:
            assert bool((q[r] == 0).all())
            continue
        written.add(slot)
        # alone, in a sequence in which its place is p
        one = LayerCache(*(torch.zeros_like(t[:4]) if t is not None else None for t in c.layer))
        step = CacheStep(_i32([0, 1]), _i32([p + 1]), _i32([[0, 1, 2, 3]]), 1, 1, 64)
        want = ops.kv_cache_write(qkv[r : r + 1], one, step, H, cos, sin)
        assert torch.equal(q[r : r + 1], want)
        for mine, alone in zip(c.layer, one):
            if mine is not None:
                assert torch.equal(mine.view(torch.uint8 if e4m3 else mine.dtype)[where],
                                   alone.view(torch.uint8 if e4m3 else alone.dtype)[p // page, :, p % page])
    for mine, old in zip(c.layer[:2], before):
        bits = torch.uint8 if e4m3 else dtype
        flat = lambda t: t.view(bits).transpose(1, 2).reshape(-1, KV, hd)  # noqa: E731
        left = [s for s in range(mine.shape[0] * page) if s not in written]
        assert torch.equal(flat(mine)[left], flat(old)[left])


KEPT = {
    # new tokens of each sequence, kept nodes, counts
    "roots alone": ([1, 3], [[0, -1, -1], [0, -1, -1]], [1, 1]),
    "branches": ([12, 5, 9], [[0, 3, 7, 11], [0, 2, -1, -1], [0, 1, 2, 8]], [4, 2, 4]),
    "steps of one": ([12, 0, 12], [[0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [-1] * 11, [0, 1, 3, 5, 6, 7, 9, 10, 11, -1, -1]], [11, 0, 9]),
    "more than there are": ([4, 4], [[0, 2, 9, 3], [1, 3, -5, 2]], [99, 3]),
    "long": ([64], [[0] + list(range(13, 64))], [52]),
}


@pytest.mark.parametrize("layers", [0, 3])
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
@pytest.mark.parametrize("name", sorted(KEPT))
def test_kept_branches_move(name, dtype, layers):
    new, kept, counts = KEPT[name]
    KV, hd, page, n_pages = 3, 32, 16, 11
    g = torch.Generator().manual_seed(6)
    shape = ((layers,) if layers else ()) + (n_pages, KV, page, hd)
    bits = {BF16: torch.int16, F32: torch.int32, E4M3: torch.uint8}[dtype]
    lim = {torch.int16: 2**15 - 1, torch.int32: 2**31 - 1, torch.uint8: 255}[bits]
    k, v = (torch.randint(0, lim, shape, generator=g).to(bits) for _ in range(2))
    exps = [torch.randint(-9, 9, shape[:-1], generator=g).to(torch.int8) for _ in range(2)] if dtype == E4M3 else [None] * 2
    rows = sum(new)
    slots = torch.randperm(n_pages * page, generator=g)[:rows].tolist()
    if name == "branches":
        slots[3], slots[14] = -1, n_pages * page  # rows that are cached nowhere
    layer = LayerCache(*(t.to(DEV).view(dtype) for t in (k, v)), *(None if e is None else e.to(DEV) for e in exps))
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    step = DraftStep(_i32(starts), _i32(new), _i32([[0]] * len(new)), rows, max(new), 64, _i32([0] * len(new)),
                     _i32([0] * rows), torch.tensor(slots, device=DEV))
    ops.kv_cache_keep(layer, step, _i32(kept), _i32(counts))
    for got, want in zip(layer, [k, v, *exps]):
        if want is None:
            continue
        flat = want.view(-1, n_pages, KV, page, *want.shape[len(shape) - 1 :]).transpose(2, 3).reshape(max(layers, 1), n_pages * page, -1).clone()
        old = flat.clone()
        for b, n in enumerate(new):
            for j in range(min(counts[b], n, len(kept[b]))):
                if 0 <= kept[b][j] < n:
                    src, dst = slots[starts[b] + kept[b][j]], slots[starts[b] + j]
                    if 0 <= src < n_pages * page and 0 <= dst < n_pages * page:
                        flat[:, dst] = old[:, src]
        back = flat.view(max(layers, 1), n_pages, page, KV, *want.shape[len(shape) - 1 :]).transpose(2, 3).reshape(want.shape)
        assert torch.equal(got.view(want.dtype).cpu(), back)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_kept_branches_move_whichever_of_them_are_left_out(dtype):
    """Up to three rounds of eight nodes, of which any may have no slot, or one
    past the pages, or be no node: the moves of the others do not change."""
    KV, hd, page, n_pages, B = 2, 32, 16, 12, 4
    bits = torch.uint8 if dtype == E4M3 else torch.int16
    for seed in range(40):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        new = [rng.randint(0, 24) for _ in range(B)]
        rows, starts = sum(new), [sum(new[:b]) for b in range(B + 1)]
        order = torch.randperm(n_pages * page, generator=g)[:rows].tolist()
        odd = rng.choice([0.0, 0.1, 0.5])
        slots = [rng.choice([-1, n_pages * page, 2**40]) if rng.random() < odd else s for s in order]
        kept = [sorted(rng.sample(range(n), rng.randint(min(n, 1), n))) for n in new]
        counts = [len(k) for k in kept]
        kept = [[rng.choice([-1, 99, 2**31 - 1]) if rng.random() < odd else x for x in k] + [-1] * (24 - len(k)) for k in kept]
        cpu = [torch.randint(0, 127, (n_pages, KV, page, hd), generator=g).to(bits) for _ in range(2)]
        exps = [torch.randint(-9, 9, (n_pages, KV, page), generator=g).to(torch.int8) for _ in range(2)] if dtype == E4M3 else []
        layer = LayerCache(*(t.to(DEV).view(dtype) for t in cpu), *([e.to(DEV) for e in exps] or [None, None]))
        step = DraftStep(_i32(starts), _i32(new), _i32([[0]] * B), rows, 24, 64, _i32([0] * B), _i32([0] * rows),
                         torch.tensor(slots, dtype=torch.int64, device=DEV))
        ops.kv_cache_keep(layer, step, _i32(kept), _i32(counts))
        inside = lambda x: 0 <= x < n_pages * page  # noqa: E731
        for got, want in zip([x for x in layer if x is not None], [*cpu, *exps]):
            flat = want.transpose(1, 2).reshape(n_pages * page, -1).clone()
            old = flat.clone()
            for b, n in enumerate(new):
                for j in range(counts[b]):
                    if 0 <= kept[b][j] < n and inside(src := slots[starts[b] + kept[b][j]]) and inside(dst := slots[starts[b] + j]):
                        flat[dst] = old[src]
            back = flat.view(n_pages, page, KV, *want.shape[3:]).transpose(1, 2)
            assert torch.equal(got.view(want.dtype).cpu(), back), seed


def test_keep_is_refused():
    layer = LayerCache(*(torch.zeros(4, 2, 16, 32, dtype=BF16, device=DEV) for _ in range(2)))
    step = DraftStep(_i32([0, 3]), _i32([3]), _i32([[0]]), 3, 3, 16, _i32([0]), _i32([0] * 3),
                     torch.zeros(3, dtype=torch.int64, device=DEV))
    kept, counts = _i32([[0, 1]]), _i32([1])
    ops.kv_cache_keep(layer, step, kept, counts)
    for args in ((LayerCache(layer.k, layer.v.float()), step, kept, counts), (layer, step._replace(slots=step.slots[:2]), kept, counts),
                 (layer, step._replace(slots=step.slots.int()), kept, counts), (layer, step, kept[0], counts),
                 (layer, step, kept, _i32([1, 1])), (layer, step, kept.long(), counts), (layer, step, kept.cpu(), counts),
                 (LayerCache(layer.k.to(E4M3), layer.v.to(E4M3)), step, kept, counts),
                 (LayerCache(layer.k.transpose(0, 1), layer.v.transpose(0, 1)), step, kept, counts)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.kv_cache_keep(*args)
    with pytest.raises(TypeError, match="DraftStep"):
        ops.kv_cache_keep(layer, CacheStep(*step[:6]), kept, counts)


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------

class Pool:
    """PageTables as Python lists, and what a call makes of them."""

    def __init__(self, lengths, width, page, spare, seed=0, slack=0):
        self.page, self.width = page, width
        rng = random.Random(seed)
        need = [min(-(-max(l, 0) // page), width) for l in lengths]
        ids = list(range(sum(need) + spare))
        rng.shuffle(ids)
        self.table = [[ids.pop() for _ in range(n)] + [-1] * (width - n) for n in need]
        self.lengths = list(lengths)
        self.free = ids + [-1] * (sum(need) + slack)
        self.n_free = len(ids)

    def device(self):
        return PageTables(_i32(self.table), _i32(self.lengths), _i32(self.free), _i32([self.n_free]), self.page)

    def step(self, new, rows, max_new, max_len, keep=None, base=None, parents=None):
        P, cap = self.page, self.width * self.page
        now = [min(max(l, 0), cap) for l in self.lengths]
        keep = now if keep is None else [min(max(k, 0), l) for k, l in zip(keep, now)]
        back = []
        for b, (k, l) in enumerate(zip(keep, now)):
            for i in range(-(-k // P), -(-l // P)):
                back.append(self.table[b][i])
                self.table[b][i] = -1
        self.free[self.n_free : self.n_free + len(back)] = back[::-1]
        top, asked, pages = self.n_free + len(back), 0, 0
        have = top
        starts, lens, bases, positions, slots, masks = [0], [], [], [], [], []
        trees = None if parents is None else parents if isinstance(parents[0], list) else [parents] * len(new)
        words = -(-len(trees[0]) // 32) if trees else 0
        for b, (k, n) in enumerate(zip(keep, new)):
            need = 0
            if 0 < n <= min(max_new, rows) and k + n <= min(max_len, cap):
                need = -(-(k + n) // P) - -(-k // P)
                asked, pages = asked + n, pages + need
                if (need and pages > have) or asked > rows:
                    n = need = 0
            else:
                n = 0
            for i in range(need):
                top -= 1
                self.table[b][-(-k // P) + i] = self.free[top]
            at = k if base is None else base[b]
            if trees:
                sets, depth = _closure(trees[b])
            for place in range(k, k + n):
                page = self.table[b][place // P]
                slots.append(page * P + place % P if page >= 0 else -1)
                node = place - at
                known = trees and 0 <= node < len(trees[b])
                positions.append(at + depth[node] if known else place)
                masks.append([sum(1 << j % 32 for j in sets[node] if j // 32 == w) if known else 0 for w in range(words)])
            starts.append(starts[-1] + n)
            lens.append(k + n)
            bases.append(at)
        self.lengths, self.n_free = lens, top
        none = rows - starts[-1]
        mask = torch.tensor(masks + [[0] * words] * none, dtype=torch.int64).view(rows, words).to(torch.int32) if trees else None
        return starts, lens, bases, positions + [-1] * none, slots + [-1] * none, mask

    def check(self, tables, step, want):
        starts, lens, bases, positions, slots, mask = want
        for name, got, to in (("row_start", step.row_start, starts), ("kv_len", step.kv_len, lens), ("base", step.base, bases),
                              ("positions", step.positions, positions), ("slots", step.slots, slots),
                              ("table", tables.page_table, self.table), ("lengths", tables.lengths, self.lengths),
                              ("free", tables.free, self.free), ("n_free", tables.n_free, [self.n_free])):
            assert got.tolist() == to, name
        assert (step.mask is None) == (mask is None)
        if mask is not None:
            assert torch.equal(step.mask.cpu(), mask)


def _trees(rng, n, nodes):
    return [[rng.randint(-1, i - 1) if i else -1 for i in range(nodes)] for _ in range(n)]


@pytest.mark.parametrize("B", [1, 3, 64, 65, 1023, 1025, 4096])
def test_tables_over_many_steps(B):
    """Sequences grow, are cut back, wait for pages and end, step after step."""
    rng = random.Random(B)
    page, width = 16, 9
    pool = Pool([rng.choice([0, 1, 15, 16, 17, rng.randint(0, 100)]) for _ in range(B)], width, page, spare=B + 3, slack=2, seed=B)
    tables = pool.device()
    for turn in range(4):
        nodes = rng.choice([1, 7, 33, 70])
        new = [rng.choice([0, 1, rng.randint(0, nodes), nodes, nodes + 1, -3]) for _ in range(B)]
        keep = None if turn == 0 else [rng.choice([l, l, max(0, l - rng.randint(0, 40)), l + 5, 0, -2]) for l in pool.lengths]
        rows = rng.choice([sum(max(n, 0) for n in new), sum(max(n, 0) for n in new) // 2, 5])
        parents = rng.choice([None, _trees(rng, 1, nodes)[0], _trees(rng, B, nodes)])
        max_len = rng.choice([page * width, 90])
        args = [rows, nodes, max_len]
        step = ops.cache_tables(tables, _i32(new), *args, keep=None if keep is None else _i32(keep),
                                parents=None if parents is None else _i32(parents))
        pool.check(tables, step, pool.step(new, *args, keep=keep, parents=parents))
        assert (step.rows, step.max_new, step.max_len) == tuple(args) and step.page_table is tables.page_table


def test_an_ask_of_more_than_all_rows_holds_up_nobody():
    """It could not be served in any order, so it counts for nothing; one that
    does not fit beside those before it counts, and those behind it wait."""
    for new, want in (([70, 3], [0, 0, 3]), ([6, 5], [0, 0, 5]), ([3, 3, 2], [0, 3, 3, 3])):
        pool = Pool([4] * len(new), 8, 16, spare=16)
        tables = pool.device()
        step = ops.cache_tables(tables, _i32(new), 5, 70, 128)
        assert step.row_start.tolist() == want
        pool.check(tables, step, pool.step(new, 5, 70, 128))


def test_tables_of_prompts():
    """More rows than one workgroup describes, sequences that do not all fit."""
    rng = random.Random(1)
    new = [rng.randint(1, 700) for _ in range(40)]
    pool = Pool([0] * 40, 64, 16, spare=sum(-(-n // 16) for n in new) - 30, slack=5)
    tables = pool.device()
    step = ops.cache_tables(tables, _i32(new), sum(new), 700, 1024)
    want = pool.step(new, sum(new), 700, 1024)
    assert 0 < want[0][-1] < sum(new)
    pool.check(tables, step, want)


def test_tables_of_a_tree_that_grows():
    """A tree that is cached level by level: base stays, nodes are counted from it."""
    parents = [-1, 0, 0, 1, 1, 2, 3, 5, 5, 7]
    pool = Pool([30, 17], 8, 16, spare=6)
    tables = pool.device()
    base = [30, 17]
    for n in (1, 2, 3, 4):
        step = ops.cache_tables(tables, _i32([n, n]), 2 * n, n, 128, base=_i32(base), parents=_i32(parents))
        pool.check(tables, step, pool.step([n, n], 2 * n, n, 128, base=base, parents=parents))
    # rows outside the tree see the text alone
    step = ops.cache_tables(tables, _i32([2, 2]), 4, 2, 128, base=_i32([50, 17]), parents=_i32(parents))
    pool.check(tables, step, pool.step([2, 2], 4, 2, 128, base=[50, 17], parents=parents))


def test_a_rejected_drafts_pages_are_taken_again():
    pool = Pool([20, 33, 64, 5], 12, 16, spare=20)
    tables = pool.device()
    keep = _i32(pool.lengths)
    first = ops.cache_tables(tables, _i32([40, 30, 50, 20]), 140, 50, 192)
    table, free = tables.page_table.clone(), int(tables.n_free)
    again = ops.cache_tables(tables, _i32([40, 30, 50, 20]), 140, 50, 192, keep=keep)
    assert torch.equal(tables.page_table, table) and int(tables.n_free) == free
    assert torch.equal(first.slots, again.slots)


def test_tables_that_say_nonsense_stay_inside():
    """Lengths, counts and stacks of any value: what is not theirs is left."""
    far = [2**31 - 1, -(2**31), 7, 130, -1]
    guard = torch.full((3, 5, 4), -7, dtype=torch.int32, device=DEV)
    table = guard[1]
    table[:] = torch.arange(20, dtype=torch.int32, device=DEV).view(5, 4)
    stack = torch.full((3, 8), -7, dtype=torch.int32, device=DEV)
    for n_free in (2**31 - 1, -(2**31), 3):
        for new in ([2**31 - 1] * 5, [-(2**31)] * 5, [3] * 5):
            for keep in (None, far[::-1]):
                tables = PageTables(table, _i32(far), stack[1], _i32([n_free]), 16)
                step = ops.cache_tables(tables, _i32(new), 11, 9, 2**31 - 1, keep=None if keep is None else _i32(keep),
                                        base=_i32(far), parents=_i32([-1, 5, 0]))
                starts = step.row_start.tolist()
                assert starts[0] == 0 and all(a <= b <= 11 for a, b in zip(starts, starts[1:]))
                assert 0 <= int(tables.n_free) <= 8 and all(0 <= l <= 64 for l in tables.lengths.tolist())
    assert bool((guard[[0, 2]] == -7).all()) and bool((stack[[0, 2]] == -7).all())


def test_tables_in_a_graph():
    """A captured step, its lengths and counts changing from replay to replay."""
    B, nodes = 6, 20
    pool = Pool([10, 0, 33, 47, 16, 90], 12, 16, spare=30, slack=3)
    tables = pool.device()
    new, keep, parents = _i32([1] * B), tables.lengths.clone(), _i32([[-1] + [0] * (nodes - 1)] * B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step = ops.cache_tables(tables, new, 70, nodes, 192, keep=keep, parents=parents)
    rng = random.Random(9)
    for _ in range(5):
        n = [rng.randint(0, nodes) for _ in range(B)]
        k = [max(0, l - rng.randint(0, 30)) for l in pool.lengths]
        trees = _trees(rng, B, nodes)
        new.copy_(_i32(n))
        keep.copy_(_i32(k))
        parents.copy_(_i32(trees))
        graph.replay()
        torch.cuda.synchronize()
        pool.check(tables, step, pool.step(n, 70, nodes, 192, keep=k, parents=trees))


def test_tables_are_refused():
    t = Pool([10, 0], 4, 16, spare=4).device()
    new = _i32([1, 1])
    call = lambda t, new=new, rows=2, max_new=1, max_len=64, **k: ops.cache_tables(t, new, rows, max_new, max_len, **k)  # noqa: E731
    call(t)
    for bad in (lambda: call(t._replace(page_size=24)), lambda: call(t, new.long()), lambda: call(t, _i32([1])),
                lambda: call(t, rows=-1), lambda: call(t, max_new=-1), lambda: call(t, keep=_i32([1])),
                lambda: call(t, parents=_i32([[-1]])), lambda: call(t, max_new=3, parents=_i32([-1, 0])),
                lambda: call(t, parents=_i32([])), lambda: call(t, parents=torch.full((4097,), -1, dtype=torch.int32, device=DEV)), lambda: call(t, new.cpu()), lambda: call(t._replace(n_free=_i32([1, 2]))),
                lambda: call(t._replace(page_table=t.page_table.t())), lambda: call(t._replace(free=t.free[:0]))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    with pytest.raises(TypeError, match="PageTables"):
        call(tuple(t[:4]))


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------

def _pick(weights, u):
    sums = weights.cumsum(0)
    if not float(sums[-1]) > 0:
        return -1
    over = (sums > max(u, 0.0) * sums[-1]).nonzero()
    return int(over[0]) if len(over) else int((weights > 0).nonzero()[-1])


def _verify(logits, tokens, starts, max_new, uniform, heat, parents=None, probs=None):
    """One sequence after another, in float64."""
    x, u, V = logits.double().cpu(), uniform.double().tolist(), logits.shape[1]
    counts, kept, chosen = [], [], []
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        n, t = min(hi - lo, max_new), heat[b]

        def weights(row):
            row = x[row]
            if bool(row.isnan().any()) or float(row.max()) == -math.inf or (t > 0 and float(row.max()) == math.inf):
                return None
            if not t > 0:
                return torch.nn.functional.one_hot(row.argmax(), V).double()
            return torch.exp((row - row.max()) / t)

        nodes, said = ([0], []) if n else ([], [])
        while nodes:
            at = nodes[-1]
            w = weights(lo + at)
            if probs is not None:
                nxt = at + 1
                if nxt < n:
                    tok, q = tokens[lo + nxt], probs[lo + nxt].double().cpu()
                    if w is not None and 0 <= tok < V and u[lo + nxt] * float(q[tok]) < float(w[tok] / w.sum()):
                        nodes.append(nxt)
                        said.append(tok)
                        continue
                    if w is not None:
                        rest = (w / w.sum() - q).clamp(min=0)
                        w = rest if float(rest.sum()) > 0 else w
                said.append(-1 if w is None else _pick(w, u[lo]))
                break
            tok = -1 if w is None else _pick(w, u[lo + at])
            said.append(tok)
            tree = parents[b] if parents and isinstance(parents[0], list) else parents
            child = [i for i in range(at + 1, n) if (tree[i] if tree else i - 1) == at and tokens[lo + i] == tok and tok >= 0]
            if not child:
                break
            nodes.append(child[0])
        counts.append(len(nodes))
        kept.append(nodes + [-1] * (max_new - len(nodes)))
        chosen.append(said + [-1] * (max_new - len(said)))
    return counts, kept, chosen


def _check_verify(logits, tokens, new, uniform, heat=1.0, parents=None, probs=None, max_new=None, pad=0):
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    max_new = max(new) if max_new is None else max_new
    each = heat if isinstance(heat, list) else [heat] * len(new)
    got = ops.verify_draft(logits.to(DEV) if not logits.is_cuda else logits, torch.tensor(tokens, device=DEV), _i32(starts), max_new,
                           uniform.to(DEV), temperature=torch.tensor(heat, device=DEV) if isinstance(heat, list) else heat,
                           parents=None if parents is None else _i32(parents), draft_probs=None if probs is None else probs.to(DEV))
    want = _verify(logits, tokens, starts, max_new, uniform, each, parents, probs)
    for name, g, w in zip(("counts", "kept", "chosen"), got, want):
        assert g.tolist() == w, name
    return want


def _drafted(seed, new, V, dtype=F32, scale=4.0, trees=False, likely=3):
    """Logits, and tokens among the likely ones of their parents' rows."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    rows = sum(new)
    logits = (scale * torch.randn(rows, V, generator=g)).to(dtype)
    parents = _trees(rng, len(new), max(new)) if trees else None
    tokens, lo = [], 0
    top = logits.float().topk(min(likely, V)).indices.tolist()
    for b, n in enumerate(new):
        for i in range(n):
            up = (parents[b][i] if trees else i - 1) if i else 0
            tokens.append(rng.choice(top[lo + max(up, 0)]))
        lo += n
    return logits, tokens, parents, torch.rand(rows, generator=g, dtype=torch.float64)


SIZES = [([1], 1), ([1, 4], 2), ([5], 7), ([3, 0, 6, 1], 513), ([8] * 5, 2048), ([2, 9], 2049), ([17, 4, 30], 5003), ([70, 3], 300)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("new,V", SIZES)
@pytest.mark.parametrize("trees", [False, True])
def test_own_choices(dtype, new, V, trees):
    for seed in range(3):
        logits, tokens, parents, u = _drafted(seed, new, V, dtype, trees=trees)
        for heat in (0.0, 0.7, [0.0 if b % 2 else 0.5 + b for b in range(len(new))]):
            _check_verify(logits, tokens, new, u if seed else u.float(), heat, parents)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("new,V", SIZES)
def test_drawn_tokens(dtype, new, V):
    for seed in range(3):
        logits, _, _, u = _drafted(seed, new, V, dtype)
        g = torch.Generator().manual_seed(seed)
        for heat in (0.0, 1.3, [0.0 if b % 2 else 0.5 + b for b in range(len(new))]):
            noisy = logits.float() + torch.randn(logits.shape, generator=g)
            probs = torch.softmax(noisy, -1).roll(1, 0).contiguous()  # a row's token follows the row before it
            tokens = torch.multinomial(probs, 1, generator=g)[:, 0].tolist()
            _check_verify(logits, tokens, new, u, heat, None, probs)


def test_large_vocabularies():
    """More pieces than lanes, uneven ends."""
    for V, new in ((128256, [8] * 5), (40001, [3] * 40), (151937, [30])):
        logits, tokens, parents, u = _drafted(V, new, V, BF16, scale=5.0, trees=True)
        _check_verify(logits, tokens, new, u, 1.0, parents)
    logits, _, _, u = _drafted(1, [4] * 12, 131071, F32, scale=5.0)
    probs = torch.softmax(logits + 0.5, -1).roll(1, 0).contiguous()
    tokens = torch.multinomial(probs, 1).squeeze(1).tolist()
    counts = _check_verify(logits, tokens, [4] * 12, u, 1.0, None, probs)[0]
    assert sum(counts) == 48  # q = p: everything is kept


@pytest.mark.parametrize("V,new,dtype", [(128256, [14] * 5, BF16), (33001, [20] * 14, F32), (33001, [60, 9, 200], F16)])
@pytest.mark.parametrize("drawn", [False, True])
def test_many_rows_of_large_vocabularies(V, new, dtype, drawn):
    """Enough rows for pieces of 2048."""
    logits, tokens, parents, u = _drafted(V, new, V, dtype, scale=5.0, trees=not drawn)
    probs = None
    if drawn:
        g = torch.Generator().manual_seed(V)
        noisy = logits.float() + torch.randn(logits.shape, generator=g)
        probs = torch.softmax(noisy, -1).roll(1, 0).contiguous()
        tokens = torch.multinomial(probs, 1, generator=g)[:, 0].tolist()
    for heat in (1.0, [0.0 if b % 2 else 0.7 for b in range(len(new))]):
        _check_verify(logits, tokens, new, u, heat, parents, probs)


def test_strided_rows():
    logits, tokens, parents, u = _drafted(3, [6, 9], 1001, BF16, trees=True)
    wide = torch.randn(15, 3, 1011, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    wide[:, 1, 5:1006] = logits.to(DEV)
    view = wide[:, 1, 5:1006]
    for heat in (0.0, 1.0):
        _check_verify(view, tokens, [6, 9], u, heat, parents)
    probs = torch.softmax(logits.float(), -1).roll(1, 0)
    wide = torch.zeros(15, 1003, device=DEV)
    wide[:, 1:1002] = probs.to(DEV)
    _check_verify(view, tokens, [6, 9], u, 1.0, None, wide[:, 1:1002])


def test_borders_and_ties():
    """Equal weights: token floor(4 u), whatever lies behind the border; the
    first of equal logits; numbers outside [0, 1)."""
    x = torch.full((9, 10), -math.inf)
    x[:, [1, 4, 5, 8]] = 2.5
    at = [1, 4, 5, 8]
    u = torch.tensor([0.0, 0.25, math.nextafter(0.25, 0), 0.5, 0.75, math.nextafter(1.0, 0.0), 1.0, -3.0, math.nan],
                     dtype=torch.float64)
    want = [at[0], at[1], at[0], at[2], at[3], at[3], at[3], at[0], at[0]]
    got = ops.verify_draft(x.to(DEV), torch.zeros(9, dtype=torch.int64, device=DEV), _i32(list(range(10))), 1, u.to(DEV))
    assert got[2][:, 0].tolist() == want and got[0].tolist() == [1] * 9
    got = ops.verify_draft(x.to(DEV), torch.zeros(9, dtype=torch.int64, device=DEV), _i32(list(range(10))), 1, u.to(DEV), temperature=0)
    assert got[2][:, 0].tolist() == [1] * 9


def test_numbers_outside_of_the_range_keep_as_those_at_its_ends():
    """Below 0 and NaN as 0: what p does not hold is not kept, the rest is.  From
    1 on as just under it: where p is q, everything is kept."""
    V = 8
    x = torch.full((2, V), -math.inf)
    x[:, :4] = 1.0  # p = 1/4 each
    q = torch.zeros(2, V)
    q[:, :4] = 0.25
    q[:, 4:] = 0.5
    just = math.nextafter(1.0, 0.0)
    for u, token, counts in ((-3.0, 5, 1), (-3.0, 2, 2), (-math.inf, 5, 1), (math.nan, 5, 1), (math.nan, 2, 2), (0.0, 2, 2), (0.0, 5, 1),
                             (just, 3, 2), (1.0, 3, 2), (7.0, 3, 2), (math.inf, 3, 2), (1.0, 5, 1)):
        for kind in (torch.float64, torch.float32):
            got = ops.verify_draft(x.to(DEV), torch.tensor([0, token], device=DEV), _i32([0, 2]), 2,
                                   torch.tensor([0.5, u], dtype=kind, device=DEV), draft_probs=q.to(DEV))
            assert got[0].tolist() == [counts], (u, token, kind)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V", [700, 40000])
def test_tokens_at_the_types_lowest_value_are_not_chosen(dtype, V):
    """A mask of finite values: their probability is zero, for numbers at either
    end of the range too, in sampling and in what is kept of a draft."""
    n = 200 if V == 700 else 40
    x = (3 * torch.randn(n, V, generator=torch.Generator().manual_seed(V))).to(dtype)
    x[:, V - 200 :] = torch.finfo(dtype).min
    x[:, :5] = torch.finfo(dtype).min
    x = x.to(DEV)
    tokens = torch.zeros(n, dtype=torch.int64, device=DEV)
    for u in (0.0, math.nextafter(1.0, 0.0), 1.0):
        uniform = torch.full((n,), u, dtype=torch.float64, device=DEV)
        chosen = ops.verify_draft(x, tokens, _i32(list(range(n + 1))), 1, uniform)[2]
        assert bool(((chosen >= 5) & (chosen < V - 200)).all()), u
        # chains of one drafted token that the mask forbids, with a number of 0, and what follows
        probs = torch.full((n, V), 1.0 / V, device=DEV)
        uniform[1::2] = 0.0
        counts, _, chosen = ops.verify_draft(x, tokens, _i32(list(range(0, n + 1, 2))), 2, uniform, draft_probs=probs)
        assert bool((counts == 1).all())
        assert bool(((chosen[:, 0] >= 5) & (chosen[:, 0] < V - 200)).all())


def test_an_infinite_temperature_takes_from_all():
    x = 3 * torch.randn(40, 4, generator=torch.Generator().manual_seed(6))
    x[:, 2] = -math.inf
    u = (torch.arange(40, dtype=torch.float64) + 0.5) / 40
    got = ops.verify_draft(x.to(DEV), torch.zeros(40, dtype=torch.int64, device=DEV), _i32(list(range(41))), 1, u.to(DEV),
                           temperature=torch.full((40,), math.inf, device=DEV))[2][:, 0].tolist()
    assert got == [(0, 1, 3)[int(3 * v)] for v in u.tolist()]
    with pytest.raises(ValueError, match="finite"):
        ops.verify_draft(x.to(DEV), torch.zeros(40, dtype=torch.int64, device=DEV), _i32(list(range(41))), 1, u.to(DEV),
                         temperature=math.inf)


def test_each_token_has_its_share():
    """K equally spaced numbers: token v is chosen by K p_v of them, to within one."""
    K, V = 4000, 37
    x = 1.5 * torch.randn(V, generator=torch.Generator().manual_seed(2))
    u = (torch.arange(K, dtype=torch.float64) + 0.5) / K
    got = ops.verify_draft(x.expand(K, V).contiguous().to(DEV), torch.zeros(K, dtype=torch.int64, device=DEV),
                           _i32(list(range(K + 1))), 1, u.to(DEV), temperature=0.8)[2][:, 0].cpu()
    p = torch.softmax(x.double() / 0.8, 0)
    assert bool(((got.bincount(minlength=V) - K * p).abs() <= 1).all())


def test_rows_that_leave_nothing_to_choose():
    new, V = [2, 2, 2, 2, 2, 3], 600
    logits, tokens, _, u = _drafted(4, new, V)
    logits[0] = -math.inf               # a grammar that allows nothing
    logits[2, 599] = math.nan
    logits[4, 3] = math.inf
    logits[6, :] = -math.inf
    logits[6, 77] = 1e30
    tokens[7] = 77
    logits[9, 5] = math.nan             # the row after the kept token
    tokens[9] = int(logits[8].argmax())
    for heat in (0.0, 1.0):
        counts, _, chosen = _check_verify(logits, tokens, new, u, heat)
        assert chosen[0][0] == -1 and chosen[1][0] == -1 and chosen[2][0] == (3 if heat == 0 else -1) and counts[3] == 2
    probs = torch.softmax(torch.nan_to_num(logits, nan=0, posinf=0, neginf=-9), -1).roll(1, 0).contiguous()
    for heat in (0.0, 1.0):
        _check_verify(logits, tokens, new, u, heat, None, probs)


def test_tokens_and_parents_that_are_none():
    V = 300
    logits, tokens, _, u = _drafted(5, [6, 6, 6], V)
    best = logits.argmax(-1).tolist()
    tokens[1], tokens[2], tokens[3] = -1, V, 2**40            # ids outside the vocabulary are never chosen
    tokens[4] = best[0]
    tokens[7] = tokens[8] = tokens[9] = best[6]               # of the same tokens the first child counts
    tokens[10] = best[8]
    parents = [[-1, 0, 0, 0, 0, 4], [5, 3, 0, 0, 2, 2**31 - 1], [-1, -1, -1, 1, 7, -(2**31)]]
    kept = _check_verify(logits, tokens, [6, 6, 6], u, 0.0, parents)[1]
    assert kept[0][:2] == [0, 4] and kept[1][:3] == [0, 2, 4]
    # a chain of more rows than max_new: those behind it are not read
    _check_verify(logits, best[-1:] + best[:-1], [9, 9], u, 0.0, max_new=4)
    # draft probabilities of zero, and a draft that is the model's own law
    probs = torch.softmax(logits, -1).roll(1, 0).contiguous()
    p = probs.clone()
    p[3] = 0
    _check_verify(logits, [t % V for t in tokens], [6, 6, 6], u, 1.0, None, p)
    _check_verify(logits, [2**40] * 18, [6, 6, 6], u, 1.0, None, probs)


def test_the_chosen_tokens_law_is_the_models():
    """Chains of one drafted token: over all numbers for the draft, for keeping
    and for what follows, the gained token's law is p."""
    K, V = 30, 7
    g = torch.Generator().manual_seed(3)
    x, y = torch.randn(2, V, generator=g)
    p, q = torch.softmax(x.double(), 0), torch.softmax(y, 0)
    u = (torch.arange(K, dtype=torch.float64) + 0.5) / K
    keep, after = torch.meshgrid(u, u, indexing="ij")
    n = K * K
    uniform = torch.stack([after.reshape(-1), keep.reshape(-1)], 1).reshape(-1)
    law = torch.zeros(V, dtype=torch.float64)
    for token in range(V):
        chosen = ops.verify_draft(x.expand(2 * n, V).contiguous().to(DEV), torch.full((2 * n,), token, device=DEV),
                                  _i32(list(range(0, 2 * n + 1, 2))), 2, uniform.to(DEV), draft_probs=q.expand(2 * n, V).contiguous().to(DEV))[2]
        law += float(q[token]) * chosen[:, 0].cpu().bincount(minlength=V).double() / n
    # each border of the grid is off by half a step of 1 / K at most, in keeping and in choosing
    assert bool(((law - p).abs() <= 1.0 / K).all())


def test_verify_in_a_graph():
    new, V = [5, 5, 5], 900
    drafts = [_drafted(s, new, V, BF16, trees=True) for s in range(4)]
    logits, tokens, parents, u = (drafts[0][0].to(DEV), torch.tensor(drafts[0][1], device=DEV), _i32(drafts[0][2]),
                                  drafts[0][3].to(DEV))
    probs, starts, heat = torch.zeros(15, V, device=DEV), _i32([0, 5, 10, 15]), torch.ones(3, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tree = ops.verify_draft(logits, tokens, starts, 5, u, temperature=heat, parents=parents)
        chain = ops.verify_draft(logits, tokens, starts, 5, u, temperature=heat, draft_probs=probs)
    for s in (1, 2, 3, 1):
        x, t, p, r = drafts[s]
        q = torch.softmax(x.float(), -1).roll(1, 0).contiguous()
        for to, value in ((logits, x), (tokens, torch.tensor(t)), (parents, _i32(p)), (u, r), (probs, q)):
            to.copy_(value)
        heat.fill_(0.5 * s)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in ((tree, _verify(x, t, [0, 5, 10, 15], 5, r, [0.5 * s] * 3, p)),
                          (chain, _verify(x, t, [0, 5, 10, 15], 5, r, [0.5 * s] * 3, None, q))):
            assert [g.tolist() for g in got] == list(want)


def test_verify_is_refused():
    x, t, starts, u = torch.zeros(4, 9, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV), _i32([0, 2, 4]), torch.zeros(4, device=DEV)
    call = lambda x=x, t=t, starts=starts, n=2, u=u, **k: ops.verify_draft(x, t, starts, n, u, **k)  # noqa: E731
    call()
    for bad in (lambda: call(x=x[0]), lambda: call(x=x.t()), lambda: call(t=t.int()), lambda: call(t=t[:3]), lambda: call(n=0),
                lambda: call(n=5000), lambda: call(u=u.half()), lambda: call(u=u[:3]), lambda: call(starts=starts.long()),
                lambda: call(starts=starts[:1]), lambda: call(temperature=math.nan), lambda: call(temperature=torch.ones(3, device=DEV)),
                lambda: call(parents=_i32([0])), lambda: call(parents=_i32([[-1, 0]])), lambda: call(draft_probs=x[:3]),
                lambda: call(draft_probs=x.half()), lambda: call(parents=_i32([-1, 0]), draft_probs=x), lambda: call(t=t.cpu())):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            bad()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("e4m3", [False, True])
def test_steps_together(e4m3):
    """Several steps of a layer, without the host: what is kept in the cache is
    what writing the kept tokens alone gives, and a row's attention that of its
    branch written as a text."""
    dtype, H, KV, hd, page, V, B, nodes = BF16, 4, 2, 64, 16, 50, 3, 9
    g = torch.Generator().manual_seed(1)
    rng = random.Random(1)
    angle = torch.rand(256, hd, generator=g) * 6
    cos, sin = angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV)

    def layer(n):
        store = torch.float8_e4m3fn if e4m3 else dtype
        exps = [torch.zeros(n, KV, page, dtype=torch.int8, device=DEV) for _ in range(2)] if e4m3 else [None] * 2
        return LayerCache(*(torch.zeros(n, KV, page, hd, device=DEV).to(store) for _ in range(2)), *exps)

    cache = layer(40)
    order = torch.randperm(40, generator=g).to(torch.int32)
    tables = PageTables(torch.full((B, 12), -1, dtype=torch.int32, device=DEV), _i32([0] * B), order.to(DEV), _i32([40]), page)
    embed = torch.randn(V, (H + 2 * KV) * hd, generator=g).to(dtype).to(DEV)
    prompts = [[rng.randrange(V) for _ in range(n)] for n in (5, 30, 17)]
    texts = [list(p) for p in prompts]
    step = ops.cache_tables(tables, _i32([len(p) for p in prompts]), 52, 30, 192)
    ops.kv_cache_write(embed[torch.tensor(sum(prompts, []), device=DEV)], cache, step, H, cos, sin)
    keep = tables.lengths.clone()
    roots = [rng.randrange(V) for _ in range(B)]
    for turn in range(4):
        parents = _trees(rng, B, nodes)
        for tree in parents:
            for i in range(1, nodes):
                tree[i] = max(tree[i], 0)
        ids = [[roots[b]] + [rng.randrange(3) for _ in range(nodes - 1)] for b in range(B)]
        flat = torch.tensor(sum(ids, []), device=DEV)
        step = ops.cache_tables(tables, _i32([nodes] * B), B * nodes, nodes, 192, keep=keep, parents=_i32(parents))
        qkv = embed[flat]
        q = ops.kv_cache_write(qkv, cache, step, H, cos, sin)
        y = ops.paged_attention(q, cache, step, H, hd**-0.5)
        logits = torch.randn(B * nodes, V, generator=g)
        logits[:, :3] += 5  # few likely tokens: branches are kept
        u = torch.rand(B * nodes, generator=g, dtype=torch.float64)
        counts, kept, chosen = ops.verify_draft(logits.to(DEV), flat, step.row_start, nodes, u.to(DEV), parents=_i32(parents))
        # every row alone, its branch behind the text
        for b in range(B):
            sets, _ = _closure(parents[b])
            for i in rng.sample(range(nodes), 3):
                text = texts[b] + [ids[b][j] for j in sorted(sets[i])]
                one, n = layer(12), len(text)
                s = CacheStep(_i32([0, n]), _i32([n]), _i32([list(range(12))]), n, n, 192)
                alone = ops.paged_attention(ops.kv_cache_write(embed[torch.tensor(text, device=DEV)], one, s, H, cos, sin), one, s, H, hd**-0.5)
                r = b * nodes + i
                # the same values in another order of places: two roundings of the output, and sums in fp32
                assert float((alone[-1].float() - y[r].float()).abs().max()) <= 2 * _u(dtype) * float(y[r].float().abs().max()) + 1e-4
        ops.kv_cache_keep(cache, step, kept, counts)
        keep = keep + counts
        got = counts.tolist()
        for b in range(B):
            path = kept[b, : got[b]].tolist()
            texts[b] += [ids[b][j] for j in path]
            roots[b] = int(chosen[b, got[b] - 1])
            assert chosen[b, : got[b] - 1].tolist() == [ids[b][j] for j in path[1:]]
        if turn == 1:
            assert max(got) > 1
    # the cache holds the texts
    step = ops.cache_tables(tables, _i32([0] * B), 0, 1, 192, keep=keep)
    assert step.kv_len.tolist() == [len(t) for t in texts]
    start = _i32([0] + [sum(len(t) for t in texts[: b + 1]) for b in range(B)])
    total = sum(map(len, texts))
    k, v = ops.kv_cache_read(cache, tables.page_table, start, total, dtype)
    for b, text in enumerate(texts):
        one, n = layer(12), len(text)
        s = CacheStep(_i32([0, n]), _i32([n]), _i32([list(range(12))]), n, n, 192)
        ops.kv_cache_write(embed[torch.tensor(text, device=DEV)], one, s, H, cos, sin)
        wk, wv = ops.kv_cache_read(one, s.page_table, _i32([0, n]), n, dtype)
        lo = int(start[b])
        assert torch.equal(k[lo : lo + n], wk) and torch.equal(v[lo : lo + n], wv)


def test_a_captured_step_on_its_own_stream():
    """Tables, write, attention, verification and keep in one graph, replayed
    with other inputs beside eager work, against the same calls one by one."""
    dtype, H, KV, hd, page, V, B, nodes = BF16, 4, 2, 64, 16, 700, 4, 8
    g = torch.Generator().manual_seed(2)
    rng = random.Random(2)
    angle = torch.rand(256, hd, generator=g) * 6
    cos, sin = angle.cos().to(dtype).to(DEV), angle.sin().to(dtype).to(DEV)
    parents = _i32(_trees(rng, B, nodes))

    def state():
        gen = torch.Generator().manual_seed(7)
        k, v = (torch.randn(3, 60, KV, page, hd, generator=gen).to(dtype).to(DEV) for _ in range(2))
        tables = PageTables(torch.full((B, 14), -1, dtype=torch.int32, device=DEV), _i32([0] * B),
                            torch.arange(60, dtype=torch.int32, device=DEV), _i32([60]), page)
        ops.cache_tables(tables, _i32([50, 3, 20, 100]), 173, 100, 224)
        return LayerCache(k, v), tables

    def one(cache, tables, keep, qkv, ids, logits, u):
        step = ops.cache_tables(tables, _new, B * nodes, nodes, 224, keep=keep, parents=parents)
        outs = []
        for i in range(3):
            layer = LayerCache(cache.k[i], cache.v[i])
            q = ops.kv_cache_write(qkv, layer, step, H, cos, sin)
            outs.append(ops.paged_attention(q, layer, step, H, hd**-0.5))
        counts, kept, chosen = ops.verify_draft(logits, ids, step.row_start, nodes, u, parents=parents)
        ops.kv_cache_keep(cache, step, kept, counts)
        keep.add_(counts)
        return [*outs, counts, kept, chosen]

    _new = _i32([nodes] * B)
    (ca, ta), (cb, tb) = state(), state()
    ka, kb = ta.lengths.clone(), tb.lengths.clone()
    inputs = [torch.randn(B * nodes, (H + 2 * KV) * hd, generator=g).to(dtype).to(DEV), torch.randint(0, 3, (B * nodes,), generator=g).to(DEV),
              torch.randn(B * nodes, V, generator=g).to(DEV), torch.rand(B * nodes, generator=g, dtype=torch.float64).to(DEV)]
    _lib.tensor_calls()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = one(cb, tb, kb, *inputs)
    for turn in range(4):
        inputs[0].copy_(torch.randn(inputs[0].shape, generator=g).to(dtype))
        inputs[2].copy_(torch.randn(inputs[2].shape, generator=g) + 8 * (torch.arange(V) < 3))
        inputs[3].copy_(torch.rand(B * nodes, generator=g, dtype=torch.float64))
        graph.replay()
        want = one(ca, ta, ka, *inputs)
        torch.cuda.synchronize()
        for x, y in zip(captured, want):
            assert torch.equal(x, y)
        assert torch.equal(ca.k, cb.k) and torch.equal(ca.v, cb.v) and torch.equal(ka, kb)
        assert torch.equal(ta.page_table, tb.page_table) and torch.equal(ta.free[: int(ta.n_free)], tb.free[: int(tb.n_free)])


def test_two_graphs_on_two_streams():
    """Calls with workspaces, captured twice and replayed at the same time."""
    H, KV, hd, V = 16, 4, 64, 40001
    cases, graphs, outs, wants = [], [], [], []
    for seed in range(2):
        c, _ = _tree_case([(16, 4500), (9, 3000), (0, 70)], [4484, 2990, 70], KV, hd, 64, BF16, seed=seed)
        q = torch.randn(c.rows, H * hd, generator=c.g).to(BF16).to(DEV)
        logits = 3 * torch.randn(c.rows, V, generator=c.g).to(DEV)
        probs = torch.softmax(logits.roll(1, 0) + torch.randn(c.rows, V, generator=c.g).to(DEV), -1)
        tokens, u = torch.multinomial(probs, 1)[:, 0], torch.rand(c.rows, generator=c.g).to(DEV)
        cases.append((c, q, logits, probs, tokens, u))

    def run(c, q, logits, probs, tokens, u):
        return [ops.paged_attention(q, c.layer, c.draft, H, hd**-0.5),
                *ops.verify_draft(logits, tokens, c.draft.row_start, 16, u, draft_probs=probs),
                *ops.verify_draft(logits, tokens, c.draft.row_start, 16, u)]

    for case in cases:
        wants.append(run(*case))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(*case))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for s, g, out in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                for o in out:
                    o.zero_()
                g.replay()
        again = run(*cases[0])  # beside them
        torch.cuda.synchronize()
        for out, want in zip([*outs, again], [*wants, wants[0]]):
            assert all(torch.equal(x, y) for x, y in zip(out, want))
