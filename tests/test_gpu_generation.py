"""Generation from a paged key/value cache: cache write and read, attention
over the cache, logit adjustment, and the model's cached forward, against
plain float64 restatements on the CPU.

Tolerances count roundings: u = finfo.eps / 2 of a type is the most that one
rounding to it changes a value, relative to it; u32 = 2^-24.
"""
from __future__ import annotations

import math

import pytest
import torch

from lzhip import ops
from lzhip.cache import CacheStep, KVCache, LayerCache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
U32 = 2.0**-24
# A bound on the lengths (CacheStep.max_len) with which sequences of 64 packed
# rows or more take 128-row tiles, however short they are.
MUCH = 2**20


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _exp_of(x, dtype):
    """The exponent of a float32 head's e4m3 storage, one at a time."""
    finite = [abs(float(y)) for y in x if math.isfinite(float(y))]
    amax = max(finite, default=0.0)
    if amax == 0.0:
        return 0
    e = math.frexp(amax)[1] - 9
    while amax > 448 * 2.0**e:
        e += 1
    return min(max(e, -15), 7) if dtype == F16 else min(max(e, -120), 119)


def _quantise(x, dtype):
    """float32 [..., hd] -> (e4m3 bytes as float64 values, exponents)."""
    flat = x.reshape(-1, x.shape[-1])
    e = torch.tensor([_exp_of(row, dtype) for row in flat], dtype=torch.int32).view(x.shape[:-1])
    y = x.double() * torch.ldexp(torch.ones(e.shape, dtype=torch.float64), -e)[..., None]
    y = torch.where(x.isinf(), torch.full_like(y, math.nan), y.clamp(-448, 448))
    return y.float().to(E4M3), e.to(torch.int8)


class Case:
    """A cache layer in random pages, the step of (new, length) sequences and
    the same on the CPU in float64."""

    def __init__(self, seqs, KV, hd, page, dtype, e4m3=False, seed=0, spare=2, fill=None, most=0):
        self.seqs, self.KV, self.hd, self.page, self.dtype, self.e4m3 = seqs, KV, hd, page, dtype, e4m3
        g = torch.Generator().manual_seed(seed)
        self.g = g
        need = [-(-l // page) for _, l in seqs]
        n_pages = sum(need) + spare
        order = torch.randperm(n_pages, generator=g).tolist()
        width = max(1, max(need))
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.starts, self.rows = starts, starts[-1]
        shape = (n_pages, KV, page, hd)
        self.cpu, self.exps = [], [None, None]
        for i in range(2):
            x = torch.randn(shape, generator=g)
            if fill is not None:  # what lies in slots of no token
                x = x.to(dtype)
                used = torch.zeros(n_pages, page, dtype=torch.bool)
                for b, (_, l) in enumerate(seqs):
                    for p in range(l):
                        used[self.table[b, p // page], p % page] = True
                x = torch.where(used[:, None, :, None], x, torch.full_like(x, fill))
            if e4m3:
                self.exps[i] = torch.randint(-9, -5, shape[:3], generator=g).to(torch.int8)
                x = (x * 64).clamp(-448, 448).float().to(E4M3)
            else:
                x = x.to(dtype)
            self.cpu.append(x)
        dev = [t.to(DEV) for t in self.cpu]
        self.layer = LayerCache(*dev, *(None if e is None else e.to(DEV) for e in self.exps))
        self.step = CacheStep(torch.tensor(starts, dtype=torch.int32, device=DEV),
                              torch.tensor([l for _, l in seqs], dtype=torch.int32, device=DEV), self.table.to(DEV),
                              self.rows, max(n for n, _ in seqs), max(most, max(l for _, l in seqs)))

    def tokens(self, side, b, length=None):
        """[length, KV, hd] float64 of sequence b's keys (0) or values (1)."""
        length = self.seqs[b][1] if length is None else length
        p = torch.arange(length)
        pages, slots = self.table[b, p // self.page].long(), p % self.page
        x = self.cpu[side][pages, :, slots].double()
        if self.e4m3:
            x = x * torch.ldexp(torch.ones(1, dtype=torch.float64), self.exps[side][pages, :, slots].int())[..., None]
        return x

    def attention(self, q, H, scale):
        """(o, bound) in float64: bound counts one rounding of the weights and
        of the output to the type, and fp32 sums."""
        q = q.double().cpu().view(-1, H, self.hd)
        o, tol = torch.zeros_like(q), torch.zeros_like(q)
        u = _u(self.dtype)
        for b, (n, l) in enumerate(self.seqs):
            k, v = self.tokens(0, b), self.tokens(1, b)
            for i in range(n):
                seen, r = l - n + i + 1, self.starts[b] + i
                if seen <= 0:
                    continue
                for h in range(H):
                    g = h // (H // self.KV)
                    s = k[:seen, g] @ q[r, h] * scale
                    size = float((k[:seen, g].abs() @ q[r, h].abs()).max()) * scale
                    p = torch.softmax(s, 0)
                    o[r, h] = p @ v[:seen, g]
                    a = p @ v[:seen, g].abs()
                    # a score is hd products and adds of fp32 and a few units
                    # of the exponent's argument; sums of `seen` terms
                    fp32 = (2 * (self.hd + 4) * size + 8 + seen) * U32
                    weights = u if self.dtype != F32 else 0.0
                    tol[r, h] = u * o[r, h].abs() + (weights + fp32) * a
        return o.view(-1, H * self.hd), tol.view(-1, H * self.hd)


def _tables(positions, hd, dtype):
    inv = 10_000.0 ** (-torch.arange(0, hd, 2).double() / hd)
    a = torch.arange(positions).double()[:, None] * inv
    a = torch.cat([a, a], 1)
    return a.cos().to(dtype), a.sin().to(dtype)


def _rotated(x, positions, cos, sin):
    """float32 rotation, each product and sum rounded (IEEE on the CPU)."""
    h = x.shape[-1] // 2
    c, s = cos.float()[positions][:, None], sin.float()[positions][:, None]
    x = x.float()
    half = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * c + half * s


SEQS = {
    "one": [(1, 1)],
    "decode": [(1, 5), (1, 130), (1, 64), (1, 1), (1, 33)],
    "ragged": [(3, 3), (0, 17), (40, 100), (1, 16), (17, 17), (0, 0), (5, 65)],
}


@pytest.mark.parametrize("seqs", sorted(SEQS))
@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (F32, False), (BF16, True), (F16, True), (F32, True)])
@pytest.mark.parametrize("H,KV,hd,page", [(8, 4, 32, 16), (12, 4, 64, 32), (5, 5, 128, 16)])
def test_cache_write(seqs, dtype, e4m3, H, KV, hd, page):
    """q, the pages' new tokens and nothing else."""
    c = Case(SEQS[seqs], KV, hd, page, dtype, e4m3, seed=hd + page)
    wide = (torch.randn(c.rows, (H + 2 * KV) * hd + 16, generator=c.g) * 3).to(dtype)
    qkv = wide[:, : (H + 2 * KV) * hd]
    cos, sin = _tables(c.step.max_len + 3, hd, dtype)
    q = ops.kv_cache_write(wide.to(DEV)[:, : (H + 2 * KV) * hd], c.layer, c.step, H, cos.to(DEV), sin.to(DEV))
    pos = torch.cat([torch.arange(l - n, l) for n, l in c.seqs])
    x = qkv.reshape(c.rows, H + 2 * KV, hd)
    qk = _rotated(x[:, : H + KV], pos, cos, sin)
    assert torch.equal(q.cpu(), qk[:, :H].reshape(c.rows, -1).to(dtype))
    at = 0
    for side, new in ((0, qk[:, H:]), (1, x[:, H + KV :].float())):
        want, exps = c.cpu[side].clone().view(torch.uint8) if e4m3 else c.cpu[side].clone(), c.exps[side]
        vals = _quantise(new, dtype) if e4m3 else (new.to(dtype), None)
        exps = exps.clone() if e4m3 else None
        at = 0
        for b, (n, l) in enumerate(c.seqs):
            for i in range(n):
                p = l - n + i
                want[c.table[b, p // page], :, p % page] = vals[0][at].view(torch.uint8) if e4m3 else vals[0][at]
                if e4m3:
                    exps[c.table[b, p // page], :, p % page] = vals[1][at]
                at += 1
        got = (c.layer.k, c.layer.v)[side].cpu()
        assert torch.equal(got.view(torch.uint8) if e4m3 else got, want)
        if e4m3:
            assert torch.equal((c.layer.k_exp, c.layer.v_exp)[side].cpu(), exps)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_cache_write_e4m3_borders(dtype):
    """Heads of zeros, at and around 448 * 2^e, of the type's smallest and
    largest values, with ties, infinities and NaN."""
    hd, top = 32, float(torch.finfo(dtype).max)
    rows = [[0.0] * hd, [448.0] + [1.0] * 31, [-450.0] + [17.0, 19.0, 21.0] + [0.0] * 28, [top, -top, 1.0] + [0.5] * 29,
            [float(torch.finfo(dtype).tiny)] * hd, [2.0**-24] + [0.0] * 31, [math.inf, 3.0, -2.0] + [0.0] * 29,
            [math.nan, -math.inf, 100.0] + [-0.0] * 29, [math.nan] * hd, [65504.0, 2.0**-20] + [57344.0] * 30]
    x = torch.tensor(rows).clamp(-top, top).to(dtype)
    n = len(rows)
    c = Case([(n, n)], 1, hd, 16, dtype, True)
    qkv = torch.cat([torch.zeros(n, hd, dtype=dtype), x, x.flip(1)], 1)  # q, k, v
    cos, sin = torch.ones(n, hd, dtype=dtype), torch.zeros(n, hd, dtype=dtype)
    ops.kv_cache_write(qkv.to(DEV), c.layer, c.step, 1, cos.to(DEV), sin.to(DEV))
    start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    k, v = ops.kv_cache_read(c.layer, c.step.page_table, start, n, F32)
    for got, rows_ in ((k, x.float()), (v, x.flip(1).float())):
        if got is k:  # 0 * inf in the rotation
            rows_ = _rotated(rows_[:, None], torch.arange(n), cos, sin)[:, 0]
        y, e = _quantise(rows_, dtype)
        want = y.float() * torch.ldexp(torch.ones(n), e.int())[:, None]
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=1e30), torch.nan_to_num(want, nan=1e30))
        ok = torch.isfinite(rows_) & (rows_.abs() <= 448 * torch.ldexp(torch.ones(n), e.int())[:, None])
        err = (got.cpu().double() - rows_.double()).abs()
        # half a step: 2^-4 of a normal value, 2^-10 * 2^e below 2^-6 * 2^e
        half = torch.maximum(2.0**-4 * rows_.double().abs(), torch.ldexp(torch.ones(n).double(), e.int() - 10)[:, None])
        assert bool((err <= half)[ok].all())


@pytest.mark.parametrize("dtype,e4m3,out", [(BF16, False, BF16), (F16, False, F16), (F32, False, F32), (BF16, True, BF16),
                                            (F16, True, F16), (F32, True, F32)])
@pytest.mark.parametrize("KV,hd,page", [(3, 32, 16), (4, 64, 64), (8, 128, 32)])
def test_cache_read(dtype, e4m3, out, KV, hd, page):
    c = Case(SEQS["ragged"], KV, hd, page, dtype, e4m3)
    lens = [min(l, 70) for _, l in c.seqs]
    start = torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32)
    k, v = ops.kv_cache_read(c.layer, c.step.page_table, start.to(DEV), int(start[-1]), out)
    for side, got in ((0, k), (1, v)):
        want = torch.cat([c.tokens(side, b, n) for b, n in enumerate(lens)]).reshape(-1, KV * hd)
        assert torch.equal(got.cpu(), want.to(out))


def test_cache_read_rows_of_no_sequence():
    c = Case([(1, 20), (1, 20)], 2, 64, 16, BF16)
    spare = torch.full((13, 128), 7.0, dtype=BF16, device=DEV)  # what new memory may hold
    del spare
    k, v = ops.kv_cache_read(c.layer, c.step.page_table, torch.tensor([2, 6, 9], dtype=torch.int32, device=DEV), 13, BF16)
    for side, got in ((0, k), (1, v)):
        want = torch.zeros(13, 2, 64, dtype=torch.float64)
        want[2:6], want[6:9] = c.tokens(side, 0, 4), c.tokens(side, 1, 3)
        assert torch.equal(got.cpu().double(), want.view(13, 128))


def _check_attention(c, H, scale=None, q=None, **kw):
    scale = c.hd**-0.5 if scale is None else scale
    q = torch.randn(c.rows, H * c.hd, generator=c.g).to(c.dtype) if q is None else q
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, scale, **kw).cpu().double()
    want, tol = c.attention(q, H, scale)
    assert bool(torch.isfinite(got).all())
    over = (got - want).abs() - tol
    assert float(over.max()) <= 0, (float((got - want).abs().max()), float(over.max()))
    return got


@pytest.mark.parametrize("seqs", sorted(SEQS))
@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (F32, False), (BF16, True), (F16, True), (F32, True)])
@pytest.mark.parametrize("H,KV,hd,page", [(10, 2, 32, 16), (12, 4, 64, 32), (5, 5, 128, 16), (32, 8, 128, 64)])
@pytest.mark.parametrize("most", [0, MUCH])
def test_paged_attention(seqs, dtype, e4m3, H, KV, hd, page, most):
    _check_attention(Case(SEQS[seqs], KV, hd, page, dtype, e4m3, seed=H + hd, fill=None if e4m3 else math.nan, most=most), H)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, True), (F32, False)])
@pytest.mark.parametrize("n,length,H,KV,hd,page", [
    (1, 1500, 8, 4, 32, 16),      # one token over many pages
    (1, 4100, 2, 1, 64, 256),
    (2, 2047, 4, 1, 128, 64),     # few rows, long
    (129, 129, 6, 2, 64, 32),     # a prompt one past a tile
    (64, 700, 4, 2, 128, 16),     # a chunk whose first rows end inside a page
    (33, 257, 33, 1, 32, 128),    # 33 heads on one
])
@pytest.mark.parametrize("most", [0, MUCH])
def test_paged_attention_lengths(dtype, e4m3, n, length, H, KV, hd, page, most):
    c = Case([(n, length), (min(n, 3), 3)], KV, hd, page, dtype, e4m3, seed=length, fill=None if e4m3 else math.inf, most=most)
    _check_attention(c, H)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("seqs,H,KV", [
    ([(1, 1 + 7 * b % 40) for b in range(300)], 2, 1),                          # more sequences than threads
    ([(1, 1 + b % 3) for b in range(1100)], 1, 1),                              # more than the tables in LDS hold
    ([(1 + b % 5, 1 + b % 5 + b % 17) for b in range(1030)], 1, 1),
    ([(b % 37, b % 37 + 11 * b % 50) for b in range(70)], 8, 2),                # chunks of more than 64 sequences
    ([(3, 90), (70, 71), (0, 0), (33, 400), (1, 1)], 12, 3),                    # chunks beside single tokens
    ([(1, 1 + 237 * b % 1500) for b in range(40)], 8, 8),                       # a few more heads than CUs
])
def test_many_sequences(seqs, H, KV, e4m3):
    """Attention, write and read of long lists of sequences."""
    c = Case(seqs, KV, 32, 16, BF16, e4m3, seed=len(seqs), fill=None if e4m3 else math.nan)
    _check_attention(c, H)
    step, c.step = c.step, c.step._replace(max_len=MUCH)
    _check_attention(c, H)
    c.step = step
    n = [min(l, 20) for _, l in seqs]
    start = torch.tensor([sum(n[:b]) for b in range(len(n) + 1)], dtype=torch.int32)
    k, _ = ops.kv_cache_read(c.layer, c.step.page_table, start.to(DEV), int(start[-1]), BF16)
    want = torch.cat([c.tokens(0, b, m) for b, m in enumerate(n)]).reshape(-1, KV * 32)
    assert torch.equal(k.cpu(), want.to(BF16))
    cos, sin = _tables(c.step.max_len, 32, BF16)
    qkv = torch.randn(c.rows, (H + 2 * KV) * 32, generator=c.g).to(BF16)
    q = ops.kv_cache_write(qkv.to(DEV), c.layer, c.step, H, cos.to(DEV), sin.to(DEV))
    pos = torch.cat([torch.arange(l - m, l) for m, l in seqs])
    x = _rotated(qkv.view(c.rows, -1, 32)[:, : H + KV], pos, cos, sin)
    assert torch.equal(q.cpu(), x[:, :H].reshape(c.rows, -1).to(BF16))
    start = torch.tensor([sum(l for _, l in seqs[:b]) for b in range(len(seqs) + 1)], dtype=torch.int32)
    _, v = ops.kv_cache_read(c.layer, c.step.page_table, start.to(DEV), int(start[-1]), F32 if e4m3 else BF16)
    new = torch.cat([torch.arange(int(start[b]) + l - m, int(start[b]) + l) for b, (m, l) in enumerate(seqs)])
    want = qkv[:, (H + KV) * 32 :].reshape(-1, 32)
    if e4m3:
        y, e = _quantise(want.float(), BF16)
        want = y.float() * torch.ldexp(torch.ones(1), e.int())[:, None]
    assert torch.equal(v.cpu()[new].reshape(-1, 32), want)


@pytest.mark.parametrize("new,bound", [(1, 100), (1, 5000), (40, 100), (40, 5000), (40, 12000), (130, 12000), (130, 6000)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_bound_on_the_length_only_splits(new, bound, e4m3):
    """max_len below and above the sequences' lengths: the same attention."""
    c = Case([(new, 1300), (1, 40)], 2, 64, 32, BF16, e4m3, seed=bound)
    c.step = c.step._replace(max_len=bound)
    _check_attention(c, 8)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (BF16, True), (F32, False), (F16, True)])
@pytest.mark.parametrize("news", [[64, 1, 1, 30, 1], [1, 1, 1], [200, 90]])
@pytest.mark.parametrize("most", [0, MUCH])
def test_steps_of_a_layer(news, dtype, e4m3, most):
    """Write, then attend, step after step: each row against the attention of
    the whole text over what the cache holds."""
    H, KV, hd, page = 8, 2, 64, 32
    total = sum(news)
    g = torch.Generator().manual_seed(total)
    cache = KVCache(1, KV, hd, batch=2, n_pages=2 * -(-total // page), page_size=page, dtype=dtype,
                    storage=E4M3 if e4m3 else None, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(total, hd, dtype))
    done = 0
    for n in news:
        step = cache.step([n, n])
        qkv = torch.randn(2 * n, (H + 2 * KV) * hd, generator=g).to(dtype).to(DEV)
        q = ops.kv_cache_write(qkv, cache.layers[0], step, H, cos, sin)
        step = step._replace(max_len=max(most, step.max_len))
        o = ops.paged_attention(q, cache.layers[0], step, H, hd**-0.5).double().cpu().view(2, n, H, hd)
        for b in range(2):
            k, v = (t.double().cpu() for t in cache.read(0, b))
            x = q.double().cpu().view(2, n, H, hd)[b]
            for i in (0, n // 2, n - 1):
                seen = done + i + 1
                for h in range(H):
                    kk, vv = k[:seen, h // 4], v[:seen, h // 4]
                    p = torch.softmax(kk @ x[i, h] * hd**-0.5, 0)
                    size = float((kk.abs() @ x[i, h].abs()).max()) * hd**-0.5
                    u = _u(dtype)
                    fp32 = (2 * (hd + 4) * size + 8 + seen) * U32
                    tol = u * (p @ vv).abs() + ((u if dtype != F32 else 0.0) + fp32) * (p @ vv.abs())
                    assert bool(((o[b, i, h] - p @ vv).abs() <= tol).all()), (n, b, i, h)
        done += n


def test_a_captured_step_follows_its_tables():
    """One decoded token captured with its lengths on the device: every replay
    one token further, against eager calls."""
    H, KV, hd, page = 8, 2, 64, 16
    caches = [KVCache(1, KV, hd, batch=3, n_pages=60, page_size=page, device=DEV) for _ in range(2)]
    lens, most = [5, 250, 31], 320
    g = torch.Generator().manual_seed(2)
    cos, sin = (t.to(DEV) for t in _tables(most, hd, BF16))
    first = torch.randn(sum(lens), (H + 2 * KV) * hd, generator=g).to(BF16).to(DEV)
    filled = [cache.step(lens) for cache in caches]
    # the captured side: pages for what comes, lengths and the input in place
    cache = caches[0]
    table = cache.step([40] * 3).page_table.clone()
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    each = CacheStep(torch.arange(4, dtype=torch.int32, device=DEV), kv, table, 3, 1, most)
    x = torch.zeros(3, (H + 2 * KV) * hd, dtype=BF16, device=DEV)
    layer = cache.layers[0]

    def once():
        return ops.paged_attention(ops.kv_cache_write(x, layer, each, H, cos, sin), layer, each, H, 0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for cache, step in zip(caches, filled):  # after the warm-up, which wrote its last tokens
        ops.kv_cache_write(first, cache.layers[0], step, H, cos, sin)
    for turn in range(6):
        new = torch.randn(3, (H + 2 * KV) * hd, generator=g).to(BF16)
        x.copy_(new)
        kv += 1
        graph.replay()
        torch.cuda.synchronize()
        s = caches[1].step([1] * 3)._replace(max_len=most)  # split alike
        q = ops.kv_cache_write(new.to(DEV), caches[1].layers[0], s, H, cos, sin)
        assert torch.equal(out, ops.paged_attention(q, caches[1].layers[0], s, H, 0.125)), turn


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,length,most", [(1, 600, 0), (70, 300, 0), (200, 200, 0), (70, 300, MUCH), (200, 200, MUCH)])
def test_paged_attention_large_scores(dtype, n, length, most):
    """Scores in the hundreds: one key takes nearly all the weight, and the
    running maximum moves late."""
    c = Case([(n, length)], 2, 64, 32, dtype, seed=n, most=most)
    q = (torch.randn(c.rows, 4 * 64, generator=c.g) * 12).to(dtype)
    _check_attention(c, 4, scale=0.5, q=q)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (F32, False), (BF16, True)])
@pytest.mark.parametrize("n,length,most", [(1, 200, 0), (150, 200, 0), (16, 40, 0), (150, 200, MUCH), (40, 40, MUCH)])
def test_paged_attention_nonfinite_reaches_only_who_sees_it(dtype, e4m3, n, length, most):
    """An infinity or NaN among the last new token's keys and values leaves
    the rows before it as they were."""
    c = Case([(n, length), (1, 9)], 2, 64, 32, dtype, e4m3, seed=7, most=most)
    q = torch.randn(c.rows, 4 * 64, generator=c.g).to(dtype).to(DEV)
    before = ops.paged_attention(q, c.layer, c.step, 4, 0.125)
    p = length - 1
    page, slot = int(c.table[0, p // 32]), p % 32
    bad = math.nan if e4m3 else math.inf
    c.layer.v[page, :, slot, 3:5] = torch.tensor(bad, device=DEV).to(c.layer.v.dtype)
    c.layer.k[page, 1, slot, 2] = torch.tensor(math.nan, device=DEV).to(c.layer.k.dtype)
    after = ops.paged_attention(q, c.layer, c.step, 4, 0.125)
    assert torch.equal(after[: n - 1], before[: n - 1])
    assert torch.equal(after[n:], before[n:])
    assert not torch.isfinite(after[n - 1]).all()


def test_paged_attention_rows_that_see_nothing():
    """More new tokens than the sequence has, and a sequence of none: their
    rows are zeros; rows past the last sequence stay."""
    c = Case([(4, 4), (1, 1), (3, 40)], 2, 64, 16, BF16)
    step = c.step._replace(kv_len=torch.tensor([2, 0, 40], dtype=torch.int32, device=DEV))
    q = torch.randn(c.rows + 5, 4 * 64, generator=c.g).to(BF16).to(DEV)
    out = torch.full((c.rows + 5, 256), 7.0, dtype=BF16, device=DEV)
    ops.paged_attention(q, c.layer, step, 4, 0.125, out=out)
    assert bool((out[:2] == 0).all()) and bool((out[4] == 0).all()) and bool((out[c.rows :] == 7).all())
    assert bool((out[2:4] != 0).any()) and bool((out[5:8] != 0).any())
    fresh = ops.paged_attention(q, c.layer, step, 4, 0.125)
    assert torch.equal(fresh[: c.rows], out[: c.rows]) and bool((fresh[c.rows :] == 0).all())
    # and in the write: no position, no page, nothing written
    cos, sin = (t.to(DEV) for t in _tables(64, 64, BF16))
    qkv = torch.randn(c.rows + 5, 8 * 64, generator=c.g).to(BF16).to(DEV)
    k0 = c.layer.k.clone()
    out.fill_(7.0)
    ops.kv_cache_write(qkv, c.layer, step, 4, cos, sin, out=out)
    assert bool((out[:2] == 0).all()) and bool((out[4] == 0).all()) and bool((out[c.rows :] == 7).all())
    changed = (c.layer.k != k0).flatten(2).any(2).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {int(c.table[0, 0]), int(c.table[2, 2])}


def test_bad_pages_are_left_out():
    """Page ids outside the pool: nothing is written or read there, and
    attention goes over the other pages."""
    c = Case([(2, 80), (1, 20)], 1, 64, 16, F32)
    table = c.table.clone()
    table[0, 1], table[0, 4], table[1, 1] = -5, 10_000_000, 2**31 - 1
    step = c.step._replace(page_table=table.to(DEV))
    q = torch.randn(3, 64, generator=c.g)
    got = ops.paged_attention(q.to(DEV), c.layer, step, 1, 0.125).cpu().double()
    for row, b, keep in ((0, 0, [p for p in range(79) if p // 16 not in (1, 4)]),
                         (1, 0, [p for p in range(80) if p // 16 not in (1, 4)]), (2, 1, list(range(16)))):
        k, v = c.tokens(0, b)[keep, 0], c.tokens(1, b)[keep, 0]
        want = torch.softmax(k @ q[row].double() * 0.125, 0) @ v
        assert float((got[row] - want).abs().max()) <= 400 * U32 * float(v.abs().max())
    k0, v0 = c.layer.k.clone(), c.layer.v.clone()
    cos, sin = (t.to(DEV) for t in _tables(80, 64, F32))
    ops.kv_cache_write(torch.randn(3, 3 * 64, generator=c.g).to(DEV), c.layer, step, 1, cos, sin)
    assert torch.equal(c.layer.k, k0) and torch.equal(c.layer.v, v0)  # all three new tokens are on bad pages
    start = torch.tensor([0, 80, 100], dtype=torch.int32, device=DEV)
    k, _ = ops.kv_cache_read(c.layer, step.page_table, start, 100, F32)
    assert bool((k[16:32] == 0).all()) and bool((k[64:80] == 0).all()) and bool((k[96:] == 0).all())
    assert torch.equal(k[:16].cpu().double(), c.tokens(0, 0)[:16, 0])


@pytest.mark.parametrize("most", [0, MUCH])
@pytest.mark.parametrize("e4m3", [False, True])
def test_chunks_that_see_nothing_and_bad_pages(e4m3, most):
    """Chunks with more new tokens than the sequence has, one of no sequence at
    all and one over pages outside the pool."""
    c = Case([(90, 90), (40, 40), (70, 200)], 1, 64, 16, BF16, e4m3, most=most)
    table = c.table.clone()
    table[2, 1], table[2, 4], table[2, 9] = -5, 10_000_000, 2**31 - 1
    step = c.step._replace(kv_len=torch.tensor([50, 0, 200], dtype=torch.int32, device=DEV), page_table=table.to(DEV))
    q = torch.randn(c.rows + 3, 64, generator=c.g).to(BF16)
    got = ops.paged_attention(q.to(DEV), c.layer, step, 1, 0.125, out=torch.full((c.rows + 3, 64), 7.0, dtype=BF16, device=DEV))
    got = got.cpu().double()
    assert bool((got[:40] == 0).all()) and bool((got[90:130] == 0).all()) and bool((got[c.rows :] == 7).all())
    u = _u(BF16)
    for row in range(c.rows):
        b, keep = (0, range(row - 40 + 1)) if row < 90 else (2, [p for p in range(row + 1) if p // 16 not in (1, 4, 9)])
        if len(keep) == 0 or 90 <= row < 130:
            continue
        k, v = c.tokens(0, b)[list(keep), 0], c.tokens(1, b)[list(keep), 0]
        p = torch.softmax(k @ q[row].double() * 0.125, 0)
        want, size = p @ v, p @ v.abs()
        top = float((k.abs() @ q[row].double().abs()).max()) * 0.125
        fp32 = (2 * (64 + 4) * top + 8 + len(keep)) * U32  # as in Case.attention
        assert bool(((got[row] - want).abs() <= u * want.abs() + (u + fp32) * size).all()), row


def test_pages_past_two_to_the_31_elements():
    """Page ids whose element offsets need 64 bits."""
    pages, page, hd = 2**15 + 40, 1024, 64
    k, v = (torch.empty(pages, 1, page, hd, dtype=BF16, device=DEV) for _ in range(2))
    far = [pages - 1, 2**15 - 1, 2**15 + 1]
    for p in far:
        k[p].normal_()
        v[p].normal_()
    length = 2 * page + 100
    step = CacheStep(*(torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 1], [length], [far])), 1, 1, length)
    layer = LayerCache(k, v)
    cos, sin = (t.to(DEV) for t in _tables(length, hd, BF16))
    qkv = torch.randn(1, 3 * hd, device=DEV).to(BF16)
    q = ops.kv_cache_write(qkv, layer, step, 1, cos, sin)
    got = ops.paged_attention(q, layer, step, 1, 0.125).double()
    kk, vv = (torch.cat([t[p, 0] for p in far])[:length].double() for t in (k, v))
    assert torch.equal(vv[-1].to(BF16), qkv[0, 2 * hd :])
    p = torch.softmax(kk @ q[0].double() * 0.125, 0)
    tol = _u(BF16) * (p @ vv).abs() + (_u(BF16) + 4096 * U32) * (p @ vv.abs())
    assert bool(((got[0] - p @ vv).abs() <= tol).all())
    rk, _ = ops.kv_cache_read(layer, step.page_table, torch.tensor([0, length], dtype=torch.int32, device=DEV), length, BF16)
    assert torch.equal(rk.double(), kk)


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------

def _logits_oracle(x, tokens, lengths, prompts, rep, pres, freq, bias, mask):
    x = x.double().clone()
    size = x.abs()
    for b in range(x.shape[0]):
        V = x.shape[1]
        text = tokens[b, : lengths[b]].tolist() if tokens is not None else []
        for t in set(text):
            if 0 <= t < V:
                x[b, t] = x[b, t] / rep[b] if x[b, t] > 0 else x[b, t] * rep[b]
        answer = text[prompts[b] :]
        for t in set(answer):
            if 0 <= t < V:
                x[b, t] -= freq[b] * answer.count(t) + pres[b]
                size[b, t] += freq[b] * answer.count(t) + pres[b]
    size = size * max(1.0, max(float(r) for r in rep))
    if bias is not None:
        x = x + bias.double()
        size = size + bias.double().abs()
    if mask is not None:
        x = x.masked_fill(~mask, -math.inf)
    return x, 6 * U32 * size  # at most six fp32 operations


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,V,T,bias,mask", [(1, 1, 1, "", ""), (1, 32000, 37, "shared", ""), (3, 4097, 300, "rows", "bits"),
                                             (2, 8191, 5000, "", "bools"), (5, 100, 0, "rows", "shared bits"),
                                             (2, 10007, 64, "shared", "shared bools"),
                                             (64, 70001, 20, "rows", "bits"), (70, 65536, 9, "shared", "bools")])
def test_process_logits(dtype, B, V, T, bias, mask):
    g = torch.Generator().manual_seed(B * V + T)
    wide = (3 * torch.randn(B, 2, V + 3, generator=g)).to(dtype)
    x = wide[:, 1, :V]
    tokens = torch.randint(-3, min(V, 50) + 3, (B, T + 2), generator=g)
    lengths = torch.randint(0, T + 1, (B,), generator=g)
    lengths[0] = T
    prompts = (lengths * torch.rand(B, generator=g)).long()
    rep, pres, freq = 1 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g)
    bs = torch.randn((V,) if bias == "shared" else (B, V), generator=g) if bias else None
    allowed = torch.rand((V,) if "shared" in mask else (B, V), generator=g) < 0.5 if mask else None
    packed = allowed
    if "bits" in mask:
        pad = torch.zeros(*allowed.shape[:-1], -(-V // 32) * 32, dtype=torch.int64)
        pad[..., :V] = allowed
        packed = (pad.view(*allowed.shape[:-1], -1, 32) << torch.arange(32)).sum(-1).to(torch.int32)
    want, tol = _logits_oracle(x, tokens, lengths, prompts, rep, pres, freq, bs, allowed)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got = ops.process_logits(dev(wide)[:, 1, :V], tokens=dev(tokens)[:, : T + 1], lengths=dev(lengths),
                             prompt_lengths=dev(prompts.int()), repetition_penalty=dev(rep), presence_penalty=dev(pres),
                             frequency_penalty=dev(freq), bias=dev(bs), mask=dev(packed)).cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    assert bool(((got - want).abs() <= tol)[fine].all())


def test_process_logits_scalars_and_defaults():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 999, generator=g)
    assert torch.equal(ops.process_logits(x.to(DEV)).cpu(), x)
    tokens = torch.randint(0, 999, (4, 20), generator=g)
    got = ops.process_logits(x.to(DEV), tokens=tokens.to(DEV), repetition_penalty=1.3, frequency_penalty=0.2)
    want, tol = _logits_oracle(x, tokens, [20] * 4, [0] * 4, [1.3] * 4, [0.0] * 4, [0.2] * 4, None, None)
    # 1.3 and 0.2 reach the kernel as fp32: three more roundings
    assert bool(((got.cpu().double() - want).abs() <= 2 * tol).all())


def test_process_logits_nonfinite():
    """What a mask forbids is -inf, whatever was there; infinities stay."""
    x = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, math.nan, -math.inf]])
    mask = torch.tensor([False, True, True, True, True, False])
    t = torch.tensor([[1, 2, 2]])
    got = ops.process_logits(x.to(DEV), tokens=t.to(DEV), repetition_penalty=2.0, presence_penalty=1.0, mask=mask.to(DEV)).cpu()[0]
    assert got[0] == -math.inf and got[1] == math.inf and got[2] == -math.inf and got[3] == 1.0
    assert math.isnan(got[4]) and got[5] == -math.inf
    none = ops.process_logits(x.to(DEV), mask=torch.zeros(1, dtype=torch.int32, device=DEV)).cpu()
    assert bool((none == -math.inf).all())


# ---------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------

def _pass(c, H, qkv, cos, sin, logits, tokens):
    q = ops.kv_cache_write(qkv, c.layer, c.step, H, cos, sin)
    o = ops.paged_attention(q, c.layer, c.step, H, c.hd**-0.5)
    n = c.step.max_len
    k, v = ops.kv_cache_read(c.layer, c.step.page_table[:1], torch.tensor([0, n], dtype=torch.int32, device=DEV)
                             if not torch.cuda.is_current_stream_capturing() else c.start, n, c.dtype)
    return q, o, k, v, ops.process_logits(logits, tokens=tokens, repetition_penalty=1.2, frequency_penalty=0.1)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 900), (1, 3)], [(150, 300), (7, 90)], [(400, 1200), (70, 90)]])
def test_two_graphs_and_eager_calls_in_turn(seqs, e4m3):
    """Two captured passes and eager ones between their replays, on contents
    that change: every replay gives what the eager call gives."""
    H, KV, hd = 8, 2, 64
    cases = [Case(seqs, KV, hd, 32, BF16, e4m3, seed=s) for s in (1, 2)]
    inputs = []
    for c in cases:
        c.start = torch.tensor([0, c.step.max_len], dtype=torch.int32, device=DEV)
        cos, sin = (t.to(DEV) for t in _tables(c.step.max_len, hd, BF16))
        inputs.append([torch.randn(c.rows, (H + 2 * KV) * hd, generator=c.g).to(BF16).to(DEV), cos, sin,
                       torch.randn(2, 5000, generator=c.g).to(DEV), torch.randint(0, 5000, (2, 99), generator=c.g).to(DEV)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for c, x in zip(cases, inputs):
            _pass(c, H, *x)
    torch.cuda.current_stream().wait_stream(side)
    for c, x in zip(cases, inputs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_pass(c, H, *x))
        graphs.append(graph)
    for turn in range(4):
        for c, x in zip(cases, inputs):
            x[0].copy_(torch.randn(x[0].shape, generator=c.g))
            x[3].copy_(torch.randn(x[3].shape, generator=c.g))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for c, x, o in zip(cases, inputs, got):
            for a, b in zip(o, _pass(c, H, *x)):
                assert torch.equal(a, b), turn


@pytest.mark.parametrize("most", [0, MUCH])
def test_calls_on_another_stream(most):
    c = Case([(1, 700), (30, 64)], 2, 64, 32, BF16, most=most)
    q = torch.randn(c.rows, 4 * 64, generator=c.g).to(BF16).to(DEV)
    want = ops.paged_attention(q, c.layer, c.step, 4, 0.125)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.paged_attention(q, c.layer, c.step, 4, 0.125) for _ in range(3)]
    also = [ops.paged_attention(q, c.layer, c.step, 4, 0.125) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got + also)


def test_unaligned_rows():
    """Rows at odd strides and offsets are taken as they are."""
    c = Case([(3, 50)], 2, 32, 16, BF16)
    flat = torch.randn(3 * 131 + 1, generator=c.g).to(BF16).to(DEV)
    q = flat[1:].view(3, 131)[:, :128]
    assert torch.equal(ops.paged_attention(q, c.layer, c.step, 4, 0.2),
                       ops.paged_attention(q.contiguous(), c.layer, c.step, 4, 0.2))
    cos, sin = (t.to(DEV) for t in _tables(50, 32, BF16))
    wide = torch.randn(3, 263, generator=c.g).to(BF16).to(DEV)
    a = ops.kv_cache_write(wide[:, 1:257], c.layer, c.step, 4, cos, sin)
    assert torch.equal(a, ops.kv_cache_write(wide[:, 1:257].contiguous(), c.layer, c.step, 4, cos, sin))


@pytest.mark.parametrize("seqs", [[(1, 5), (1, 900)], [(90, 300), (3, 3)], [(1, 4000)]])
@pytest.mark.parametrize("most", [0, MUCH])
def test_output_in_place_of_the_queries(seqs, most):
    c = Case(seqs, 2, 64, 16, BF16, most=most)
    wide = torch.randn(c.rows, 4 * 256, generator=c.g).to(BF16).to(DEV)
    want = ops.paged_attention(wide[:, 256:512], c.layer, c.step, 4, 0.2)
    rest = wide.clone()
    assert ops.paged_attention(wide[:, 256:512], c.layer, c.step, 4, 0.2, out=wide[:, 256:512]).data_ptr() == wide[:, 256:].data_ptr()
    rest[:, 256:512] = want
    assert torch.equal(wide, rest)


def test_refusals():
    c = Case([(2, 20)], 2, 64, 16, BF16)
    q = torch.zeros(2, 256, dtype=BF16, device=DEV)
    qkv = torch.zeros(2, 8 * 64, dtype=BF16, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(20, 64, BF16))
    att = lambda q=q, layer=c.layer, step=c.step, H=4: ops.paged_attention(q, layer, step, H, 0.1)  # noqa: E731
    wr = lambda x=qkv, layer=c.layer, step=c.step, H=4, cs=cos, sn=sin: ops.kv_cache_write(x, layer, step, H, cs, sn)  # noqa: E731
    L, S = c.layer, c.step
    e = torch.zeros(L.k.shape[:3], dtype=torch.int8, device=DEV)
    for call, err in [
        (lambda: att(q=q.float()), TypeError), (lambda: att(q=q.cpu()), RuntimeError), (lambda: att(H=3), ValueError),
        (lambda: att(q=q[:, :200]), ValueError), (lambda: att(layer=L._replace(v=L.v[:1])), ValueError),
        (lambda: att(layer=L._replace(k_exp=e, v_exp=e)), TypeError),
        (lambda: att(layer=LayerCache(L.k.to(E4M3), L.v.to(E4M3))), ValueError),
        (lambda: att(layer=LayerCache(L.k.transpose(1, 2), L.v.transpose(1, 2))), ValueError),
        (lambda: att(step=S._replace(kv_len=S.kv_len.long())), ValueError),
        (lambda: att(step=S._replace(row_start=S.row_start[:1])), ValueError),
        (lambda: att(step=S._replace(page_table=S.page_table[0])), ValueError),
        (lambda: att(layer=LayerCache(L.k[:, :, :8].contiguous(), L.v[:, :, :8].contiguous())), RuntimeError),
        (lambda: att(q=q[:, :192], layer=LayerCache(L.k[..., :48].contiguous(), L.v[..., :48].contiguous())), RuntimeError),
        (lambda: wr(x=qkv[:, :-1]), ValueError), (lambda: wr(cs=cos.float()), ValueError),
        (lambda: wr(cs=cos[:10], sn=sin[:10]), ValueError), (lambda: wr(x=qkv.half()), TypeError),
        (lambda: ops.kv_cache_read(L, S.page_table, S.row_start, 2, F32), TypeError),
        (lambda: ops.kv_cache_read(L, S.page_table, S.kv_len, 2, BF16), ValueError),
        (lambda: ops.process_logits(q[0]), ValueError), (lambda: ops.process_logits(q.t()), ValueError),
        (lambda: ops.process_logits(q, tokens=torch.zeros(2, 3, device=DEV)), ValueError),
        (lambda: ops.process_logits(q, lengths=S.kv_len), ValueError),
        (lambda: ops.process_logits(q, repetition_penalty=0.0), ValueError),
        (lambda: ops.process_logits(q, repetition_penalty=1e-60), ValueError),
        (lambda: ops.process_logits(q, frequency_penalty=1e60), ValueError),
        (lambda: att(step=S._replace(rows=3)), ValueError), (lambda: wr(step=S._replace(rows=-1)), ValueError),
        (lambda: att(step=S._replace(max_new=1)), ValueError), (lambda: wr(step=S._replace(max_len=-1)), ValueError),
        (lambda: ops.process_logits(q, presence_penalty=math.nan), ValueError),
        (lambda: ops.process_logits(q, bias=torch.zeros(255, device=DEV)), ValueError),
        (lambda: ops.process_logits(q, mask=torch.zeros(2, 7, dtype=torch.int32, device=DEV)), ValueError),
        (lambda: ops.process_logits(q, mask=torch.zeros(256, device=DEV)), ValueError),
    ]:
        with pytest.raises(err):
            call()
    empty = S._replace(rows=0)
    assert att(q=q[:0], step=empty).shape == (0, 256) and wr(x=qkv[:0], step=empty).shape == (0, 256)


# ---------------------------------------------------------------------------
# the cache object and the model
# ---------------------------------------------------------------------------

def test_cache_pages_come_and_go():
    cache = KVCache(2, 2, 32, batch=3, n_pages=5, page_size=16, device=DEV)
    s = cache.step([20, 0, 16])
    assert (s.rows, s.max_new, s.max_len) == (36, 20, 20) and s.row_start.tolist() == [0, 20, 20, 36]
    assert s.kv_len.tolist() == [20, 0, 16] and sorted(p for row in s.page_table.tolist() for p in row if p >= 0) == [0, 1, 2]
    with pytest.raises(RuntimeError):
        cache.step([0, 40, 0])
    assert cache.lengths == [20, 0, 16]
    cache.free(0)
    s = cache.step([0, 40, 1])
    used = [p for row in s.page_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 5 and cache.lengths == [0, 40, 17]
    for bad in ([1, 1], [1, -1, 0]):
        with pytest.raises(ValueError):
            cache.step(bad)
    for kw in (dict(head_dim=48), dict(page_size=24), dict(n_pages=0), dict(storage=torch.int8), dict(dtype=torch.int32)):
        args = dict(n_layers=1, n_kv_heads=1, head_dim=32, batch=1, n_pages=1, device=DEV) | kw
        with pytest.raises((ValueError, TypeError)):
            KVCache(**args)


def _model(dtype, **kw):
    from model import LlamaForCausalLM, ModelConfig

    cfg = ModelConfig(**(dict(name="t", vocab_size=500, max_seq_len=48, dim=256, n_layers=2, n_heads=4, n_kv_heads=2,
                              ffn_dim=384, initializer_range=0.1) | kw))
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg).to(device=DEV, dtype=dtype).eval()


@pytest.mark.parametrize("dtype,storage,most", [
    # float32: sums of at most 512 terms, two layers of ten operations; the
    # others: twenty roundings to the type of values that add up to the
    # logits, at worst all one way
    (F32, None, 1e-4), (BF16, None, 20 * 2.0**-8), (F16, None, 20 * 2.0**-11),
])
def test_cached_forward_is_the_forward(dtype, storage, most):
    """Prompts of different lengths, then chunks and single tokens, against
    the uncached forward of each text."""
    model = _model(dtype)
    g = torch.Generator().manual_seed(3)
    texts = [torch.randint(0, 500, (n,), generator=g).to(DEV) for n in (40, 25, 31)]
    cache = model.new_cache(3, 48, storage, page_size=16)
    done = [0, 0, 0]
    with torch.no_grad():
        for new in ([7, 1, 20], [1, 1, 1], [10, 0, 3], [1, 17, 1], [1, 1, 1]):
            step = cache.step(new)
            ids = torch.cat([t[d : d + n] for t, d, n in zip(texts, done, new)])
            got = model.forward_cached(ids, cache, step)
            done = [d + n for d, n in zip(done, new)]
            for b, n in enumerate(new):
                if n:
                    want = model(texts[b][None, : done[b]]).logits[0, -1].double()
                    assert float((got[b].double() - want).norm() / want.norm()) <= most, (new, b)
    k, v = cache.read(0, 1)
    assert k.shape == v.shape == (done[1], 2, 64) and k.dtype == dtype


def test_cached_forward_has_no_dropout_and_no_gradients():
    model = _model(F32, dropout=0.5)
    ids = torch.randint(0, 500, (9,), generator=torch.Generator().manual_seed(6)).to(DEV)
    want = model(ids[None]).logits[0, -1].detach()
    model.train()
    model.layers[0].mlp.eval()
    modes = [m.training for m in model.modules()]
    cache = model.new_cache(3, 16)
    got = model.forward_cached(ids, cache, cache.step([0, 9, 0]))  # no new tokens before and after
    assert [m.training for m in model.modules()] == modes and not got.requires_grad
    assert float((got[1] - want).norm() / want.norm()) <= 1e-4  # as in test_cached_forward_is_the_forward
    x = torch.randn(3, 256, device=DEV, requires_grad=True)
    assert not model.layers[1].forward_cached(x, cache.layers[1], cache.step([1, 1, 1])).requires_grad


def test_cached_forward_in_e4m3():
    """The first layer's keys and values, which no attention comes before, are
    the float32 cache's, each off by at most half a step: 2^-4 of it, or, where
    it is below 2^-6 of the head's unit 2^e, 2^-10 units, and 448 units hold
    the head's largest value with 2^e at most its 224th part."""
    model = _model(F32)
    ids = torch.randint(0, 500, (37,), generator=torch.Generator().manual_seed(4)).to(DEV)
    caches = [model.new_cache(1, 48, storage, page_size=16) for storage in (None, E4M3)]
    for cache in caches:
        for lo, hi in ((0, 30), (30, 31), (31, 37)):
            assert bool(torch.isfinite(model.forward_cached(ids[lo:hi], cache, cache.step([hi - lo]))).all())
    for full, small in zip(*(cache.read(0, 0) for cache in caches)):
        unit = full.abs().amax(-1, keepdim=True) / 224
        assert bool(((full - small).abs() <= torch.maximum(full.abs() * 2.0**-4, unit * 2.0**-10)).all())
        assert not torch.equal(full, small)


@pytest.mark.parametrize("new", [3, 12])
def test_generate_with_a_cache(new):
    """Greedy tokens of a float32 model with and without the cache, across the
    end of the window, and the adjustments against their own definition."""
    model = _model(F32)
    prompt = torch.randint(0, 500, (2, 42), generator=torch.Generator().manual_seed(5)).to(DEV)
    plain = model.generate(prompt, new, temperature=0.0)
    assert torch.equal(model.generate(prompt, new, temperature=0.0, use_cache=True), plain)
    # every token forbidden but one, which a bias cannot help
    mask = torch.zeros(500, dtype=torch.bool, device=DEV)
    mask[123] = True
    only = model.generate(prompt, new, temperature=0.0, use_cache=True, token_mask=mask,
                          logit_bias=torch.randn(500, device=DEV))
    assert bool((only[:, 42:] == 123).all())
    # a mask that moves: token t at step t
    def at(seq):
        m = torch.zeros(2, 500, dtype=torch.bool, device=DEV)
        m[:, seq.shape[1]] = True
        return m
    moving = model.generate(prompt, new, temperature=0.0, token_mask=at)
    assert moving[0, 42:].tolist() == list(range(42, 42 + new))
    # a presence penalty larger than any logit: no token twice
    once = model.generate(prompt, new, temperature=0.0, use_cache=True, presence_penalty=1e6)
    for b in range(2):
        assert len(set(once[b, 42:].tolist())) == new
    assert model.generate(prompt, 2, temperature=0.0, use_cache=True, cache_dtype=E4M3).shape == (2, 44)
    assert torch.equal(model.generate(prompt, 0, use_cache=True), prompt)
    # a row that may take nothing
    nothing = torch.ones(2, 500, dtype=torch.bool, device=DEV)
    nothing[1] = False
    for how in (dict(temperature=0.0), dict(temperature=1.0), dict(temperature=1.0, top_k=3, use_cache=True)):
        with pytest.raises(ValueError, match="token 42"):
            model.generate(prompt, new, token_mask=nothing, **how)
    torch.manual_seed(9)
    a = model.generate(prompt, 3, temperature=0.8, top_k=5, use_cache=True)
    torch.manual_seed(9)
    assert torch.equal(a, model.generate(prompt, 3, temperature=0.8, top_k=5, use_cache=True))


def test_model_refusals():
    model = _model(F32, dim=96, n_heads=2, n_kv_heads=1)  # head dim 48
    with pytest.raises(ValueError):
        model.generate(torch.zeros(1, 4, dtype=torch.int64, device=DEV), 2, use_cache=True)
    model = _model(F32)
    cache = model.new_cache(1, 16)
    step = cache.step([4])
    with pytest.raises(ValueError):
        model.forward_cached(torch.zeros(3, dtype=torch.int64, device=DEV), cache, step)
    with pytest.raises(ValueError):
        model.forward_cached(torch.zeros(0, dtype=torch.int64, device=DEV), cache, cache.step([0]))
    other = _model(F32, n_layers=3).new_cache(1, 16)
    with pytest.raises(ValueError):
        model.forward_cached(torch.zeros(4, dtype=torch.int64, device=DEV), other, other.step([4]))
    with pytest.raises(ValueError):
        model.generate(torch.zeros(1, 4, dtype=torch.int64, device=DEV), 2, cache_dtype=E4M3)
    model._zero3_executor = object()
    with pytest.raises(RuntimeError):
        model.forward_cached(torch.zeros(4, dtype=torch.int64, device=DEV), cache, step)
