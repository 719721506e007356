"""Generation from a paged key/value cache: what random steps do not reach.

Tolerances count roundings, as in test_gpu_generation.
"""
from __future__ import annotations

import math

import pytest
import torch

from lzhip import ops
from lzhip.cache import CacheStep, LayerCache
from test_gpu_generation import BF16, DEV, E4M3, F16, F32, MUCH, U32, Case, _model, _u

pytestmark = pytest.mark.gpu
DEV0 = torch.device("cuda", 0)


def _attention(c, q, H, scale, weights, terms):
    """(o, bound) in float64: the output rounded to the type once, each weight
    off by `weights` of it, sums of `terms` terms a key in fp32."""
    q = q.double().view(-1, H, c.hd)
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b, (n, l) in enumerate(c.seqs):
        k, v = c.tokens(0, b), c.tokens(1, b)
        for i in range(n):
            seen, r = l - n + i + 1, c.starts[b] + i
            for h in range(H):
                g = h // (H // c.KV)
                p = torch.softmax(k[:seen, g] @ q[r, h] * scale, 0)
                size = float((k[:seen, g].abs() @ q[r, h].abs()).max()) * scale
                o[r, h] = p @ v[:seen, g]
                # a score is hd products and adds and a few units of the
                # exponent's argument
                fp32 = (2 * (c.hd + 4) * size + 8 + terms * seen) * U32
                tol[r, h] = _u(c.dtype) * o[r, h].abs() + (weights + fp32) * (p @ v[:seen, g].abs())
    return o.view(-1, H * c.hd), tol.view(-1, H * c.hd)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("seqs,H,KV,hd,page", [
    ([(1, 900), (1, 40)], 8, 4, 64, 32),  # single tokens, one in parts
    ([(1, 300)] * 3, 16, 8, 128, 16),
    ([(15, 700), (3, 3)], 10, 2, 32, 16),  # short chunks
    ([(40, 333)], 6, 2, 64, 64),
])
def test_weights_of_few_rows_keep_their_fp32_bits(seqs, H, KV, hd, page, dtype, e4m3):
    """Single tokens and short chunks: the only rounding to the type is the
    output's.  A weight enters the second product as two or three terms that
    add up to it (in fp16 to u^2 of it)."""
    c = Case(seqs, KV, hd, page, dtype, e4m3, seed=hd)
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, hd**-0.5).cpu().double()
    want, tol = _attention(c, q, H, hd**-0.5, weights=_u(F16) ** 2 if dtype == F16 else 0.0, terms=3)
    assert float(((got - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("seqs,H,KV,hd,page", [
    ([(150, 300), (70, 90)], 8, 2, 64, 32),
    ([(129, 129)], 4, 4, 128, 16),
    ([(200, 1000)], 5, 1, 32, 64),
])
def test_weights_of_tiles_keep_sixteen_bits(seqs, H, KV, hd, page, dtype, e4m3):
    """Chunks in 128-row tiles: a weight 2^e (1 <= x < 2) is two terms, x cut to
    the type (the rest is below 2 u) and the rest rounded (off by u of what is
    below 2 u, so by u^2 2^e: half a step of the rest's)."""
    c = Case(seqs, KV, hd, page, dtype, e4m3, seed=hd, most=MUCH)
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, hd**-0.5).cpu().double()
    want, tol = _attention(c, q, H, hd**-0.5, weights=_u(dtype) ** 2, terms=2)
    assert float(((got - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("most", [0, MUCH])
def test_starts_past_the_last_row(most):
    """Sequences whose rows the tables put far behind the call's: nothing is
    computed for them, the others are as ever."""
    c = Case([(80, 100), (5, 30), (9, 9)], 2, 64, 16, BF16, most=most)
    q = torch.randn(c.rows, 16 * 64, generator=c.g).to(BF16).to(DEV)
    want = ops.paged_attention(q, c.layer, c.step, 16, 0.125)
    start = torch.tensor([0, 80, 10**9, 2 * 10**9], dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, c.layer, c.step._replace(row_start=start), 16, 0.125, out=out)
    assert torch.equal(out[:80], want[:80])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,length,most", [(1, 40, 0), (1, 3000, 0), (20, 90, 0), (20, 2500, 0), (90, 300, MUCH), (130, 3000, MUCH)])
def test_scores_of_minus_infinity(dtype, n, length, most):
    """A row that sees keys whose scores are all -inf is NaN, as a softmax is;
    one that sees others too gives them all the weight; one that sees no key
    (or none with a page) is zeros."""
    H, KV, hd, page = 4, 2, 64, 16
    seqs = [(n, length), (n, length), (n, n + 20), (n, length)]
    c = Case(seqs, KV, hd, page, dtype, seed=length, most=most)
    q = torch.randn(c.rows, H * hd, generator=c.g)
    q.view(-1, H, hd)[..., 5] = 1.0 + q.view(-1, H, hd)[..., 5].abs()
    q = q.to(dtype)
    k = c.cpu[0]
    low = [length, length - n // 2 - 1, 0, length]  # of each sequence, the first tokens whose keys overflowed (kv head 1)
    for b, m in enumerate(low):
        p = torch.arange(m)
        k[c.table[b, p // page].long(), 1, p % page, 5] = -float("inf")
    c.layer.k.copy_(k)
    table = c.table.clone()
    table[2] = -1  # no page at all
    table[3, : (length - n) // page] = 10**6  # pages of the last tokens alone
    step = c.step._replace(page_table=table.to(DEV))
    got = ops.paged_attention(q.to(DEV), c.layer, step, H, 0.125).cpu().view(-1, H, hd)
    own = got[: c.starts[2]].view(2, n, H, hd)
    assert bool(torch.isfinite(own[:, :, :2]).all())
    assert bool(torch.isnan(own[0, :, 2:]).all())
    assert bool((got[c.starts[2] : c.starts[3]] == 0).all())
    assert bool(torch.isnan(got[c.starts[3] :][:, 2:]).all()) and bool(torch.isfinite(got[c.starts[3] :][:, :2]).all())
    kk, vv = c.tokens(0, 1)[:, 1], c.tokens(1, 1)[:, 1]
    for i in range(n):
        seen = length - n + i + 1
        for h in (2, 3):
            x = q[c.starts[1] + i].view(H, hd)[h].double()
            if seen <= low[1]:
                assert bool(torch.isnan(own[1, i, h]).all()), i
                continue
            keys, vals = kk[low[1] : seen], vv[low[1] : seen]
            p = torch.softmax(keys @ x * 0.125, 0)
            size = float((keys.abs() @ x.abs()).max()) * 0.125
            tol = _u(dtype) * (p @ vals).abs() + (_u(dtype) ** 2 + (2 * (hd + 4) * size + 8 + 3 * len(p)) * U32) * (p @ vals.abs())
            assert bool(((own[1, i, h].double() - p @ vals).abs() <= tol).all()), (i, h)


def test_no_key_at_all_beside_scores_of_minus_infinity():
    """Rows before a sequence's first token are zeros, those after it NaN."""
    c = Case([(6, 6)], 1, 32, 16, F32)
    c.layer.k[..., 0] = -float("inf")
    q = torch.ones(6, 32, device=DEV)
    step = c.step._replace(kv_len=torch.tensor([2], dtype=torch.int32, device=DEV))
    got = ops.paged_attention(q, c.layer, step, 1, 0.5)
    assert bool((got[:4] == 0).all()) and bool(torch.isnan(got[4:]).all())


@pytest.mark.parametrize("recompute", [True, False])
def test_a_sharded_model_generates_from_a_cache_where_its_parameters_are_gathered(recompute):
    """As the refusal of a ZeRO-3 model says: within summon_full_params, and
    at all times where the engine keeps the parameters."""
    from zero import ZeROStage3Optimizer

    ids = torch.randint(0, 500, (2, 7), generator=torch.Generator().manual_seed(1)).to(DEV)
    want = _model(BF16).generate(ids, 3, temperature=0.0, use_cache=True)
    model = _model(BF16)
    engine = ZeROStage3Optimizer(model=model, lr=1e-3, recompute=recompute)
    if recompute:
        with pytest.raises(RuntimeError, match="summon_full_params"):
            model.generate(ids, 3, temperature=0.0, use_cache=True)
    with engine.summon_full_params():
        assert torch.equal(model.generate(ids, 3, temperature=0.0, use_cache=True), want)
        assert model.generate(ids, 3, temperature=0.0).shape == (2, 10)
        if recompute:  # a forward of its own hands each module's parameters back
            with pytest.raises(RuntimeError, match="summon_full_params"):
                model.generate(ids, 3, temperature=0.0, use_cache=True)
    if not recompute:
        assert torch.equal(model.generate(ids, 3, temperature=0.0, use_cache=True), want)


def test_a_captured_model_step_outlives_longer_eager_ones():
    """A decoded token captured once for all layers: eager calls of longer
    sequences, which need longer rotary tables, between its replays."""
    model = _model(BF16, max_seq_len=600)
    g = torch.Generator().manual_seed(3)
    lens, most = [5, 40], 200
    prompt = torch.randint(0, 500, (sum(lens),), generator=g).to(DEV)
    caches = [model.new_cache(2, 256) for _ in range(2)]
    for cache in caches:
        model.forward_cached(prompt, cache, cache.step(lens))
    table = caches[0].step([most - 40] * 2).page_table.clone()  # pages for what comes
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    step = CacheStep(torch.arange(3, dtype=torch.int32, device=DEV), kv, table, 2, 1, most)
    ids = torch.zeros(2, dtype=torch.int64, device=DEV)
    kv += 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.forward_cached(ids, caches[0], step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.forward_cached(ids, caches[0], step)
    kv -= 1
    for turn in range(5):
        other = model.new_cache(1, 300 + 256 * turn)
        model.forward_cached(torch.randint(0, 500, (260 + 256 * turn,), generator=g).to(DEV), other,
                             other.step([260 + 256 * turn]))
        junk = [torch.full((256 * 64,), 3.0, dtype=BF16, device=DEV) for _ in range(40)]
        new = torch.randint(0, 500, (2,), generator=g).to(DEV)
        ids.copy_(new)
        kv += 1
        graph.replay()
        torch.cuda.synchronize()
        s = caches[1].step([1, 1])._replace(max_len=most)  # split alike
        assert torch.equal(out, model.forward_cached(new, caches[1], s)), turn
        del junk


def test_process_logits_lengths_past_32_bits():
    """int64 lengths larger than any text: all of it counts; prompts as long:
    nothing is the answer."""
    g = torch.Generator().manual_seed(4)
    x, tokens = torch.randn(3, 50, generator=g).to(DEV), torch.randint(0, 50, (3, 9), generator=g).to(DEV)
    far = torch.tensor([2**63 - 1, 2**32, 2**31], device=DEV)
    how = dict(tokens=tokens, repetition_penalty=1.5, presence_penalty=2.0, frequency_penalty=0.5)
    got = ops.process_logits(x, lengths=far, **how)
    assert torch.equal(got, ops.process_logits(x, **how)) and not torch.equal(got, x)
    got = ops.process_logits(x, prompt_lengths=far, **how)
    assert torch.equal(got, ops.process_logits(x, tokens=tokens, repetition_penalty=1.5))
    none = ops.process_logits(x, lengths=torch.tensor([-(2**63), -(2**32) + 5, -1], device=DEV), **how)
    assert torch.equal(none, x)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("seqs,bound,most", [
    ([(200, 300), (3, 50), (1, 9)], 128, MUCH),           # tiles, in the order of their keys
    ([(300, 2000), (3, 50), (260, 700)], 250, MUCH),
    ([(150, 150)] + [(b % 7, 20 + b) for b in range(70)], 130, MUCH),  # tiles, sequence after sequence
    ([(60, 80), (3, 50)], 40, 0),                         # waves
    ([(20, 3000), (1, 50)], 12, 0),                       # in parts
])
def test_rows_past_max_new_are_left(seqs, bound, most, e4m3):
    """Tables that grew past a step's bound: a sequence's first max_new rows
    are computed, the others left as they are."""
    c = Case(seqs, 2, 64, 16, BF16, e4m3, seed=bound, most=most)
    c.step = c.step._replace(max_new=bound)
    q = torch.randn(c.rows, 2 * 64, generator=c.g).to(BF16)
    out = torch.full_like(q, 7.0).to(DEV)
    ops.paged_attention(q.to(DEV), c.layer, c.step, 2, 0.125, out=out)
    got = out.cpu().double()
    want, tol = c.attention(q, 2, 0.125)
    for b, (n, _) in enumerate(seqs):
        lo, hi = c.starts[b], c.starts[b + 1]
        mid = min(lo + bound, hi)
        assert bool(((got - want).abs() <= tol)[lo:mid].all()), b
        assert bool((got[mid:hi] == 7).all()), b


@pytest.mark.parametrize("most", [0, MUCH])
def test_rows_between_the_last_sequence_and_the_step(most):
    """Tables that cover fewer rows than the step was made for: the caller's
    rows of no sequence stay, and new outputs are zeros from step.rows on."""
    c = Case([(70, 90), (1, 5), (9, 20)], 2, 64, 16, BF16, most=most)
    start = torch.tensor([0, 70, 71, 71], dtype=torch.int32, device=DEV)
    step = c.step._replace(row_start=start)
    wide = torch.randn(c.rows + 4, 8 * 64, generator=c.g).to(BF16).to(DEV)
    cos, sin = (torch.randn(c.step.max_len if not most else 90, 64, generator=c.g).to(BF16).to(DEV) for _ in range(2))
    out = torch.full((c.rows + 4, 256), 7.0, dtype=BF16, device=DEV)
    q = ops.kv_cache_write(wide, c.layer, step._replace(max_len=90), 4, cos, sin, out=out)
    assert q.data_ptr() == out.data_ptr() and bool((out[71:] == 7).all()) and not bool((out[:71] == 7).any())
    o = ops.paged_attention(q, c.layer, step, 4, 0.125, out=torch.full_like(out, 7.0))
    assert bool((o[71:] == 7).all()) and bool(torch.isfinite(o[:71]).all())
    fresh = ops.kv_cache_write(wide, c.layer, step._replace(max_len=90), 4, cos, sin)
    assert torch.equal(fresh[:71], q[:71]) and bool((fresh[c.rows :] == 0).all())
    fresh = ops.paged_attention(q, c.layer, step, 4, 0.125)
    assert torch.equal(fresh[:71], o[:71]) and bool((fresh[c.rows :] == 0).all())


def test_positions_past_the_page_table():
    """A sequence longer than its row of pages: its tokens there are not
    written and not seen, their queries are rotated and see what is there."""
    c = Case([(3, 64)], 1, 32, 16, F32)
    step = c.step._replace(kv_len=torch.tensor([66], dtype=torch.int32, device=DEV), max_len=66)
    cos, sin = (torch.randn(66, 32, generator=c.g) for _ in range(2))
    qkv = torch.randn(3, 3 * 32, generator=c.g)
    before = c.layer.k.clone()
    q = ops.kv_cache_write(qkv.to(DEV), c.layer, step, 1, cos.to(DEV), sin.to(DEV))
    pos = torch.tensor([63, 64, 65])
    x = qkv[:, :64].view(3, 2, 32)
    y = x * cos[pos][:, None] + torch.cat([-x[..., 16:], x[..., :16]], -1) * sin[pos][:, None]
    assert torch.equal(q.cpu(), y[:, 0])
    k = before.cpu()
    k[c.table[0, 3], 0, 15] = y[0, 1]
    assert torch.equal(c.layer.k.cpu(), k)
    got = ops.paged_attention(q, c.layer, step, 1, 0.25).cpu()
    kk = k[c.table[0].long(), 0].reshape(64, 32).double()
    vv = c.layer.v.cpu()[c.table[0].long(), 0].reshape(64, 32).double()
    for i in range(3):
        p = torch.softmax(kk @ y[i, 0].double() * 0.25, 0)
        size = float((kk.abs() @ y[i, 0].double().abs()).max()) * 0.25
        tol = U32 * (p @ vv).abs() + (2 * 36 * size + 8 + 64) * U32 * (p @ vv.abs())
        assert bool(((got[i].double() - p @ vv).abs() <= tol).all()), i


def test_outputs_over_other_inputs_are_refused():
    """out may be q itself, or the q columns of qkv, or columns beside them;
    what would be written over values still to be read is refused."""
    c = Case([(5, 50)], 2, 32, 16, BF16)
    cos, sin = (torch.randn(50, 32, generator=c.g).to(BF16).to(DEV) for _ in range(2))
    first = torch.randn(12, 640, generator=c.g).to(BF16).to(DEV)
    wide = first.clone()
    q, qkv = wide[:5, :128], wide[:5, :256]

    def attend(out):
        return ops.paged_attention(q, c.layer, c.step, 4, 0.2, out=out)

    def write(out):
        return ops.kv_cache_write(qkv, c.layer, c.step, 4, cos, sin, out=out)

    want = write(None), attend(None)
    for out in (wide[:5, 8:136], wide[1:6, :128], wide.view(-1)[520 : 520 + 5 * 640].view(5, 640)[:, :128],
                wide.view(-1)[: 5 * 128].view(5, 128)):
        for call in (attend, write):
            with pytest.raises(ValueError, match="overlap"):
                call(out)
    with pytest.raises(ValueError, match="overlap"):  # the keys' columns
        write(wide[:5, 128:256])
    assert torch.equal(wide, first)
    for out in (wide[:5, 256:384], wide[:5, 512:], wide[5:10, 64:192], wide[:5, :128]):
        for call, result in ((write, want[0]), (attend, want[1])):
            assert torch.equal(call(out), result)
            wide.copy_(first)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 70])
def test_chunks_on_pages_past_two_to_the_31_elements(new, e4m3):
    """Page ids whose element offsets need 64 bits, in the 128-row tiles and in
    8 bits."""
    pages, page, hd = 2**15 + 40, 1024, 64
    store = E4M3 if e4m3 else BF16
    k, v = (torch.empty(pages, 1, page, hd, dtype=store, device=DEV) for _ in range(2))
    e = [torch.zeros(pages, 1, page, dtype=torch.int8, device=DEV) for _ in range(2)] if e4m3 else [None, None]
    far = [pages - 1, 2**15 - 1, 2**15 + 1]
    g = torch.Generator().manual_seed(8)
    for p in far:
        for t in (k, v):
            t[p] = torch.randn(1, page, hd, generator=g).to(DEV).to(store)
    length = 2 * page + 100
    step = CacheStep(*(torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, new], [length], [far])), new, new, MUCH)
    q = torch.randn(new, 2 * hd, generator=g).to(BF16)
    got = ops.paged_attention(q.to(DEV), LayerCache(k, v, *e), step, 2, 0.125).cpu().double()
    kk, vv = (torch.cat([t[p, 0] for p in far])[:length].cpu().double() for t in (k, v))
    for i in range(new):
        for h in range(2):
            seen, x = length - new + i + 1, q[i, h * hd : (h + 1) * hd].double()
            p = torch.softmax(kk[:seen] @ x * 0.125, 0)
            size = float((kk[:seen].abs() @ x.abs()).max()) * 0.125
            want, a = p @ vv[:seen], p @ vv[:seen].abs()
            tol = _u(BF16) * want.abs() + (_u(BF16) ** 2 + (2 * (hd + 4) * size + 8 + 3 * seen) * U32) * a
            assert bool(((got[i, h * hd : (h + 1) * hd] - want).abs() <= tol).all()), (i, h)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,length,most", [(1, 1, 0), (1, 40, 0), (1, 3000, 0), (20, 90, 0), (20, 2500, 0), (90, 300, MUCH),
                                           (130, 3000, MUCH)])
def test_infinities_that_rows_see(dtype, n, length, most):
    """An infinite value of a token that every row sees: the weighted sum's, of
    its sign, and NaN where both signs meet; the other columns as ever."""
    H, KV, hd, page = 4, 2, 64, 16
    c = Case([(n, length), (1, 3)], KV, hd, page, dtype, seed=length, most=most)
    q = (torch.randn(c.rows, H * hd, generator=c.g) * 0.1).to(dtype)
    first = 0 if length == n else length - n  # the last token that all rows see
    for tok, col, sign in ((0, 5, 1), (first, 6, -1), (first // 2, 7, 1), (0, 9, 1), (first, 9, -1), (first // 3, 20, 1)):
        if length == 1 and col == 9 and sign < 0:
            continue
        c.cpu[1][c.table[0, tok // page], :, tok % page, col] = sign * math.inf
    c.layer.v.copy_(c.cpu[1])
    got = ops.paged_attention(q.to(DEV), c.layer, c.step, H, 0.125).cpu().double()
    want, tol = c.attention(q, H, 0.125)
    assert bool(torch.isposinf(want.view(-1, H, hd)[:n, :, 5]).all())
    assert torch.equal(got.nan_to_num(nan=7e30, posinf=8e30, neginf=-8e30)[~torch.isfinite(want)],
                       want.nan_to_num(nan=7e30, posinf=8e30, neginf=-8e30)[~torch.isfinite(want)])
    fine = torch.isfinite(want)
    assert bool(((got - want).abs() <= tol)[fine].all())


def test_two_threads_generate_at_once():
    """Cached steps of one model in training mode, with dropout, from two
    threads on streams of their own: the bits of the same steps alone, and the
    modes as they were."""
    import threading

    model = _model(BF16, dropout=0.5).train()
    modes = [m.training for m in model.modules()]
    g = torch.Generator().manual_seed(2)
    texts = [torch.randint(0, 500, (2, 30), generator=g).to(DEV) for _ in range(2)]

    def steps(text, out):
        cache = model.new_cache(2, 48)
        out.append(model.forward_cached(text[:, :20].reshape(-1), cache, cache.step([20, 20])))
        for t in range(20, 30):
            out.append(model.forward_cached(text[:, t].contiguous(), cache, cache.step([1, 1])))

    want = [[], []]
    for text, out in zip(texts, want):
        steps(text, out)
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream() for _ in range(2)]

    def run(i):
        with torch.cuda.stream(streams[i]):
            steps(texts[i], got[i])

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert [m.training for m in model.modules()] == modes
    for a, b in zip(want, got):
        assert len(a) == len(b) == 11 and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("grow", [False, True])
def test_rotary_tables_on_another_stream_than_they_were_built_on(grow):
    """Tables that one stream has still to build, used by another; and old
    ones, which another stream has still to read, replaced by longer ones."""
    import copy

    from model.llama import RotaryEmbedding

    def rotary():
        return RotaryEmbedding(64, 10_000.0).to(DEV)

    want = [t.clone() for t in rotary().tables(100, DEV0, F32)]
    rope, side = rotary(), torch.cuda.Stream()
    if grow:
        rope.tables(100, DEV0, F32)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got = [t.clone() for t in rope.tables(100, DEV0, F32)]
        rope.tables(5000, DEV0, F32)  # the old ones are free for what comes
        junk = [torch.full((100, 64), 9.0, device=DEV) for _ in range(64)]
    else:
        junk = [torch.full((100, 64), 9.0, device=DEV) for _ in range(64)]
        del junk
        torch.cuda._sleep(20_000_000)
        rope.tables(100, DEV0, F32)
        with torch.cuda.stream(side):
            got = [t.clone() for t in rope.tables(100, DEV0, F32)]
            assert all(torch.equal(a, b) for a, b in zip(copy.deepcopy(rope).tables(100, DEV0, F32), got))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
