"""The model's side of drafted tokens: cached passes over trees, the cache whose
tables are on the device, and generation with a draft model."""
from __future__ import annotations

import math

import pytest
import torch

from lzhip import ops
from lzhip.cache import DraftCache
from test_gpu_generation import BF16, DEV, E4M3, F16, F32, _model

pytestmark = pytest.mark.gpu


def _cache(model, batch, max_len, page=16, pages=None, **kw):
    c = model.cfg
    return DraftCache(c.n_layers, c.n_kv_heads, c.head_dim, batch=batch, n_pages=pages or batch * -(-max_len // page),
                      page_size=page, dtype=model.tok_embeddings.weight.dtype, device=DEV, max_len=max_len, **kw)


def _ids(*shape, seed=1, vocab=500):
    return torch.randint(0, vocab, shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("dtype,most", [
    # as the cached forward's: float32 sums, or twenty roundings to the type
    (F32, 1e-4), (BF16, 20 * 2.0**-8), (F16, 20 * 2.0**-11),
])
def test_a_tree_of_tokens_is_its_branches(dtype, most):
    """The logits of every node are the uncached forward's of its branch, and
    after keep() the text goes on as if the kept branch had been written."""
    model = _model(dtype)
    texts = [_ids(n, seed=n) for n in (20, 7, 13)]
    cache = _cache(model, 3, 48)
    model.forward_cached(torch.cat(texts), cache, cache.step([20, 7, 13]), rows="none")
    parents = [[-1, 0, 0, 1, 1, 2, 4], [-1, 0, 1, 2, 3, 4, 5], [-1, 0, 0, 0, 0, 3, 3]]
    drafted = _ids(3, 7, seed=9)
    base = cache.tables.lengths.clone()
    step = cache.step([7] * 3, parents=torch.tensor(parents, dtype=torch.int32, device=DEV))
    got = model.forward_cached(drafted.view(-1), cache, step, rows="all").view(3, 7, -1)
    last = model.forward_cached(drafted.view(-1), cache, step)  # written and computed again
    assert torch.equal(last, got[:, -1])
    for b in range(3):
        for i in range(7):
            branch, at = [], i
            while at >= 0:
                branch.append(int(drafted[b, at]))
                at = parents[b][at]
            text = torch.cat([texts[b], torch.tensor(branch[::-1], device=DEV)])
            with torch.no_grad():
                want = model(text[None]).logits[0, -1].double()
            assert float((got[b, i].double() - want).norm() / want.norm()) <= most, (b, i)
    kept = [[0, 1, 4, 6], [0, -1, -1, -1], [0, 3, 6, -1]]
    counts = torch.tensor([4, 1, 3], dtype=torch.int32, device=DEV)
    cache.keep(step, torch.tensor(kept, dtype=torch.int32, device=DEV), counts)
    more = _ids(3, seed=4)
    got = model.forward_cached(more, cache, cache.step([1] * 3, keep=base + counts))
    for b, nodes in enumerate(kept):
        text = torch.cat([texts[b], drafted[b, [n for n in nodes if n >= 0]], more[b : b + 1]])
        with torch.no_grad():
            want = model(text[None]).logits[0, -1].double()
        assert float((got[b].double() - want).norm() / want.norm()) <= most


def test_the_cache_hands_out_and_takes_back():
    model = _model(F32)
    cache = _cache(model, 3, 40, pages=6)  # three pages of 16 a sequence would be nine
    step = cache.step([20, 33, 10])
    assert step.row_start.tolist() == [0, 20, 53, 63] and int(cache.tables.n_free) == 0
    model.forward_cached(_ids(63), cache, step, rows="none")
    k, v = cache.read(1, 1)
    assert k.shape == v.shape == (33, 2, 64)
    late = cache.step([0, 0, 10])  # needs a page, and there is none
    assert late.row_start.tolist() == [0, 0, 0, 0] and cache.tables.lengths.tolist() == [20, 33, 10]
    cache.free(1)
    assert cache.tables.lengths.tolist() == [20, 0, 10] and int(cache.tables.n_free) == 3
    assert cache.step([0, 0, 10]).row_start.tolist() == [0, 0, 0, 10]
    new = torch.tensor([1, 2, 0], dtype=torch.int32, device=DEV)
    assert cache.step(new, rows=3, max_new=2).kv_len.tolist() == [21, 2, 20]
    for bad in (lambda: cache.step([1, 1]), lambda: cache.step([1, -1, 0]), lambda: cache.step(new), lambda: cache.step(new, rows=-1, max_new=2),
                lambda: _cache(model, 1, 0, pages=1)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("draft_tokens", [1, 4, (3,), (2, 2, 1), (1, 1)])
@pytest.mark.parametrize("same", [False, True])
def test_greedy_tokens_are_the_models_own(draft_tokens, same):
    """Whatever is drafted; prompts that end at different places of the pages."""
    model = _model(F32, max_seq_len=96)
    draft = model if same else _model(F32, max_seq_len=96, dim=128, n_layers=1, n_heads=2, n_kv_heads=1)
    for t0, new in ((1, 20), (30, 31), (64, 5)):
        prompt = _ids(3, t0, seed=t0)
        want = model.generate(prompt, new, temperature=0.0, use_cache=True)
        assert torch.equal(model.generate(prompt, new, temperature=0.0, draft_model=draft, draft_tokens=draft_tokens), want)


@pytest.mark.parametrize("draft_tokens", [3, (2, 1)])
def test_sampled_tokens_follow_the_models_law(draft_tokens):
    """Of n texts with one prompt, token v begins n p_v: within five standard
    deviations, and the same for the pairs that begin so."""
    model = _model(F32, vocab_size=16, max_seq_len=24, initializer_range=0.4)
    torch.manual_seed(5)
    draft = _model(F32, vocab_size=16, max_seq_len=24, dim=128, n_layers=1, n_heads=2, n_kv_heads=1, initializer_range=0.6)
    n = 3000
    prompt = _ids(1, 6, seed=2, vocab=16).expand(n, 6).contiguous()
    torch.manual_seed(11)
    got = model.generate(prompt, 3, temperature=0.9, top_k=12, draft_model=draft, draft_tokens=draft_tokens)[:, 6:]

    def law(text):
        x = model(text).logits[:, -1].double() / 0.9
        kth = x.topk(12).values[:, -1:]
        return torch.softmax(x.masked_fill(x < kth, -math.inf), -1)

    with torch.no_grad():
        p = law(prompt[:1])[0]
        count = got[:, 0].bincount(minlength=16).double()
        assert bool(((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1e-9).all())
        texts = torch.cat([prompt[:16], torch.arange(16, device=DEV)[:, None]], 1)
        pair = (p[:, None] * law(texts)).view(-1)
        count = (got[:, 0] * 16 + got[:, 1]).bincount(minlength=256).double()
        # the smallest: a Poisson count of mean m is over m + 5 sqrt(m) + 8 less than once in 10^6
        assert bool(((count - n * pair).abs() <= 5 * (n * pair * (1 - pair)).sqrt() + 8 * (pair > 0)).all())
    assert bool((count[pair == 0] == 0).all())


def test_drafted_generation_of_other_types():
    for dtype, storage in ((BF16, None), (F16, E4M3), (BF16, E4M3)):
        model, draft = _model(dtype), _model(BF16, dim=128, n_layers=1, n_heads=2, n_kv_heads=1)
        prompt = _ids(2, 17)
        for how in (dict(temperature=0.0), dict(temperature=1.0), dict(temperature=0.7, top_k=4)):
            for tokens in (2, (2, 2)):
                out = model.generate(prompt, 9, draft_model=draft, draft_tokens=tokens, cache_dtype=storage, **how)
                assert out.shape == (2, 26) and torch.equal(out[:, :17], prompt)
                assert bool(((out >= 0) & (out < 500)).all())
    # top_k 1 leaves the arg-max alone
    model = _model(F32)
    want = model.generate(prompt, 9, temperature=0.0)
    assert torch.equal(model.generate(prompt, 9, temperature=1.0, top_k=1, draft_model=model, draft_tokens=3), want)
    assert torch.equal(model.generate(prompt, 0, draft_model=model), prompt)


def test_drafted_generation_is_refused():
    model = _model(F32)
    prompt = _ids(2, 17)
    other = _model(F32, vocab_size=300)
    short = _model(F32, max_seq_len=20)
    for kw in (dict(draft_model=other), dict(draft_model=short), dict(draft_model=model, draft_tokens=0),
               dict(draft_model=model, draft_tokens=()), dict(draft_model=model, draft_tokens=(2, 0)),
               dict(draft_model=model, draft_tokens=(501,)), dict(draft_model=model, repetition_penalty=1.1),
               dict(draft_model=model, token_mask=torch.ones(500, dtype=torch.bool, device=DEV))):
        with pytest.raises(ValueError):
            model.generate(prompt, 9, **kw)
    with pytest.raises(ValueError):
        model.generate(prompt, 40, draft_model=model)  # past the window
    with pytest.raises(ValueError):
        model.forward_cached(prompt[0], _cache(model, 1, 48), None, rows="some")
    bad = _model(F32)
    with torch.no_grad():
        bad.norm.weight.fill_(math.nan)
    with pytest.raises(ValueError, match="no token"):
        bad.generate(prompt, 3, temperature=1.0, draft_model=model)


def test_a_servers_loop_of_trees():
    """Steps whose lengths the host never sees: texts go on as the model writes
    them, right guesses or wrong, shared tree or one for each."""
    N, made = 6, 24
    model = _model(F32, max_seq_len=128)  # generate() moves its window where a text passes it
    prompts = [_ids(n, seed=20 + n) for n in (9, 17, 4)]
    want = [model.generate(p[None], made + 2 * N, temperature=0, use_cache=True)[0, len(p):] for p in prompts]
    right = torch.stack(want)
    cache = _cache(model, 3, 17 + made + 3 * N)
    model.forward_cached(torch.cat([p[:-1] for p in prompts]), cache, cache.step([len(p) - 1 for p in prompts]), rows="none")
    root = torch.stack([p[-1] for p in prompts])
    start = cached = cache.tables.lengths.clone()
    new = torch.full((3,), N, dtype=torch.int32, device=DEV)
    one = torch.tensor([-1, 0, 0, 2, 3, 2], dtype=torch.int32, device=DEV)
    each = torch.stack([one, torch.tensor([-1, 0, 1, 1, 2, 4], device=DEV), torch.tensor([-1, 0, 1, 2, 3, 4], device=DEV)]).int()
    texts, steps = [[], [], []], 0
    while min(len(t) for t in texts) < made:
        parents = each if steps % 2 else one
        depth = torch.zeros(3, N, dtype=torch.int64, device=DEV)
        for i in range(1, N):
            up = parents[:, i] if steps % 2 else parents[i].expand(3)
            depth[:, i] = depth.gather(1, up.long()[:, None])[:, 0] + 1
        done = (cached - start).long()[:, None]
        ids = right.gather(1, (done + depth - 1).clamp(0, right.shape[1] - 1))  # what follows, at each depth
        wrong = torch.rand(3, N, generator=torch.Generator().manual_seed(steps)).to(DEV) < 0.3
        ids = torch.where(wrong, (ids + 1) % 500, ids)
        ids[:, 0] = root
        step = cache.step(new, rows=3 * N, max_new=N, keep=cached, parents=parents)
        logits = model.forward_cached(ids.view(-1), cache, step, rows="all")
        u = torch.rand(3 * N, dtype=torch.float64, device=DEV)
        counts, kept, chosen = ops.verify_draft(logits, ids.view(-1), step.row_start, N, u, temperature=0, parents=parents)
        cache.keep(step, kept, counts)
        root = chosen.gather(1, counts.long()[:, None] - 1)[:, 0]
        cached = cached + counts
        steps += 1
        for t, c, n in zip(texts, chosen.tolist(), counts.tolist()):
            t += c[:n]
        if max(len(t) for t in texts) > made + N:
            break
    assert steps < made
    for b, (t, w) in enumerate(zip(texts, want)):
        assert t == w[: len(t)].tolist(), b


def test_drafted_rows_are_adjacent():
    """As generate's without a draft: they can be viewed as one row of tokens."""
    model = _model(F32)
    prompt = _ids(3, 17)
    want = model.generate(prompt, 9, temperature=0.0)
    for tokens in (3, (2, 1)):
        out = model.generate(prompt, 9, temperature=0.0, draft_model=model, draft_tokens=tokens)
        assert out.is_contiguous() and torch.equal(out.view(-1), want.view(-1))


def test_counts_of_drafted_tokens_of_other_integer_types():
    np = pytest.importorskip("numpy")
    model = _model(F32)
    prompt = _ids(2, 17)
    want = model.generate(prompt, 9, temperature=0.0, draft_model=model, draft_tokens=3)
    for tokens in (np.int64(3), np.uint8(3), np.array([2, 1]), [np.int32(2), 1]):
        assert torch.equal(model.generate(prompt, 9, temperature=0.0, draft_model=model, draft_tokens=tokens), want)


def test_more_than_a_step_takes_is_refused_before_anything_is_made():
    """4096 sequences, and as many nodes of a tree."""
    model = _model(F32)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for batch, tokens in ((4097, 2), (1, 4096), (1, (500, 8))):
        with pytest.raises(ValueError, match="4096"):
            model.generate(_ids(batch, 3), 2, draft_model=model, draft_tokens=tokens)
    with pytest.raises(ValueError, match="4096"):
        _cache(model, 4097, 16)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20  # the caches of 4097 sequences alone are 1 GB


def test_reading_the_cache_counts_from_its_end_too():
    model = _model(F32)
    cache = _cache(model, 3, 40)
    model.forward_cached(_ids(31), cache, cache.step([11, 9, 11]), rows="none")
    for b in range(3):
        for x, y in zip(cache.read(0, b - 3), cache.read(0, b)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("top_k", [None, 4])
def test_a_draft_without_a_law_draws_from_all(top_k):
    """A draft model that has gone NaN costs tokens, and changes none."""
    model, draft = _model(F32), _model(F32, dim=128, n_layers=1, n_heads=2, n_kv_heads=1)
    with torch.no_grad():
        draft.norm.weight.fill_(math.nan)
    prompt = _ids(2, 17)
    out = model.generate(prompt, 9, temperature=1.0, top_k=top_k, draft_model=draft, draft_tokens=3)
    assert out.shape == (2, 26) and torch.equal(out[:, :17], prompt) and bool(((out >= 0) & (out < 500)).all())
    want = model.generate(prompt, 9, temperature=0.0)
    assert torch.equal(model.generate(prompt, 9, temperature=1.0, top_k=1, draft_model=draft, draft_tokens=3), want)


def test_a_servers_loop_in_which_sequences_end():
    """One reaches the cache's max_len, and gets no rows from then on; those of
    the others move up, and their texts go on as the model writes them."""
    N, limit, steps = 5, 60, 9
    model = _model(F32, max_seq_len=128)
    prompts = [_ids(n, seed=30 + n) for n in (30, 50, 6)]
    want = [model.generate(p[None], limit, temperature=0, use_cache=True)[0, len(p):] for p in prompts]
    cache = _cache(model, 3, limit)
    model.forward_cached(torch.cat([p[:-1] for p in prompts]), cache, cache.step([len(p) - 1 for p in prompts]), rows="none")
    root = torch.stack([p[-1] for p in prompts])
    start = cached = cache.tables.lengths.clone()
    new = torch.full((3,), N, dtype=torch.int32, device=DEV)
    parents = torch.tensor([-1, 0, 0, 2, 3], dtype=torch.int32, device=DEV)
    depth = torch.tensor([0, 1, 1, 2, 3], device=DEV)
    right = torch.stack(want)
    texts, unserved = [[], [], []], 0
    for _ in range(steps):
        ids = right.gather(1, ((cached - start).long()[:, None] + depth - 1).clamp(0, limit - 1))
        ids[:, 1] = (ids[:, 1] + 1) % 500  # a wrong branch beside the right one
        ids[:, 0] = root
        step = cache.step(new, rows=3 * N, max_new=N, keep=cached, parents=parents)
        served = step.row_start.diff()
        ids = ids[served.argsort(descending=True, stable=True)].view(-1)
        logits = model.forward_cached(ids, cache, step, rows="all")
        u = torch.rand(3 * N, dtype=torch.float64, device=DEV)
        counts, kept, chosen = ops.verify_draft(logits, ids, step.row_start, N, u, temperature=0, parents=parents)
        cache.keep(step, kept, counts)
        last = chosen.gather(1, (counts.long() - 1).clamp(min=0)[:, None])[:, 0]
        root = torch.where(served > 0, last, root)
        cached = cached + counts
        unserved += int((served == 0).sum())
        for t, c, n in zip(texts, chosen.tolist(), counts.tolist()):
            t += c[:n]
    assert unserved > 0 and len(texts[1]) < len(texts[0]) and len(texts[2]) > 20
    assert cached.tolist() == [len(p) - 1 + len(t) for p, t in zip(prompts, texts)] and max(cached.tolist()) <= limit
    for t, w in zip(texts, want):
        assert t == w[: len(t)].tolist()
    cache.free(1)
    new[1] = 0
    first = N * (int(cached[0]) + N <= limit)
    assert cache.step(new, rows=3 * N, max_new=N, keep=cached, parents=parents).row_start.tolist() == [0, first, first, first + N]
