"""The model's cached forward around its kernels, which these tests replace,
on the CPU."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from lzhip import functional as LF
from lzhip import ops
from lzhip.cache import CacheStep, LayerCache
from model import LlamaForCausalLM, ModelConfig


def _config(**kw):
    return ModelConfig(**(dict(name="t", vocab_size=64, max_seq_len=48, dim=64, n_layers=1, n_heads=2, n_kv_heads=1,
                               ffn_dim=96, dropout=0.5) | kw))


def test_a_cached_block_leaves_the_modes_alone(monkeypatch):
    """No dropout, though the module says training, and during the MLP's
    kernels (another thread may read it then) it still does."""
    block = LlamaForCausalLM(_config()).train().layers[0]
    block.input_norm = block.post_attn_norm = nn.Identity()
    block.attn.forward_cached = lambda x, layer, step, residual: residual
    seen = []

    def apply(x, wg, wu, wd, residual, grad, p, seed, compute=True):
        seen.append((block.mlp.training, p))
        return residual

    monkeypatch.setattr(ops, "require_gpu", lambda *t: None)
    monkeypatch.setattr(LF.MLPFn, "apply", apply)
    x = torch.ones(3, 64)
    assert block.forward_cached(x, None, None) is x
    assert seen == [(True, 0.0)] and block.mlp.training


class Fixed(LlamaForCausalLM):
    """A model whose last logits are given."""

    def __init__(self, rows):
        super().__init__(_config(dropout=0.0, vocab_size=len(rows[0])))
        self.rows = torch.tensor(rows)

    def forward(self, ids):
        return type("Out", (), {"logits": self.rows[:, None].expand(-1, ids.shape[1], -1)})


@pytest.fixture
def plain_adjustments(monkeypatch):
    """process_logits' bias and mask on the CPU."""
    def process(x, *, bias=None, mask=None, **_):
        x = x.float() if bias is None else x.float() + bias
        return x if mask is None else x.masked_fill(~mask, -float("inf"))

    monkeypatch.setattr(ops, "process_logits", process)


def test_an_infinite_bias_forces_a_token(plain_adjustments):
    model = Fixed([[0.0, 1.0, 2.0, 3.0], [3.0, 2.0, 1.0, 0.0]])
    bias = torch.tensor([0.0, float("inf"), 0.0, 0.0])
    ids = torch.zeros(2, 3, dtype=torch.int64)
    assert model.generate(ids, 2, temperature=0.0, logit_bias=bias)[:, 3:].tolist() == [[1, 1], [1, 1]]
    # there is no distribution to sample from
    with pytest.raises(ValueError, match="token 3.*infinite"):
        model.generate(ids, 2, temperature=1.0, logit_bias=bias)


def test_rows_without_a_token_are_refused(plain_adjustments):
    model = Fixed([[0.0, 1.0, 2.0, 3.0], [3.0, 2.0, 1.0, 0.0]])
    ids = torch.zeros(2, 3, dtype=torch.int64)
    mask = torch.ones(2, 4, dtype=torch.bool)
    mask[1] = False
    for how in (dict(temperature=0.0), dict(temperature=1.0, top_k=2)):
        with pytest.raises(ValueError, match="token 3.*no token"):
            model.generate(ids, 2, token_mask=mask, **how)
        with pytest.raises(ValueError, match="token 3.*NaN"):
            model.generate(ids, 2, logit_bias=torch.tensor([0.0, float("nan"), 0.0, 0.0]), **how)


def _cached_attention(monkeypatch, attn):
    """attn.forward_cached with its kernels replaced: the tables of each call."""
    tables = []

    def write(qkv, layer, step, heads, cos, sin, out=None):
        tables.append((cos, sin))
        return qkv[:, : heads * 32]

    monkeypatch.setattr(ops, "require_gpu", lambda *t: None)
    monkeypatch.setattr(ops, "gemm", lambda x, w: x.new_zeros(x.shape[0], w.shape[0]))
    monkeypatch.setattr(ops, "copy2d", lambda a, b: b.copy_(a))
    monkeypatch.setattr(ops, "kv_cache_write", write)
    monkeypatch.setattr(ops, "paged_attention", lambda q, *a: q)
    attn.o_proj.forward = lambda y, residual=None: y
    return tables


def _step(max_len):
    return CacheStep(None, None, None, 2, 1, max_len)


def test_replaced_rotary_tables_are_asked_for_the_sequence_alone(monkeypatch):
    """A rotary of the user's own may depend on the length or end at the
    model's: it gets the longest sequence's, as the uncached forward gives
    it its own."""
    attn = LlamaForCausalLM(_config()).layers[0].attn
    asked = []

    def forward(seq_len, device, dtype):
        asked.append(seq_len)
        assert seq_len <= 48
        return torch.ones(1, 1, seq_len, 32), torch.zeros(1, 1, seq_len, 32)

    attn.rotary.forward = forward
    tables = _cached_attention(monkeypatch, attn)
    for n in (1, 7, 48):
        attn.forward_cached(torch.ones(2, 64), None, _step(n))
    assert asked == [1, 7, 48] and [t[0].shape for t in tables] == [(1, 32), (7, 32), (48, 32)]


def test_rotary_tables_of_a_captured_call_stay(monkeypatch):
    """A graph keeps the tables' addresses: they live on where an eager call
    needs longer ones.  What is built under capture holds nothing before a
    replay, so no other call gets it."""
    import gc
    import weakref

    rotary = LlamaForCausalLM(_config()).layers[0].attn.rotary
    capturing = [False]
    monkeypatch.setattr(ops, "capturing", lambda: capturing[0])
    monkeypatch.setattr(ops, "rope_table", lambda n, dim, inv, dtype: (torch.zeros(n, dim), torch.zeros(n, dim)))
    cpu = torch.device("cpu")

    def call(n, captured, how):
        capturing[0] = captured
        try:
            return (rotary.tables if how else rotary.forward)(n, cpu, torch.float32)[0]
        finally:
            capturing[0] = False

    for how in (True, False):
        rotary.max_seq_len_cached = 0
        eager = call(8, False, how).data_ptr()
        assert call(5, True, how).data_ptr() == eager
        kept = weakref.ref(rotary.cos_cached)
        assert call(16, False, how).data_ptr() != eager  # grown
        gc.collect()
        assert kept() is not None
        inside = call(32, True, how)
        assert inside.shape[-2] == 32 and rotary.max_seq_len_cached == 16
        assert call(20, False, how).data_ptr() != inside.data_ptr() and rotary.max_seq_len_cached == 20
        assert call(8, True, how).data_ptr() == call(9, True, how).data_ptr()
    gone = weakref.ref(rotary.cos_cached)  # in no graph: not kept
    rotary.max_seq_len_cached = 0
    call(8, False, True)
    first = weakref.ref(rotary.cos_cached)
    call(64, False, True)
    gc.collect()
    assert gone() is not None and first() is None


def test_penalties_may_be_one_for_each_row(monkeypatch):
    """generate hands them on as process_logits takes them: numbers or
    tensors."""
    got = []

    def process(x, **kw):
        got.append({k: kw[k] for k in ("repetition_penalty", "presence_penalty", "frequency_penalty")})
        return x.float()

    monkeypatch.setattr(ops, "process_logits", process)
    model = Fixed([[0.0, 1.0, 2.0, 3.0], [3.0, 2.0, 1.0, 0.0]])
    ids, each = torch.zeros(2, 3, dtype=torch.int64), torch.tensor([1.0, 1.5])
    for name in ("repetition_penalty", "presence_penalty", "frequency_penalty"):
        model.generate(ids, 1, temperature=0.0, **{name: each})
        assert len(got) == 1 and got.pop()[name] is each
    model.generate(ids, 1, temperature=0.0, repetition_penalty=1, presence_penalty=0)  # nothing to adjust
    assert not got


def _cpu_cache(batch, n_pages):
    from lzhip.cache import KVCache

    cache = object.__new__(KVCache)  # its tables alone
    cache.device, cache.page_size, cache.n_pages = torch.device("cpu"), 16, n_pages
    cache.lengths, cache._pages = [0] * batch, [[] for _ in range(batch)]
    cache._free = list(range(n_pages - 1, -1, -1))
    return cache


def test_a_step_that_fails_changes_nothing():
    cache = _cpu_cache(3, 6)
    s = cache.step([20, 0, 3])
    assert s.row_start.tolist() == [0, 20, 20, 23] and s.kv_len.tolist() == [20, 0, 3]
    before = (list(cache.lengths), [list(p) for p in cache._pages], list(cache._free))
    for bad, err in (([1, 1.5, 1], TypeError), ([1, 20, "2"], TypeError), ([1, 1], ValueError), ([1, -1, 1], ValueError),
                     ([0, 70, 0], RuntimeError)):
        with pytest.raises(err):
            cache.step(bad)
    cache.device = torch.device("cuda:0")  # the tables do not arrive
    with pytest.raises(Exception):
        cache.step([20, 1, 1])
    cache.device = torch.device("cpu")
    assert (cache.lengths, cache._pages, cache._free) == before
    s = cache.step([20, 1, 1])
    used = [p for row in s.page_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 5 and cache.lengths == [40, 1, 4] and len(cache._free) == 1
