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
