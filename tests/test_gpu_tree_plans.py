"""Attention of trees over a paged cache at sizes that make every choice of
blocks and shares, each named by its test so that other thresholds cannot leave
one untested."""
from __future__ import annotations

import pytest
import torch

from lzhip import _lib, ops
from test_gpu_drafts import _reference, _seen, _tree_case
from test_gpu_generation import BF16, DEV, F16, F32

pytestmark = pytest.mark.gpu
CODE = {F32: 0, BF16: 1, F16: 2}
B16, B8 = [(BF16, False), (F16, False)], [(BF16, True), (F16, True)]


def _ragged(n, new, length):
    """n sequences, the first as long as any: (new tokens, all), every seventh without any."""
    out = [(new, length)]
    for b in range(1, n):
        m = 0 if b % 7 == 3 else 1 + (b * 5) % new
        out.append((m, max(m, length * ((b * 13) % 29) // 29)))
    return out


PLANS = {
    # types, head dims, heads, sequences, (rows of a block, 1: shared out, 2: eight waves, parts)
    "whole texts": (B16 + B8, [128], (16, 8), _ragged(33, 16, 1000), (32, 0, 1)),
    "whole texts, small heads": (B16 + B8, [32, 64], (16, 8), _ragged(33, 16, 1000), (32, 2, 1)),
    "very many": (B16 + B8, [32, 64], (16, 8), _ragged(80, 9, 300), (32, 0, 1)),
    "shortest": (B16 + B8, [32, 64, 128], (8, 2), [(40, 200), (3, 10)], (32, 0, 1)),
    "short": (B16 + B8, [32, 64, 128], (8, 2), [(40, 500), (3, 10)], (32, 2, 1)),
    "for most of the CUs": (B16, [128], (32, 8), [(100, 2200), (70, 1200), (40, 900)], (32, 2, 1)),
    "one long text": (B16, [32, 64, 128], (32, 8), [(16, 8192)], (32, 1, 17)),
    "parts end at 33": (B16, [64], (8, 1), [(4, 20000), (1, 5), (3, 17000)], (32, 1, 33)),
    "wide trees": (B16 + B8, [32, 64, 128], (16, 4), _ragged(8, 30, 4500), (64, 1, 10)),
    "converted": (B8, [128], (32, 8), [(8, 4500), (3, 4100)], (64, 1, 10)),
    "converted, shorter": (B8, [128], (16, 8), _ragged(16, 16, 3001), (64, 1, 7)),
    "a little more than the CUs": (B16 + B8, [64, 128], (32, 8), [(300, 4500)], (64, 1, 10)),
    "many sequences": (B16 + B8, [64], (4, 2), _ragged(150, 3, 2500), (32, 1, 6)),
    "far more sequences than shares": (B16, [32], (64, 64), _ragged(200, 2, 2100), (32, 1, 6)),
}
CASES = [(name, *t, hd) for name, (types, dims, *_) in sorted(PLANS.items()) for t in types for hd in dims]


@pytest.mark.parametrize("name,dtype,e4m3,hd", CASES)
def test_every_plan(name, dtype, e4m3, hd):
    _, _, (H, KV), seqs, want_plan = PLANS[name]
    bases = [max(0, l - n - b % 3) for b, (n, l) in enumerate(seqs)]
    c, bits = _tree_case(seqs, bases, KV, hd, 64, dtype, e4m3, seed=hd)
    s, code = c.step, CODE[dtype]
    p = _lib.query("lz_tree_attn_plan", code, 8 if e4m3 else code, c.rows, len(seqs), H, KV, hd, s.max_new, s.max_len)
    assert (p & 255, p >> 8 & 255, p >> 16) == want_plan
    q = torch.randn(c.rows, H * hd, generator=c.g).to(dtype)
    got = ops.paged_attention(q.to(DEV), c.layer, c.draft, H, hd**-0.5)
    again = ops.paged_attention(q.to(DEV), c.layer, c.draft, H, hd**-0.5)
    assert torch.equal(got, again)
    want, tol = _reference(c, q, H, hd**-0.5, _seen(c, bases, bits))
    got = got.double().cpu()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())
