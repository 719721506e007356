"""The paged key/value cache of generation.

LayerCache and CacheStep are what the kernels take (ops.kv_cache_write,
ops.paged_attention, ops.kv_cache_read); KVCache owns the pages of a model's
layers and hands them to sequences.  The reference has no cache: its generate
(model/llama.py:311-335) runs the whole window through the model for every
token.
"""
from __future__ import annotations

import itertools
import operator
from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import ops


class LayerCache(NamedTuple):
    """One layer's pages, [pages, KV heads, page size, head dim] each, in the
    model's dtype, or float8_e4m3fn with int8 exponents [pages, KV heads, page
    size]: the value is the stored number times 2^exponent (-126 to 127).
    8-bit pages are read in the dtype that they were written with: float16
    keeps smaller exponents than the others.  Where two rows of one step are
    given the same slot, it holds parts of both."""

    k: torch.Tensor
    v: torch.Tensor
    k_exp: Optional[torch.Tensor] = None
    v_exp: Optional[torch.Tensor] = None


class CacheStep(NamedTuple):
    """The new tokens of one pass through the layers.  Device tensors, int32:
    row_start [B + 1] (sequence b's new tokens are rows row_start[b] ..
    row_start[b + 1] - 1, from row_start[0] = 0 on), kv_len [B] (its length with
    them), page_table [B, pages of the longest].  Host numbers: rows =
    row_start[B], and upper bounds max_new and max_len of the new and of all
    tokens of a sequence.  Tables that change under a captured call keep within
    them: rows behind max_new of a sequence, or of none, are not computed (the
    caller's tensor keeps what it holds there, one of the call's own holds
    anything but in the rows from `rows` on, which are zeros)."""

    row_start: torch.Tensor
    kv_len: torch.Tensor
    page_table: torch.Tensor
    rows: int
    max_new: int
    max_len: int


class KVCache:
    """Pages for n_layers layers and up to `batch` sequences.

    storage: the model's dtype (None) or torch.float8_e4m3fn.  n_pages pages
    are shared by all sequences: each takes pages as it grows, a page holding
    page_size of its tokens in every layer, and free() gives them back."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, *, batch: int, n_pages: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, storage: Optional[torch.dtype] = None, device="cuda") -> None:
        if head_dim not in (32, 64, 128):
            raise ValueError(f"the cache's kernels take head dims 32, 64 and 128, not {head_dim}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page size must be a power of two from 16 to 1024, got {page_size}")
        if min(n_layers, n_kv_heads, batch, n_pages) < 1:
            raise ValueError("layers, heads, sequences and pages must be positive")
        if dtype not in ops._DTYPES:
            raise TypeError(f"a cache holds float32, bfloat16 or float16 rows, not {dtype}")
        if storage not in (None, dtype, torch.float8_e4m3fn):
            raise TypeError(f"a cache stores {dtype} or torch.float8_e4m3fn, not {storage}")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError(f"llama-zero HIP kernels run on a ROCm GPU; got device {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.dtype, self.page_size, self.n_pages = dtype, page_size, n_pages
        eight = storage == torch.float8_e4m3fn
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        store = torch.float8_e4m3fn if eight else dtype
        self._k, self._v = (torch.empty(shape, dtype=store, device=self.device) for _ in range(2))
        exps: List[Optional[torch.Tensor]] = [None, None]
        if eight:
            exps = [torch.empty(shape[:4], dtype=torch.int8, device=self.device) for _ in range(2)]
        self.layers = [LayerCache(self._k[i], self._v[i], *(None if e is None else e[i] for e in exps))
                       for i in range(n_layers)]
        self.lengths = [0] * batch
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(n_pages - 1, -1, -1))

    @staticmethod
    def _page_table(pages: Sequence[List[int]]) -> List[List[int]]:
        width = max(1, max(map(len, pages)))
        return [p + [-1] * (width - len(p)) for p in pages]

    def step(self, new: Sequence[int]) -> CacheStep:
        """Room for new[b] more tokens of every sequence b (0: none) and the
        CacheStep that the layers' calls take.  A call that fails (the pages do
        not suffice, say) changes nothing."""
        new = [operator.index(n) for n in new]
        if len(new) != len(self.lengths):
            raise ValueError(f"{len(new)} counts of new tokens for {len(self.lengths)} sequences")
        if min(new) < 0:
            raise ValueError("counts of new tokens must not be negative")
        lengths = [n + l for n, l in zip(new, self.lengths)]
        want = [-(-l // self.page_size) - len(p) for l, p in zip(lengths, self._pages)]
        left = len(self._free) - sum(want)
        if left < 0:
            raise RuntimeError(f"the cache has {len(self._free)} free pages of {self.page_size} tokens; {sum(want)} "
                               "more are needed: free() sequences or make it larger")
        taken = iter(self._free[: left - 1 if left else None : -1])
        more = [list(itertools.islice(taken, n)) for n in want]
        B, starts = len(new), [0, *itertools.accumulate(new)]
        table = self._page_table([p + m for p, m in zip(self._pages, more)])
        flat = torch.tensor(starts + lengths + [p for row in table for p in row], dtype=torch.int32)
        flat = flat.to(self.device)
        self.lengths[:] = lengths
        del self._free[left:]
        for p, m in zip(self._pages, more):
            p += m
        return CacheStep(flat[: B + 1], flat[B + 1 : 2 * B + 1], flat[2 * B + 1 :].view(B, -1), starts[-1], max(new),
                         max(lengths))

    def free(self, b: int) -> None:
        """Ends sequence b: its pages go back, and its slot is empty."""
        self._free += reversed(self._pages[b])
        self._pages[b], self.lengths[b] = [], 0

    def read(self, layer: int, b: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Sequence b's keys and values in one layer, [tokens, KV heads, head
        dim] each, in the model's dtype."""
        n, kv = self.lengths[b], self.layers[layer]
        flat = torch.tensor([0, n] + self._page_table([self._pages[b]])[0], dtype=torch.int32).to(self.device)
        k, v = ops.kv_cache_read(kv, flat[2:].view(1, -1), flat[:2], n, self.dtype)
        return k.view(n, *kv.k.shape[1::2]), v.view(n, *kv.v.shape[1::2])
