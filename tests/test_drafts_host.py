"""What the operators of drafted tokens refuse before a GPU is asked, and their
lookups in tables and trees that say anything, on the CPU."""
from __future__ import annotations

import pytest
import torch

from lzhip import _lib, ops
from lzhip.cache import DraftStep, LayerCache, PageTables
from test_generation_tables import run_on_host


def _int32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    layer = LayerCache(torch.zeros(2, 1, 16, 32), torch.zeros(2, 1, 16, 32))
    step = DraftStep(_int32(2), _int32(1), _int32(1, 1), 1, 1, 1, _int32(1), _int32(1), torch.zeros(1, dtype=torch.int64),
                     _int32(1, 1))
    tables = PageTables(_int32(1, 1), _int32(1), _int32(2), _int32(1), 16)
    for call in (lambda: ops.cache_tables(tables, _int32(1), 1, 1, 1),
                 lambda: ops.verify_draft(torch.zeros(1, 8), torch.zeros(1, dtype=torch.int64), _int32(2), 1, torch.zeros(1)),
                 lambda: ops.kv_cache_keep(layer, step, _int32(1, 1), _int32(1)),
                 lambda: ops.paged_attention(torch.zeros(1, 32), layer, step, 1, 1.0),
                 lambda: ops.kv_cache_write(torch.zeros(1, 96), layer, step, 1, torch.zeros(1, 32), torch.zeros(1, 32))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


# Refused before any of the pointers is used: 16 is an address that nothing reads.
P = 16
WRITE = dict(qkv=P, ld=192, dtype=1, rows=2, cos=P, sin=P, positions=8, q=P, ldq=64, k=P, v=P, k_exp=None, v_exp=None,
             cache=1, pages=4, size=16, table=P, width=2, row_start=P, kv_len=P, at=P, B=1, H=2, KV=2, hd=32, stream=None)
TREE = dict(q=P, ldq=64, dtype=1, rows=2, k=P, v=P, k_exp=None, v_exp=None, cache=1, pages=4, size=16, table=P, width=2,
            row_start=P, kv_len=P, base=P, mask=P, words=1, B=1, H=2, KV=2, hd=32, max_new=1, max_len=9, scale=1.0, o=P,
            ldo=64, ws=None, ws_bytes=0, stream=None)
TABLES = dict(table=P, width=2, lengths=P, free=P, pages=4, n_free=P, size=16, add=P, keep=None, first=None, parents=P, ldp=0,
              nodes=33, B=2, rows=3, max_new=2, max_len=32, row_start=P, kv_len=P, base=P, positions=P, slots=P, mask=P,
              words=2, stream=None)
VERIFY = dict(logits=P, ld=8, dtype=0, rows=4, V=8, tokens=P, uniform=P, u_double=0, row_start=P, B=2, nodes=3, heat=None,
              heat_s=1.0, parents=P, ldp=0, tree=3, probs=None, ldq=8, counts=P, kept=P, chosen=P, ws=P, ws_bytes=10**6,
              stream=None)
KEEP = dict(k=P, v=P, k_exp=None, v_exp=None, cache=1, layers=2, pages=4, size=16, KV=2, hd=32, slots=P, rows=3, row_start=P,
            B=1, kept=P, ldk=4, nodes=4, counts=P, stream=None)


@pytest.mark.parametrize("name,args,bad", [
    ("lz_kv_write_at", WRITE, [dict(at=None), dict(hd=48), dict(ld=191), dict(rows=-1), dict(k=None), dict(cache=8)]),
    ("lz_tree_attn", TREE, [dict(base=None), dict(mask=None), dict(words=0), dict(words=2**30), dict(H=3), dict(q=8),
                            dict(scale=0.0), dict(max_new=-1), dict(size=24)]),
    ("lz_cache_tables", TABLES, [dict(size=24), dict(size=8), dict(B=0), dict(B=4097), dict(width=0), dict(width=2**30),
                                 dict(pages=0), dict(rows=-1), dict(rows=2**31), dict(max_new=-1), dict(max_len=2**31),
                                 dict(mask=None), dict(parents=None), dict(words=1), dict(nodes=0), dict(ldp=32), dict(ldp=34),
                                 dict(table=None), dict(slots=None), dict(add=None)]),
    ("lz_verify_draft", VERIFY, [dict(dtype=5), dict(rows=-1), dict(V=0), dict(V=2**29), dict(B=0), dict(nodes=0),
                                 dict(nodes=4097), dict(probs=P), dict(tree=0), dict(ldp=2), dict(ld=7), dict(tokens=None),
                                 dict(ws=None), dict(ws_bytes=8), dict(counts=None), dict(parents=None, probs=P, ldq=7)]),
    ("lz_kv_keep", KEEP, [dict(cache=5), dict(cache=8), dict(hd=48), dict(size=24), dict(layers=0), dict(pages=0), dict(B=0),
                          dict(B=65536), dict(k=8), dict(slots=None), dict(ldk=3), dict(rows=-1), dict(counts=None)]),
])
def test_c_entries_refuse(name, args, bad):
    for change in bad:
        with pytest.raises(_lib.HipLibraryError, match=name):
            _lib.call(name, *(args | change).values())


LOOKUPS = r"""
#include "draft.h"
#include "paged_attn.h"
#include <cstdio>
#include <vector>
int main() {
  int bad = 0;
  const std::vector<int> start = {0, 0, 3, 3, 3, 9, 10, 10};  // the last two begin behind the last entry
  const int want[] = {1, 1, 1, 4, 4, 4, 4, 4, 4, 5};
  for (int x = 0; x < 10; ++x) bad += lz_last_at(start.data(), 8, x) != want[x];
  const std::vector<int> odd = {9, -4, 2000000000, 3, -2147483647 - 1};
  for (int x = -3; x < 50; ++x) {
    const int b = lz_last_at(odd.data(), 5, x);
    bad += b < 0 || b > 4;
  }
  // parents that are no parents; a chain over three words; a word without ancestors
  std::vector<int> up(100);
  for (int i = 0; i < 100; ++i) up[i] = i - 1;
  up[40] = 3, up[50] = 50, up[60] = 61, up[70] = -9, up[71] = 2147483647;
  int mask[5];
  for (int i = -2; i < 103; ++i) {
    const int depth = lz_node_depth(up.data(), 100, i, mask, 4);
    std::vector<bool> seen(128, false);
    int d = -1;
    if (i >= 0 && i < 100)
      for (int at = i;;) {
        seen[at] = true, ++d;
        if (up[at] < 0 || up[at] >= at) break;
        at = up[at];
      }
    bad += depth != d || lz_node_depth(up.data(), 100, i, nullptr, 0) != d;
    for (int j = 0; j < 128; ++j) bad += ((mask[j / 32] >> (j % 32)) & 1) != seen[j];
  }
  // a row's bits from any key on
  const uint32_t row[3] = {0x80000001u, 0x0f0f1234u, 0xdeadbeefu};
  const int offs[] = {-2147483647 - 1, -1000, -33, -32, -31, -17, -1, 0, 1, 15, 31, 32, 33, 63, 64, 90, 95, 96, 97, 500, 2147483600};
  for (int words : {1, 2, 3})
    for (int off : offs) {
      const uint32_t b = tree_bits(row, words, off);
      for (int k = 0; k < 32; ++k) {
        const long at = (long)off + k;
        const bool one = at < 0 || (at < 32 * words && (row[at / 32] >> (at % 32) & 1));
        bad += ((b >> k) & 1) != one;
      }
    }
  // a sequence's rows and keys, whatever its length and base
  const int far[] = {-2147483647 - 1, -7, 0, 1, 99, 319, 320, 321, 2147483647};
  for (int len : far)
    for (int base : far) {
      PagedArgs a{};
      a.H = 6, a.KV = 2, a.rows = 100, a.nsplit = 4, a.chunk = 256, a.most = 90;
      a.pg = LzPages{nullptr, 5, 10, 6};
      a.base = &base;
      const TreeRows rw(a, 0, 10, 60, len, 32);
      const int n = len < 0 ? 0 : len > 320 ? 320 : len, ctx = base < 0 ? 0 : base > n ? n : base;
      bad += rw.count != 90 || rw.keys(16) != n || rw.sees(0) != n || rw.all(0) != ctx || rw.row(89) != 39;
      const int parts = PagedRows::parts(a, rw.keys(16));
      bad += parts < 1 || parts > 4;
    }
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_lookups_stay_inside(tmp_path):
    run_on_host(tmp_path, LOOKUPS)


STRETCHES = r"""
#include "paged_attn.h"
#include <cstdio>
int main() {
  int bad = 0;
  // a list of any length, dealt out in order, inside it and without gaps
  for (int all : {0, 1, 4, 127, 16777208, 2147483000, 2147483647})
    for (int per : {1, 4, 4194303, 8388604, 16777208, 2147483647}) {
      bad += lz_stretch(0, per, all) != 0;
      for (int w = 0; w < 512; ++w) {
        const int at = lz_stretch(w, per, all), end = lz_stretch(w + 1, per, all);
        bad += at < 0 || at > end || end > all || (end < all && (long)end - at != per);
      }
    }
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_shares_stay_inside(tmp_path):
    """Lengths past the call's bound make shares as long as the page table: 512 of
    8388604 units of 128 keys pass 32 bits."""
    run_on_host(tmp_path, STRETCHES)
