"""What generation refuses before a GPU is asked, on the CPU."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from lzhip import _lib, ops
from lzhip.cache import CacheStep, KVCache, LayerCache

CSRC = Path(__file__).resolve().parents[1] / "cs244c-llama-zero_amd" / "csrc"


def _int32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    layer = LayerCache(torch.zeros(2, 1, 16, 32), torch.zeros(2, 1, 16, 32))
    step = CacheStep(_int32(2), _int32(1), _int32(1, 1), 1, 1, 1)
    for call in (lambda: ops.kv_cache_write(torch.zeros(1, 96), layer, step, 1, torch.zeros(1, 32), torch.zeros(1, 32)),
                 lambda: ops.kv_cache_read(layer, _int32(1, 1), _int32(2), 1, torch.float32),
                 lambda: ops.paged_attention(torch.zeros(1, 32), layer, step, 1, 1.0),
                 lambda: ops.process_logits(torch.zeros(1, 8)),
                 lambda: KVCache(1, 1, 32, batch=1, n_pages=1, device="cpu")):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


# The arguments below are refused before any of the pointers is used: 16 is a
# non-null, 16-byte aligned address that nothing reads.
P = 16
WRITE = dict(qkv=P, ld=192, dtype=1, rows=2, cos=P, sin=P, positions=8, q=P, ldq=64, k=P, v=P, k_exp=None, v_exp=None,
             cache=1, pages=4, size=16, table=P, width=2, row_start=P, kv_len=P, B=1, H=2, KV=2, hd=32, stream=None)
READ = dict(k=P, v=P, k_exp=None, v_exp=None, cache=1, pages=4, size=16, table=P, width=2, start=P, B=1, KV=2, hd=32,
            k_out=P, v_out=P, dtype=1, rows=3, stream=None)
ATTEND = dict(q=P, ldq=64, dtype=1, rows=2, k=P, v=P, k_exp=None, v_exp=None, cache=1, pages=4, size=16, table=P, width=2,
              row_start=P, kv_len=P, B=1, H=2, KV=2, hd=32, max_new=1, max_len=9, scale=1.0, o=P, ldo=64, ws=None,
              ws_bytes=0, stream=None)
LOGITS = dict(logits=P, ld=8, dtype=0, B=1, V=8, tokens=P, ldt=4, n=4, lengths=None, prompts=None, rep=None, rep_s=1.0,
              pres=None, pres_s=0.0, freq=None, freq_s=0.0, bias=None, ldb=0, mask=None, kind=0, ldm=0, out=P, ldo=8,
              stream=None)
PAGES = [dict(hd=48), dict(size=24), dict(size=8), dict(size=2048), dict(cache=0), dict(cache=8), dict(dtype=7), dict(k=24),
         dict(k=None), dict(pages=0), dict(B=0), dict(width=2**40), dict(pages=2**40), dict(KV=0)]


@pytest.mark.parametrize("name,args,bad", [
    ("lz_kv_write", WRITE, PAGES + [dict(ld=191), dict(ld=196), dict(ldq=63), dict(rows=-1), dict(H=0), dict(cos=None),
                                    dict(qkv=20), dict(positions=0), dict(rows=2**31)]),
    ("lz_kv_read", READ, PAGES + [dict(rows=-1), dict(k_out=None), dict(v_out=20)]),
    ("lz_paged_attn", ATTEND, PAGES + [dict(H=3), dict(H=0), dict(ldq=60), dict(ldo=60), dict(q=8), dict(o=None),
                                       dict(rows=-1), dict(max_new=-1), dict(kv_len=None), dict(scale=-1.0), dict(scale=0.0), dict(scale=1e-40),
                                       dict(scale=3e38), dict(scale=float("nan"))]),
    ("lz_process_logits", LOGITS, [dict(dtype=5), dict(kind=3), dict(kind=1), dict(mask=P), dict(ldo=7), dict(B=2, ld=7),
                                   dict(logits=None), dict(tokens=None), dict(n=-1), dict(V=2**40), dict(B=-1)]),
])
def test_c_entries_refuse(name, args, bad):
    for change in bad:
        if change == dict(cache=8):
            change = dict(cache=8, k_exp=P)  # exponents of one side alone
        with pytest.raises(_lib.HipLibraryError, match=name):
            _lib.call(name, *(args | change).values())


HOST = r"""
#include "kvcache.h"
#include <cstdio>
#include <vector>
int main() {
  int bad = 0;
  // rows -> sequences, ragged and empty ones among them
  const std::vector<std::vector<int>> counts = {{1}, {0}, {1, 1, 1, 1}, {3, 0, 40, 1, 17, 0, 5}, {0, 0, 2}, {5, 0, 0}, {7, 7, 7}};
  for (auto& n : counts) {
    std::vector<int> start = {0}, want;
    for (size_t b = 0; b < n.size(); ++b) {
      start.push_back(start.back() + n[b]);
      for (int i = 0; i < n[b]; ++i) want.push_back((int)b);
    }
    for (int pad = 0; pad < 4; ++pad) want.push_back(-1);  // rows of no sequence
    for (size_t r = 0; r < want.size(); ++r)
      if (lz_seq_of_row(start.data(), (int)n.size(), (int)want.size(), (int)r) != want[r]) ++bad;
  }
  // tables that say nonsense stay inside their own bounds
  const std::vector<int> odd = {9, -4, 2000000000, 3, -2147483647 - 1};
  for (int r = 0; r < 50; ++r) {
    const int b = lz_seq_of_row(odd.data(), 4, 50, r);
    if (b < -1 || b > 3) ++bad;
  }
  const std::vector<int> table = {0, 3, 4, -1, 2147483647, 2};
  const LzPages pg{table.data(), 3, 4, 4};
  const int want[2][5] = {{0, 3, -1, -1, -1}, {-1, -1, 2, -1, -1}};
  for (int b = 0; b < 2; ++b)
    for (int i = 0; i < 5; ++i)
      if (pg.page_of(b, 16 * i) != want[b][i] || pg.page_of(b, 16 * i + 15) != want[b][i]) ++bad;
  if (pg.page_of(0, -1) != -1 || pg.page_of(0, -2147483647 - 1) != -1 || pg.page_of(0, 2147483647) != -1) ++bad;
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_page_and_row_lookups_stay_inside(tmp_path):
    """The kernels' own lookups, run on the host."""
    sys.path.insert(0, str(CSRC))
    import build as B

    src = tmp_path / "lookups.hip"
    src.write_text(HOST)
    exe = tmp_path / "lookups"
    made = subprocess.run([B.find_hipcc(), "--offload-arch=gfx950", "-std=c++17", "-I", str(CSRC), str(src), "-o", str(exe)],
                          capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout
