"""What the attention over the cache makes of its device tables, whatever they
say: the kernels' own arithmetic, run on the host."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "cs244c-llama-zero_amd" / "csrc"


def run_on_host(tmp_path, source):
    sys.path.insert(0, str(CSRC))
    import build as B

    src, exe = tmp_path / "host.hip", tmp_path / "host"
    src.write_text(source)
    made = subprocess.run([B.find_hipcc(), "--offload-arch=gfx950", "-std=c++17", "-I", str(CSRC), str(src), "-o", str(exe)],
                          capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout


ROWS = r"""
#include "paged_attn.h"
#include <cstdio>
int main() {
  const int odd[] = {-2147483647 - 1, -1000000000, -7, -1, 0, 1, 3, 99, 100, 101, 1000000000, 2000000000, 2147483647};
  int bad = 0;
  for (int G : {1, 3, 8, 33})
   for (int most : {7, 100})
    for (int lo : odd)
      for (int hi : odd)
        for (int len : odd) {
          PagedArgs a{};
          a.H = 2 * G, a.KV = 2, a.rows = 100, a.nsplit = 4, a.chunk = 256, a.most = most * G;
          a.pg = LzPages{nullptr, 5, 10, 6};
          const PagedRows all(a, lo, hi, len, 0);
          // the rows of [lo, hi) that there are
          long first = lo > 0 ? lo : 0, last = hi < 100 ? hi : 100, want = last > first ? (last - first) * G : 0;
          if (want > a.most) want = a.most;
          if (all.count != want) {
            if (!bad++) printf("G %d, %d .. %d: %d rows, not %ld\n", G, lo, hi, all.count, want);
            continue;
          }
          for (int m0 = 0; m0 < all.count; m0 += 16) {
            const PagedRows rw(a, lo, hi, len, m0);
            const int m1 = m0 + 15 < rw.count ? m0 + 15 : rw.count - 1;
            for (int m : {m0, m1})
              if (rw.row(m) < 0 || rw.row(m) >= 100 || rw.sees(m) < 0 || rw.sees(m) > 5 * 64) ++bad;
            const int keys = rw.keys(16), parts = PagedRows::parts(a, keys);
            if (keys < 0 || keys > 5 * 64 || parts < 1 || parts > 4) ++bad;
          }
        }
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_rows_of_any_table_are_rows_of_the_call(tmp_path):
    """Starts far past the last row, descending, negative: no row outside q
    and no more rows than there are."""
    run_on_host(tmp_path, ROWS)


SEES = r"""
#include "paged_attn.h"
#include <cstdio>
#include <vector>
int main() {
  int bad = 0;
  for (int log_size : {4, 5, 8, 10})
    for (int there = -1; there < 7; ++there) {  // the one page that there is
      std::vector<int> table(14, -1);
      if (there >= 0) table[7 + there] = 3;
      PagedArgs a{};
      a.pg = LzPages{table.data(), 7, 10, log_size};
      for (int k_lo = 0; k_lo <= 7 << log_size; k_lo += 64)
        for (int k_hi : {k_lo, k_lo + 1, k_lo + 64, 5 << log_size, 7 << log_size, 2147483647})
          for (int sees : {0, 1, 63, 64, 65, 3 << log_size, (3 << log_size) + 1, 7 << log_size}) {
            bool want = false;
            for (int key = k_lo; key < k_hi && key < sees; ++key) want |= key >> log_size == there;
            bad += sees_any(a, 1, k_lo, k_hi, sees) != want;
          }
    }
  // the longest table there can be
  std::vector<int> longest(2147483647 / 1024, -1);
  PagedArgs a{};
  a.pg = LzPages{longest.data(), (int)longest.size(), 10, 10};
  const int cap = a.pg.width << 10;
  bad += sees_any(a, 0, 0, 2147483647, cap);
  longest.back() = 0;
  bad += !sees_any(a, 0, cap - 1024, cap, cap) || sees_any(a, 0, 0, cap, cap - 1024);
  printf("%d\n", bad);
  return bad != 0;
}
"""


def test_whether_a_row_sees_a_key(tmp_path):
    run_on_host(tmp_path, SEES)
