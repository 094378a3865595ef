"""The rule that cuts the dX product's range into splits (csrc/dx_splits.hpp), built by the host compiler with its integer checks on:
over sizes of all kinds, no live rows among them, the splits cover the range once, their partial tiles fit what is reserved, and
nothing is divided by zero."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'coupled-vae_amd', 'csrc')

PROGRAM = r'''
#include <cstdio>
#include "dx_splits.hpp"
using namespace cvae;
int main() {
  const int tiles[] = {0, 1, 2, 3, 7, 28, 29, 64, 128, 255, 256, 257, 1000, 1024, 1025, 40000};
  const int stages[] = {1, 2, 3, 4, 5, 8, 31, 32, 33, 100, 313, 625, 1563, 4096};
  const int dw[] = {1, 2, 79, 157, 255, 256, 257, 391, 3000}, d[] = {6, 7, 33, 120, 4000};
  for (int t : tiles) for (int s : stages) for (int w : dw) for (int x : d) for (int spare = 0; spare < 2; ++spare) {
    int best = 0x7fffffff, lane = -1;
    DxSplit all[65];
    for (int k = 1; k <= 64; ++k) {
      all[k] = dx_split(k, t, s, x, w, spare);
      if (all[k].cost < best) { best = all[k].cost; lane = best & 63; }
    }
    const int k = lane + 1;
    if (lane < 0 || (k > 1 && (k * 4 > s || (long)t * k > DT_DX_MOST))) { printf("k %d of %d tiles, %d stages\n", k, t, s); return 1; }
    const int rows_at_most[] = {t, t + 1, 3 * t + 2, 50000};
    for (int m : rows_at_most)
      if ((long)t * k > dx_partial_tiles(m, s)) { printf("slab: %d of %d tiles, %d stages, k %d\n", t, m, s, k); return 1; }
    const Splits r = dx_splits_of(k, all[k].size, all[k].longer, s);
    if (r.n != k || r.begin(0) != 0 || r.begin(r.n) < s) { printf("not covered: %d tiles, %d stages, k %d\n", t, s, k); return 1; }
    for (int i = 0; i < r.n; ++i)
      if (r.begin(i + 1) < r.begin(i)) { printf("order: %d tiles, %d stages, k %d\n", t, s, k); return 1; }
  }
  return 0;
}
'''


def test_splits_cover_every_range(tmp_path):
    cxx = shutil.which('g++')
    if not cxx:
        pytest.skip('no host compiler')
    src, exe = tmp_path / 'splits.cpp', tmp_path / 'splits'
    src.write_text(PROGRAM)
    subprocess.check_call([cxx, '-O1', '-std=c++17', '-fsanitize=undefined', '-fno-sanitize-recover=undefined', '-I', CSRC, str(src),
                           '-o', str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
