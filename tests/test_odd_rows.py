"""Which vectors the norm loads of rows that do not start on 16 bytes: none past the end of a tensor."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mingru_b200" / "csrc"

# Every load of OddRow::load, by its own rules: vectors from the one that a group's first element is in.
PROGRAM = """
#include <cstdio>
#include <initializer_list>
#include "odd_rows.h"
int main() {
  long long loads = 0;
  for (int v : {4, 8})
    for (int D = 1; D <= 41; ++D)
      for (long long ld = 0; ld <= 2 * D + 16; ++ld) {
        if (ld % v != D % v) continue;  // what the kernels take as odd rows
        for (int rows : {1, 2, 3, 9, 37}) {
          if (rows > 1 && !mgs::odd::steps_far_enough(ld, v)) continue;  // read element by element
          for (int groups = 1; groups <= D; ++groups) {
            if (D % groups) continue;
            const int n = D / groups;
            const long long extent = (rows - 1) * ld + D;
            for (int r = 0; r < rows; ++r)
              for (int g = 0; g < groups; ++g) {
                const long long start = r * ld + g * n;
                const int sh = (int)(start & (v - 1));
                for (int pos = 0; pos < sh + n; pos += v) {
                  const bool all = mgs::odd::whole(pos, sh + n, v, r + 1 == rows);
                  const long long first = start - sh + pos, end = all ? first + v : start + n;
                  ++loads;
                  if (first < 0 || end > extent) {
                    std::printf("v %d D %d ld %lld rows %d groups %d: row %d group %d reads %lld..%lld of %lld\\n", v, D, ld,
                                rows, groups, r, g, first, end, extent);
                    return 1;
                  }
                }
              }
          }
        }
      }
  std::printf("%lld\\n", loads);
  return loads > 100000 ? 0 : 2;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_loads_stay_inside(tmp_path):
    (tmp_path / "loads.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++20", "-O1", f"-I{CSRC}", "loads.cpp", "-o", "loads"], cwd=tmp_path, check=True)
    run = subprocess.run([tmp_path / "loads"], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
