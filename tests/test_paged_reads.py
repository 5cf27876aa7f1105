"""What paged_token's lanes read of a row (limn_amd/csrc/paged_reads.h), walked on the host over every head dim and type that the
tiled kernels of a paged cache take: nothing outside the row, and every dim of it as some lane's own."""

from __future__ import annotations

import shutil
import subprocess

from limn_amd.build import CSRC, hipcc

# the kernel's loads: a value lane W elements from value_dim on where W n < hd; a key lane 16 bytes from PER (4 s + g) on where that is below hd
WALK = r"""
#include "paged_reads.h"
#include <initializer_list>
#include <stdio.h>
using namespace limn;
int main() {
  for (int bytes : {2, 4})
    for (int hd = 1; hd <= 300; hd++) {
      if (!paged_dim(hd, bytes)) continue;
      const int D = token_width(hd), W = D / 16, PER = 16 / bytes;
      bool own[300] = {}, keys[300] = {};
      for (int n = 0; n < 16; n++) {
        if (W * n >= hd) continue;
        const int from = value_dim(n, W, hd);
        if (from < 0 || from + W > hd) printf("values of %d-byte hd %d: lane %d reads %d to %d\n", bytes, hd, n, from, from + W);
        if (from > W * n) printf("values of %d-byte hd %d: lane %d passes its first dim\n", bytes, hd, n);
        for (int d = W * n; d < from + W && d < hd; d++) {
          if (own[d]) printf("%d-byte hd %d: dim %d stored twice\n", bytes, hd, d);
          own[d] = true;
        }
      }
      for (int s = 0; s < D / (4 * PER); s++)
        for (int g = 0; g < 4; g++) {
          const int from = PER * (4 * s + g);
          if (from >= hd) continue;
          if (from + PER > hd) printf("keys of %d-byte hd %d: %d to %d\n", bytes, hd, from, from + PER);
          for (int d = from; d < from + PER; d++) keys[d] = true;
        }
      for (int d = 0; d < hd; d++)
        if (!own[d] || !keys[d]) printf("%d-byte hd %d: dim %d is nobody's\n", bytes, hd, d);
      printf("%d:%d ", bytes, hd);
    }
  return 0;
}
"""


def test_no_lane_reads_past_its_row(tmp_path):
    source, program = tmp_path / "walk.cpp", tmp_path / "walk"
    source.write_text(WALK)
    done = subprocess.run([shutil.which("g++") or hipcc(), "-std=c++17", f"-I{CSRC}", str(source), "-o", str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    out = subprocess.run([str(program)], capture_output=True, text=True).stdout
    assert out.split() == [f"2:{hd}" for hd in range(8, 129, 8)] + [f"4:{hd}" for hd in range(4, 129, 4)], out
    kernel = (CSRC / "paged_token.hip").read_text()  # the walk is of the kernel's own rule
    assert "value_dim(n, W, v.hd)" in kernel and "W * n < v.hd" in kernel and "PER * (4 * s + g) < v.hd" in kernel
