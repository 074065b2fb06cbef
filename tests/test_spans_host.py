"""Checks of what memory a call's tensors take, without a GPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "llm_gpu_kernels_amd" / "csrc"

# Every pair of small row sets against a map of the bytes.  Rows that may meet and do not are
# allowed only where the strides differ (a common divisor is what decides there).
PROGRAM = r"""
#include <stdio.h>
#include <string.h>
#include "spans.h"
static char bytes[4096];
int main() {
  using namespace moe;
  long apart = 0, between = 0, careful = 0;
  for (int row = 1; row <= 4; ++row)
    for (int n = 1; n <= 4; ++n)
      for (int sa = row; sa <= 12; ++sa)
        for (int sb = row; sb <= 12; ++sb)
          for (int at = 0; at <= 120; ++at) {
            const Rows a = {bytes + 60, sa, row, n}, b = {bytes + at, sb, row, n};
            memset(bytes, 0, 256);
            for (int i = 0; i < n * row; ++i) bytes[60 + i / row * sa + i % row] = 1;
            bool common = false;
            for (int i = 0; i < n * row; ++i) common |= bytes[at + i / row * sb + i % row] != 0;
            const bool said = may_meet(a, b);
            if (said != may_meet(b, a) || (common && !said) || (said && !common && sa == sb)) {
              printf("row %d n %d strides %d %d at %d: %d %d\n", row, n, sa, sb, at, common, said);
              return 1;
            }
            apart += !said;
            between += !said && meet(span_of(a), span_of(b));
            careful += said && !common;
          }
  const char *const far = (const char *)0x7fff00000000;  // strides and counts as large as a call's
  const int64_t stride = 1ll << 31, n = 1 << 26;
  const Rows x = {far, stride, 256, n}, y = {far + 256, stride, 256, n}, z = {far + 128, stride, 256, n};
  if (may_meet(x, y) || !may_meet(x, z) || !may_meet(x, x)) return 2;
  if (meet(span_of(nullptr, 0), span_of(nullptr, 0)) || meet(span_of(far, 0), span_of(nullptr, 16))) return 3;
  printf("%ld %ld %ld\n", apart, between, careful);
  return between > 0 ? 0 : 4;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_that_meet(tmp_path):
    (tmp_path / "test.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(tmp_path / "test.cpp"), "-o",
                    str(tmp_path / "test")], check=True)
    done = subprocess.run([str(tmp_path / "test")], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
