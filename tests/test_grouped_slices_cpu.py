"""Slices of long operands on their way to 16-byte rows: the axis of the grid that counts them holds those of two operands."""
import shutil
import subprocess

import pytest

from sparsewave_b200.build import CSRC

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "swb_index.h"
int main(int argc, char **argv) {
  for (int i = 1; i < argc; ++i) {
    const int64_t all = atoll(argv[i]), rows = swb::slice_rows(all), slices = swb::ceil_div(all, rows);
    printf("%lld %lld\n", (long long)rows, (long long)slices);
  }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_slices_of_two_operands_fit_the_grid(tmp_path):
    source, program = tmp_path / "slices.cpp", tmp_path / "slices"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(source), "-o", str(program)], check=True)
    sizes = {1, 511, 512, 513, 2 ** 31 - 513}
    for s in (512, 513, 600, 1024, 4096, 131071):
        for slices in (16383, 16384, 16385, 32767, 32768):
            sizes |= {n for n in (s * slices - 1, s * slices, s * slices + 1) if n <= 2 ** 31 - 513}
    sizes = sorted(sizes)
    out = subprocess.run([str(program), *map(str, sizes)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(out) == len(sizes)
    for all_rows, line in zip(sizes, out):
        rows, slices = map(int, line.split())
        assert rows * slices >= all_rows > rows * (slices - 1) and rows >= 512 and 2 * slices <= 65535
