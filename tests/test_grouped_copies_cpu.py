"""Copies of operands to 16-byte rows: the axis of the grid that counts slices holds those of two operands, and the copies are little
larger than the operands."""
import shutil
import subprocess

import pytest

from sparsewave_b200 import _lib
from sparsewave_b200.build import CSRC

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "swb_index.h"
int main(int argc, char **argv) {
  for (int i = 1; i < argc; ++i) {
    const int64_t all = atoll(argv[i]), rows = swb::slice_rows(all), slices = swb::ceil_div(all, rows);
    printf("%lld %lld %lld\n", (long long)rows, (long long)slices, (long long)swb::copy_pitch(all));
  }
}
"""


@pytest.fixture(scope="module")
def numbers(tmp_path_factory):
    """(rows of a slice, slices, pitch of a copied row) for each of the given numbers."""
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("copies")
    (folder / "copies.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(folder / "copies.cpp"), "-o", str(folder / "copies")], check=True)

    def run(values):
        out = subprocess.run([str(folder / "copies"), *map(str, values)], check=True, capture_output=True, text=True).stdout
        lines = [tuple(map(int, line.split())) for line in out.splitlines()]
        assert len(lines) == len(values)
        return zip(values, lines)

    return run


def test_slices_of_two_operands_fit_the_grid(numbers):
    sizes = {1, 511, 512, 513, 2 ** 31 - 513}
    for s in (512, 513, 600, 1024, 4096, 131071):
        for slices in (16383, 16384, 16385, 32767, 32768):
            sizes |= {n for n in (s * slices - 1, s * slices, s * slices + 1) if n <= 2 ** 31 - 513}
    for all_rows, (rows, slices, _) in numbers(sorted(sizes)):
        assert rows * slices >= all_rows > rows * (slices - 1) and rows >= 512 and 2 * slices <= 65535


def test_copied_rows_are_little_longer(numbers):
    for row, (_, _, pitch) in numbers([*range(1, 2100), 2 ** 32 - 1026]):
        assert pitch % 16 == 0 and row <= pitch < row + (16 if row <= 16 else 32 if row < 512 else 128)
        assert row < 512 or pitch <= 1.25 * row


def test_trim_wants_a_context():
    lib = _lib.load()
    assert lib.swb_trim(None) == _lib.SWB_ERR_INVALID_ARGUMENT and lib.swb_last_error(None) == b"context is NULL"
