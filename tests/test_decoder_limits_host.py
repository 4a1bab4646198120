"""Sizes near the documented limits of the decoder-layer operators, on a machine without a
GPU: the arithmetic of the shared headers, compiled for the host."""

import os
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT

PROGRAM = r"""
#include "fp8_block.h"
using cb::tile_bytes;
int main() {
  for (int width : {64, 128})
    for (int elem : {2, 4}) {
      const long long sizes[] = {1, 3, width - 1, width, width + 1, 1 << 20, (1 << 29) - 1, 1 << 29, (1 << 29) + 77, (1 << 30) - 1, 1 << 30};
      for (long long n : sizes) {
        const long long want = (n < width ? n : width) * elem;
        if (tile_bytes(static_cast<int>(n), width, elem) != want) return 1;
      }
    }
  return 0;
}
"""


def test_bytes_of_a_tile_of_a_long_output_row(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover", "-I" + cuda,
                    "-I" + os.path.join(PKG, "csrc"), "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)]).returncode == 0
