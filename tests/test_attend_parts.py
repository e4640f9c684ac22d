"""Borders of a split row tile's parts (csrc/parts.h), compiled for the host with ROCm's clang, against Python's whole numbers,
up to the longest request a page table may hold."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mimo-on-a-mac_amd", "csrc")
CLANG = "/opt/rocm/llvm/bin/clang++"

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>
#include "parts.h"
int main(int argc, char** argv) {
  const int units = atoi(argv[1]), parts = atoi(argv[2]);
  for (int i = 0; i <= parts; ++i) printf("%d\n", mimo::part_begin(i, units, parts));
}
"""
# 64 keys a unit: short ones, the lengths around which a 32-bit product of 512 parts wraps, the longest request
KEYS = [320, 1 << 20, (1 << 28) - 64, 1 << 28, 300_000_000, (1 << 31) - (1 << 16)]


@pytest.mark.skipif(not os.path.exists(CLANG), reason="ROCm clang not installed")
def test_part_borders(tmp_path):
    src, exe = tmp_path / "parts.cpp", tmp_path / "parts"
    src.write_text(PROGRAM)
    subprocess.run([CLANG, "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-I", CSRC,
                    str(src), "-o", str(exe)], check=True)
    for keys in KEYS:
        units = -(-keys // 64)
        for parts in (1, 2, 3, 5, 511, 512, 1024):
            out = subprocess.run([str(exe), str(units), str(parts)], check=True, capture_output=True, text=True).stdout
            got = [int(x) for x in out.split()]
            assert got == [i * units // parts for i in range(parts + 1)], (keys, parts)
