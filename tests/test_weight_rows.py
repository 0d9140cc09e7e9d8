"""The cut of the attention weights' query rows into blocks (firefly_amd/csrc/weight_rows.h), compiled for the CPU with
UndefinedBehaviorSanitizer: every row lies in one block, and a call without queries has none and divides by no zero."""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "firefly_amd" / "csrc"

PROGRAM = """
#include "weight_rows.h"
#include <cstdio>
int main()
{
    for (int most = 16; most <= 256; most += 16)
        for (int rows = 0; rows <= 1 << 20; rows += rows < 600 ? 1 : 997)
        {
            const int block = ffkv::weight_block_rows(rows, most);
            const int n = ffkv::weight_row_blocks(rows, block);
            const bool covers = rows == 0 ? n == 0 : (n - 1) * block < rows && rows <= n * block;
            if (block < 16 || block > most || block % 16 != 0 || !covers || n > 65536)
                return std::printf("%d rows, at most %d: %d blocks of %d\\n", rows, most, n, block), 1;
        }
    return std::puts("OK"), 0;
}
"""


def test_weight_rows(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(PROGRAM)
    res = subprocess.run([gxx, "-std=c++20", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{CSRC}", str(src),
                          "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout.strip() == "OK", res.stdout + res.stderr
