"""What the tiled prompt attention computes on plain numbers (csrc/paged.cuh), on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen3-tts-rsi-engine_b200" / "csrc"


def run(tmp_path, program):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("g++ not found")
    source, binary = tmp_path / "program.cpp", tmp_path / "program"
    source.write_text(program)
    build = subprocess.run([compiler, "-std=c++17", "-O1", "-ffp-contract=off", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall",
                            "-I", str(CSRC), str(source), "-o", str(binary)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    done = subprocess.run([str(binary)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout.split()


def test_sequences_are_found_through_groups(tmp_path):
    """Every call looks at 512 sequences at most for an item, of the 2^20 that it may have; up to 2048 at one."""
    out = run(tmp_path, r"""
#include <stdio.h>
#include <initializer_list>
#include "paged.cuh"
int main() {
  for (int64_t n : {1, 31, 2048, 2049, 4096, 4097, 5000, 100000, 1048575, 1048576}) {
    const int shift = q3t::group_shift(n, 2048), groups = q3t::groups_of(n, shift);
    if (groups > 2048 || (int64_t(groups) << shift) < n || (int64_t(groups - 1) << shift) >= n) return 1;
    printf("%d ", shift);
  }
  return 0;
}
""")
    assert [int(v) for v in out] == [0, 0, 0, 1, 1, 2, 2, 6, 9, 9]
