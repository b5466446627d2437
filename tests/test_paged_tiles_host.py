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


def test_the_polynomial_exponential(tmp_path):
    """2^x as the tiled kernel computes it, in fp32 operations: 2^-18.3 relative where the result is a normal number (the fit's
    own 2^-18.4, the last rounding's 2^-24, a quarter of that from the one before), 2^-126 below, and exactly 0 from -127 down."""
    relative, absolute = (float(v) for v in run(tmp_path, r"""
#include <initializer_list>
#include <math.h>
#include <stdio.h>
#include <string.h>
struct float2 { float x, y; };
namespace q3t {
float2 fma2(float2 a, float2 b, float2 c) { return {fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)}; }
float2 add2(float2 a, float2 b) { return {a.x + b.x, a.y + b.y}; }
}
#include "exp2_poly.cuh"
int main() {
  double relative = 0, absolute = 0;
  auto check = [&](float x) {
    const float2 y = q3t::exp2_poly(float2{x, x});
    const double want = exp2(double(x)), off = fabs(y.x - want);
    if (y.x != y.y) relative = 1;
    if (want >= 0x1p-126 && off / want > relative) relative = off / want;
    if (want < 0x1p-126 && off > absolute) absolute = off;
  };
  for (unsigned bits = 0x30000000; bits < 0x42fe0001; bits += 61) {   // 2^-31 .. 127, both signs
    float x;
    memcpy(&x, &bits, 4);
    check(x < 127.f ? x : 126.5f);
    check(-x);
  }
  for (float x : {0.f, -0.f, 0.5f, -0.5f, 1.5f, -1.5f, -126.f, -126.5f, -127.f, 126.f, 126.49999f}) check(x);
  for (float x : {-127.f, -127.5f, -1e4f, -3e38f, -INFINITY, NAN}) {
    const float2 y = q3t::exp2_poly(float2{x, 0.f});
    if (y.x != 0.f || signbit(y.x) || y.y != 1.f) relative = 2;
  }
  printf("%.9e %.9e", relative, absolute);
  return 0;
}
"""))
    assert 2 ** -19 < relative < 2 ** -18.3 and absolute < 2 ** -126
