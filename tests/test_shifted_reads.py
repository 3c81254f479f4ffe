"""The weights of a norm over packed rows of odd width, without a GPU: the kernel's own index
arithmetic compiled for the host, every read checked against the vector's bounds."""
from __future__ import annotations

import os
import subprocess

import pytest

from tests.conftest import ROOT

HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#include "shifted.cuh"
int main(int argc, char** argv) {
  long outside = 0, wrong = 0, calls = 0;
  for (int a = 1; a < argc; ++a) {
    const int n = atoi(argv[a]);
    auto load8 = [&](int j, float* v) {
      if (j < 0 || j % 8 || j + 8 > n) ++outside;
      for (int e = 0; e < 8; ++e) v[e] = j + e;
    };
    auto load1 = [&](int j) {
      if (j < 0 || j >= n) ++outside;
      return static_cast<float>(j);
    };
    for (int row = 0; row < 8; ++row) {  // every shift that rows of n values have
      const int shift = row * n & 7;
      for (int g = 0; g * 8 - shift < n; ++g, ++calls) {
        const int i = g * 8 - shift;
        float w[8];
        ggufmm::shifted8(i, shift, n, load8, load1, w);
        for (int e = 0; e < 8; ++e)
          if (i + e >= 0 && i + e < n && w[e] != i + e) ++wrong;
      }
    }
  }
  std::printf("%ld %ld %ld\n", outside, wrong, calls);
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    d = tmp_path_factory.mktemp("shifted")
    (d / "harness.cpp").write_text(HARNESS)
    csrc = os.path.join(ROOT, "vllm-webgpu_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", csrc, str(d / "harness.cpp"), "-o", str(d / "harness")], check=True)
    return str(d / "harness")


@pytest.mark.parametrize("widths", [range(8, 300), [2815, 4095, 9001], range(16353, 16369)], ids=["small", "odd", "widest"])
def test_no_read_outside_the_weights(harness, widths):
    out = subprocess.run([harness, *map(str, widths)], check=True, capture_output=True, text=True).stdout
    outside, wrong, calls = map(int, out.split())
    assert (outside, wrong) == (0, 0) and calls > len(list(widths))
