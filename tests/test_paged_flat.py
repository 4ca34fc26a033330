"""The flat copies of the paged tile pass stay inside the 16 rows that they copy: the rule of
csrc/paged_flat.h, compiled for the host and walked for every head dimension that takes it."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include "paged_flat.h"
int main() {
  for (int D = 4; D <= 124; D += 8) {
    const int nk = lb::flat_chunks(D);
    for (int u = 0; u < lb::flat_copies(nk); ++u)
      for (int lane = 0; lane < 32; ++lane)
        if (lb::flat_copied(nk, D, u, lane)) std::printf("%d %d %d %d\n", D, nk, lb::flat_most_d(nk), 16 * (32 * u + lane));
  }
}
"""


@pytest.fixture(scope="module")
def copies(tmp_path_factory):
    """{D: (chunks, largest D of the kernel, [first byte of every piece copied])}"""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("flat")
    (at / "walk.cc").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", os.path.join(ROOT, "lucid_b200", "csrc"), str(at / "walk.cc"), "-o",
                    str(at / "walk")], check=True, timeout=300)
    out = subprocess.run([str(at / "walk")], check=True, capture_output=True, text=True, timeout=60).stdout
    got = {}
    for line in out.splitlines():
        D, nk, most, byte = map(int, line.split())
        got.setdefault(D, (nk, most, []))[2].append(byte)
    return got


@pytest.mark.parametrize("D", range(4, 128, 8))     # odd multiples of 4 up to 124
def test_a_flat_run_is_copied_once_and_nothing_past_it(copies, D):
    nk, most, at = copies[D]
    assert 4 * 4 * nk >= D and D <= most            # 4 nk chunks of 4 elements cover a row
    assert at == list(range(0, 32 * D, 16))
