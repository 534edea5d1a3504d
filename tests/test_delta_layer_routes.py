"""The rule by which the gated delta rule cuts time (csrc/routes.hpp), on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include "routes.hpp"
int main(int, char** a) {
  if (a[3][0] == 's') std::printf("%d\n", ph::draw_split(std::atol(a[1]), std::atol(a[2])));
  else std::printf("%ld\n", ph::delta_segments(std::atol(a[1]), std::atol(a[2]), std::atoi(a[3])));
  return 0;
}
"""


@pytest.fixture(scope="module")
def segments(tmp_path_factory):
    d = tmp_path_factory.mktemp("delta_routes")
    (d / "drv.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "pufferlean_amd", "csrc"), "-o", str(d / "drv"),
                    str(d / "drv.cpp")], check=True)
    return lambda *args: int(subprocess.run([str(d / "drv")] + [str(x) for x in args], capture_output=True, text=True, check=True).stdout)


@pytest.mark.parametrize("chunks,units,P,n", [(1, 1, 32, 1), (7, 1, 64, 1), (8, 1, 64, 4), (9, 1, 32, 5), (256, 16, 64, 32), (32, 64, 64, 8), (32, 64, 32, 16),
                                              (64, 32, 128, 8), (2, 16384, 64, 1), (64, 512, 64, 1), (64, 257, 64, 1), (64, 256, 64, 2), (2 ** 26, 1, 64, 512)])
def test_segments(segments, chunks, units, P, n):
    assert segments(chunks, units, P) == n


def test_long_tests_reach_segments(segments):
    """The sequences of the GPU tests that are meant to be cut into segments are, in both types' chunks."""
    for T, units, P in ((300, 2, 32), (530, 2, 64), (515, 1, 128), (767, 1, 64), (410, 4, 32), (400, 8, 32), (600, 4, 32), (700, 36, 32)):
        for steps in (16, 32):
            assert segments(-(-T // steps), units, P) > 1


@pytest.mark.parametrize("N,A,split", [(1, 49151, 0), (1, 49152, 1), (128, 60001, 1), (129, 60001, 0), (4096, 1000, 0)])
def test_wide_rows_of_the_draw(segments, N, A, split):
    assert segments(N, A, "s") == split
