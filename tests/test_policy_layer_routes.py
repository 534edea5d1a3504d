"""The rules by which the state-space policy layer's operators choose their kernels (csrc/routes.hpp), on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "routes.hpp"
using namespace ph;
int main(int argc, char** argv) {
  long a[8] = {};
  for (int i = 2; i < argc && i < 10; i++) a[i - 2] = std::atol(argv[i]);
  long r = -1;
  if (!std::strcmp(argv[1], "dma_offsets_fit")) r = dma_offsets_fit(a[0], a[1], a[2]);
  std::printf("%ld\n", r);
  return 0;
}
"""


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    d = tmp_path_factory.mktemp("policy_layer_routes")
    (d / "drv.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "pufferlean_amd", "csrc"),
                    "-o", str(d / "drv"), str(d / "drv.cpp")], check=True)

    def call(name, *args):
        out = subprocess.run([str(d / "drv"), name] + [str(int(x)) for x in args], capture_output=True, text=True, check=True)
        return int(out.stdout)
    return call


def test_dma_offsets_fit(route):
    """The largest leading dimension that passes keeps the last element of a tile within 31 bits, in either operand: row 255 and
    the row's last k (NT), row 31 and the tile's last column (TN)."""
    for tn, rows in ((0, 256), (1, 32)):
        most = 2 ** 31 // rows
        assert route("dma_offsets_fit", tn, most, 8) and route("dma_offsets_fit", tn, 8, most)
        assert not route("dma_offsets_fit", tn, most + 8, 8) and not route("dma_offsets_fit", tn, 8, most + 8)
        last = (rows - 1) * most + (255 if tn else most - 1)
        assert last < 2 ** 31
