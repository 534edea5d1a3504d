"""The rules by which the state-space policy layer's operators choose their kernels (csrc/routes.hpp), on the host."""
import os
import subprocess

import pytest
import torch

import test_gpu_ffn as ffn
import test_gpu_ssm as ssm

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
  if (!std::strcmp(argv[1], "ssm_chunk")) r = ssm_chunk(a[0], a[1], a[2], a[3], (int)a[4], a[5]);
  if (!std::strcmp(argv[1], "ssm_block_threads")) r = ssm_block_threads(a[0], (int)a[1], a[2]);
  if (!std::strcmp(argv[1], "glu_tile")) r = glu_tile(a[0], a[1], a[2], a[3], a[4], a[5]);
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


@pytest.mark.parametrize("T,C,N,G,K,dt,gate", ssm.CHUNKED)
def test_ssm_tests_reach_chunks(route, T, C, N, G, K, dt, gate):
    """Their episodes end around the borders of chunks of 32 steps, in both directions."""
    for grad in (0, 1):
        assert route("ssm_chunk", T, 3, G, C // G, N, grad) == 32 < T


def test_ssm_tests_reach_every_last_chunk(route):
    assert {T % 32 for T, *_ in ssm.CHUNKED} >= {0, 1, 2, 3, 6, 7} and {K for _, _, _, _, K, *_ in ssm.CHUNKED} == set(range(5))
    # blocks of one and of several channel blocks, and of one and four wavefronts
    blocks = [(route("ssm_block_threads", C // G, (N + 3) // 4, 1), C // G) for _, C, N, G, *_ in ssm.CHUNKED]
    assert {nt for nt, _ in blocks} >= {64, 128, 256} and any(nt < per for nt, per in blocks)
    for T in (150, 300):
        assert route("ssm_chunk", T, 3, 1, 40, 16, 0) == 32


# (T, B, G, channels of a group, states, gradient) and the steps of a chunk
@pytest.mark.parametrize("T,B,G,per,N,grad,chunk", [(128, 1, 1, 64, 16, 0, 128), (129, 1, 1, 64, 16, 0, 32), (64, 1, 1, 64, 16, 1, 64),
                                                    (65, 1, 1, 64, 16, 1, 24), (8192, 2, 1, 512, 16, 0, 64), (2048, 8, 2, 192, 16, 1, 64),
                                                    (33, 203, 1, 96, 5, 1, 40), (64, 2048, 1, 512, 16, 1, 64), (1, 1, 1, 1, 1, 0, 8)])
def test_ssm_chunk(route, T, B, G, per, N, grad, chunk):
    assert route("ssm_chunk", T, B, G, per, N, grad) == chunk


TILES = ("64", "128", "256x128", "256")


@pytest.mark.parametrize("M,Dm,F,dt,units,grad", ffn.LARGE)
def test_ffn_tests_reach_their_tiles(route, M, Dm, F, dt, units, grad):
    bf, up = dt is torch.bfloat16, lambda n: (n + 7) // 8 * 8
    assert M > 64  # fewer rows have kernels of their own
    assert TILES[route("glu_tile", bf, 1, M, 2 * up(F), up(Dm), up(Dm))] == units
    nt = M >= 2048  # from there on the gradient's product takes transposed weights
    assert TILES[route("glu_tile", bf, nt, M, up(F), up(Dm), up(Dm) if nt else up(F))] == grad


@pytest.mark.parametrize("bf,nt,M,N,ld,tile", [(1, 1, 65536, 2752, 512, "256"), (1, 1, 65536, 1376, 512, "256x128"), (1, 1, 2048, 16384, 16, "256"),
                                               (1, 1, 2048, 16384, 2 ** 23 + 8, "128"), (1, 0, 65536, 2752, 512, "128"),
                                               (1, 1, 2048, 1024, 512, "128"), (1, 1, 300, 256, 128, "64"), (0, 1, 6699, 1072, 208, "64"),
                                               (0, 1, 65536, 512, 512, "128")])
def test_glu_tile(route, bf, nt, M, N, ld, tile):
    assert TILES[route("glu_tile", bf, nt, M, N, ld, ld)] == tile
