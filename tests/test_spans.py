"""Whether strided arrays share elements (csrc/spans.hpp), on the host: against the sets of their bytes."""
import itertools
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r"""
#include <cstdio>
#include "spans.hpp"
static bool get(ph::Span& s) {
  long p;
  if (std::scanf("%ld %ld", &p, &s.w) != 2) return false;
  s.p = (const void*)p;
  for (int i = 0; i < 3; i++)
    if (std::scanf("%ld %ld", &s.n[i], &s.s[i]) != 2) return false;
  return true;
}
int main() {
  ph::Span a, b;
  while (get(a) && get(b)) std::printf("%d %d\n", ph::meet(a, b), ph::folds(a));
  return 0;
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("spans")
    (d / "drv.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "pufferlean_amd", "csrc"), "-o", str(d / "drv"),
                    str(d / "drv.cpp")], check=True)

    def run(pairs):
        text = "\n".join(" ".join(str(x) for p, w, dims in pair for x in (p, w, *itertools.chain(*dims))) for pair in pairs)
        out = subprocess.run([str(d / "drv")], input=text, capture_output=True, text=True, check=True).stdout.split()
        return list(zip(map(int, out[::2]), map(int, out[1::2])))
    return run


def elements(p, w, dims):
    return [p + sum(i * s for i, (_, s) in zip(idx, dims)) + x for idx in itertools.product(*(range(n) for n, _ in dims)) for x in range(w)]


def test_against_the_bytes(ask):
    r = random.Random(3)
    pairs = []
    for _ in range(4000):
        pair = []
        for _ in range(2):
            kind = r.random()
            if kind < 0.6:  # nested, as slices of one buffer are
                w = r.randint(1, 5)
                dims, s = [], w + r.randint(0, 8)
                for _ in range(3):
                    n = r.randint(1, 4)
                    dims.append((n, s))
                    s = s * n + r.randint(0, 6)
                r.shuffle(dims)
            else:
                w, dims = r.randint(1, 6), [(r.randint(1, 4), r.randint(-20, 20)) for _ in range(3)]
            pair.append((1000 + r.randint(0, 90), w, dims))
        pairs.append(pair)
    for pair, (meets, folds) in zip(pairs, ask(pairs)):
        a, b = (elements(*x) for x in pair)
        assert meets == bool(set(a) & set(b)), pair
        assert folds == (len(set(a)) < len(a)), pair


def test_large_arrays(ask):
    """Columns of a wide time-major buffer, of batch-major ones, one element too far, and with nothing in them."""
    T, B, C = 1 << 20, 512, 1000
    col = lambda at, w, lead=((T, B * C * 2), (B, C * 2)), h=(1, 0): (1 << 40 | at * 2, w * 2, [*lead, h])
    batch = ((T, C * 2), (B, T * C * 2))
    pairs = [(col(0, 64), col(64, 64)), (col(0, 65), col(64, 64)), (col(0, 64, batch), col(64, 936, batch)), (col(0, 64, batch), col(64, 937, batch)),
             (col(0, 16, h=(4, 128)), col(16, 16, h=(4, 128))), (col(0, 16, h=(4, 128)), col(15, 16, h=(4, 128))),
             (col(0, 64), col(64 + C * B * (T - 1), 64)), (col(0, 64), col(C * B * T, 64)), (col(0, 64), col(0, 0)),
             (col(0, 64), (0, 64, [(1, 0)] * 3)), (col(0, 64, ((T, 0), (B, C * 2))), col(5, 1))]
    got = ask(pairs)
    assert [m for m, _ in got] == [0, 1, 0, 1, 0, 1, 0, 0, 0, 0, 1]
    assert [f for _, f in got] == [0] * 10 + [1]
