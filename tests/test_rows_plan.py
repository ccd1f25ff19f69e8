"""How swamp_gemm_rows_i8 cuts a call (csrc/rows_plan.hpp, built for the host), without a GPU:
which tile the sizes of the GPU's tests take, and that every plan is sound."""
import ctypes
import os
import random
import subprocess

import pytest

from rows_plan_sizes import ONE, PIECES

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256  # MI355X

SHIM = """
#include "rows_plan.hpp"
extern "C" void plan(int m, int n, int k, int cus, int *o) {
  const swamp_rows::Plan p = swamp_rows::plan_of(m, n, k, cus);
  o[0] = p.shape; o[1] = p.tiles_m; o[2] = p.tiles_n; o[3] = p.pieces; o[4] = p.steps;
  o[5] = p.shape < 0 ? 0 : swamp_rows::kTiles[p.shape].tm;
  o[6] = p.shape < 0 ? 0 : swamp_rows::kTiles[p.shape].tn;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("rows_plan")
    src, so = str(d / "plan.cpp"), str(d / "plan.so")
    with open(src, "w") as f:
        f.write(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    "-I" + os.path.join(REPO, "llamanyon.rs_amd", "csrc"), src, "-o", so],
                   check=True)
    lib = ctypes.CDLL(so)

    def of(m, n, k, cus=CUS):
        o = (ctypes.c_int * 7)()
        lib.plan(m, n, k, cus, o)
        return tuple(o)

    return of


def test_tiles_of_the_tested_sizes(plan):
    for sizes, split in ((ONE, False), (PIECES, True)):
        for tile, each in sizes.items():
            for m, n, k in each:
                shape, _, _, pieces, _, tm, tn = plan(m, n, k)
                assert shape >= 0 and (tm, tn) == tile and (pieces > 1) == split, (m, n, k, tm, tn, pieces)
    # every tile: whole and ragged, odd and even steps, the stages round several times
    for tile, each in ONE.items():
        whole = [m % tile[0] == 0 and n % tile[1] == 0 for m, n, _ in each]
        steps = [-(-k // 64) for *_, k in each]
        assert any(whole) and not all(whole) and len({s % 2 for s in steps}) == 2, tile
        assert max(steps) >= 15 and any(k % 64 for *_, k in each), tile


def test_plans_are_sound(plan):
    """Tiles cover the result, pieces the sum, none of them empty, and a launch holds less than
    2^32 threads."""
    rng = random.Random(3)
    sizes = [(1 << 30, 1, 131071), (1, 1 << 30, 64), (64, 1 << 30, 16), (100, 1 << 30, 16),
             (1 << 30, 255, 16), (1 << 19, (1 << 19) - 1, 64), (17, 1 << 28, 512)]
    for few in (1, 17, 65, 127, 129, 255, 257, 513, 1025, 4097):
        many = min(1 << 30, ((1 << 38) - 1) // few)
        sizes += [(few, many, 16), (many, few, 16), (few, many, 131071), (many, few, 131071)]
    for _ in range(4000):
        m, n = (int(2 ** rng.uniform(0, 20)) for _ in range(2))
        sizes.append((m, n, int(2 ** rng.uniform(0, 17)) % 131072 or 1))
    for m, n, k in sizes:
        if m * n >= 1 << 38:
            continue
        for cus in (CUS, 64, 304):
            shape, tiles_m, tiles_n, pieces, steps, tm, tn = plan(m, n, k, cus)
            total = -(-k // 64)
            if shape < 0:
                assert m <= 64 and tiles_n in (1, 2, 4) and pieces == 1, (m, n, k)
                assert (m <= 16 or -(-n // (16 * tiles_n)) <= cus) and (m <= 32 or tiles_n <= 2), (m, n, k)
                continue
            assert tiles_m == -(-m // tm) and tiles_n == -(-n // tn), (m, n, k)
            assert 1 <= pieces <= 8 and (pieces - 1) * steps < total <= pieces * steps, (m, n, k)
            assert steps % 2 == 0 or pieces == 1, (m, n, k)
            threads = 256 if (tm, tn) == (64, 128) else 512
            assert tiles_m * tiles_n * pieces * threads < 1 << 32, (m, n, k)
            # partial sums: none but where tiles are few
            assert pieces == 1 or tiles_m * tiles_n * pieces <= 3 * cus, (m, n, k)
