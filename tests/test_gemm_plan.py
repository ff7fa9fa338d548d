"""Which tiles the linear layers take by size (csrc/plans.h), so that the GPU tests' sizes are known to reach each, whole and cut."""
import ctypes
import functools
import os
import subprocess
import tempfile
from collections import namedtuple

from tests import test_gpu_feedforward as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
Plan = namedtuple("Plan", "tile S per part_bytes")
SMALL, HALF, LARGE = range(3)
TILES = {SMALL: (128, 128, 512), HALF: (256, 128, 256), LARGE: (256, 256, 256)}  # m, n, at once


@functools.lru_cache(None)
def _lib():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "p.cpp"), os.path.join(d, "p.so")
        with open(src, "w") as f:
            f.write('#include "plans.h"\nextern "C" void plan(int64_t M, int64_t N, int64_t K, int64_t parts, int64_t* o) '
                    "{ const mla::GemmPlan p = mla::gemm_plan(M, N, K, parts); "
                    "o[0] = p.tile, o[1] = p.S, o[2] = p.per, o[3] = p.part_bytes; }\n")
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "transformer_amd", "csrc"), src,
                        "-o", out], check=True)
        return ctypes.CDLL(out)


def plan(M, N, K, parts=1):
    o = (ctypes.c_int64 * 4)()
    _lib().plan(*(ctypes.c_int64(s) for s in (M, N, K, parts)), o)
    return Plan(*o)


def linear(M, N, K):
    return plan(M, N, K)


def gated(M, H, D):
    return plan(M, 2 * H, D)


def dx(M, N, K, parts):
    """of a layer [N, K], or of two"""
    return plan(M, K, N, parts)


def test_the_gpu_tests_reach_every_tile_whole_and_cut():
    from tests.test_gpu_linear_edges import TILES as more
    sizes = T.SIZES + T.LARGE + more
    for of in (linear, gated, lambda M, N, K: dx(M, N, K, 1), lambda M, N, K: dx(M, N, K, 2)):
        assert {(p.tile, p.S > 1) for p in (of(*s) for s in sizes)} == {(t, c) for t in TILES for c in (False, True)}


def test_plans_hold_their_own_terms():
    """Pieces cover every stage, each has one, there are no more pieces than one round runs, and the partials fit 64 MB."""
    for M in (1, 65, 127, 1000, 4096, 12288, 100000):
        for N in (8, 264, 1792, 4608, 9216):
            for K in (8, 64, 72, 1000, 1792, 9216):
                for parts in (1, 2):
                    p = plan(M, N, K, parts)
                    n = (K + 63) // 64 * parts
                    m_, n_, slots = TILES[p.tile]
                    tiles = -(-M // m_) * -(-N // n_)
                    assert p.S >= 1 and (p.S - 1) * p.per < n <= p.S * p.per
                    if p.S > 1:
                        assert 0 < tiles % slots * p.S <= slots
                        assert p.part_bytes == tiles % slots * p.S * m_ * n_ * 4 <= 64 << 20
                    else:
                        assert p.part_bytes == 0
