"""Which tiles the linear layers take by size (csrc/plans.h), so that the GPU tests' sizes are known to reach both, whole and cut."""
import ctypes
import functools
import os
import subprocess
import tempfile
from collections import namedtuple

import pytest

from tests import test_gpu_feedforward as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
Plan = namedtuple("Plan", "large S per part_bytes")


@functools.lru_cache(None)
def _lib():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "p.cpp"), os.path.join(d, "p.so")
        with open(src, "w") as f:
            f.write('#include "plans.h"\nextern "C" void plan(int64_t M, int64_t N, int64_t K, int64_t parts, int cut, int64_t* o) '
                    "{ const mla::GemmPlan p = mla::gemm_plan(M, N, K, parts, cut != 0); "
                    "o[0] = p.large, o[1] = p.S, o[2] = p.per, o[3] = p.part_bytes; }\n")
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "transformer_amd", "csrc"), src,
                        "-o", out], check=True)
        return ctypes.CDLL(out)


def plan(M, N, K, parts=1, cut=True):
    o = (ctypes.c_int64 * 4)()
    _lib().plan(*(ctypes.c_int64(s) for s in (M, N, K, parts)), int(cut), o)
    return Plan(*o)


def linear(M, N, K):
    return plan(M, N, K)


def gated(M, H, D):
    return plan(M, 2 * H, D, cut=False)


def dx(M, N, K, parts):
    """of a layer [N, K], or of two"""
    return plan(M, K, N, parts)


def test_the_gpu_tests_reach_both_tiles_whole_and_cut():
    assert all(not p.large for M, N, K in T.SIZES for p in (linear(M, N, K), gated(M, N, K), dx(M, N, K, 1), dx(M, N, K, 2)))
    assert linear(1000, 264, 1800).S > 1 and dx(300, 1000, 64, 1).S > 1 and dx(300, 1000, 64, 2).S > 1  # small tiles, cut
    assert dx(65, 264, 128, 2).S == 1
    whole, ragged, wide, both, cut = T.LARGE
    assert all(p.large and p.S == 1 for p in (linear(*whole), gated(*whole), linear(*ragged), gated(*ragged), dx(*wide, 1),
                                              dx(*wide, 2)))
    assert linear(*cut).large and linear(*cut).S > 1
    assert dx(*both, 2).large and dx(*both, 2).S > 1


@pytest.mark.parametrize("cut", [False, True])
def test_plans_hold_their_own_terms(cut):
    """Pieces cover every stage, each has one, there are no more pieces than one round runs, and the partials fit 64 MB."""
    for M in (1, 65, 127, 1000, 4096, 12288, 100000):
        for N in (8, 264, 1792, 4608, 9216):
            for K in (8, 64, 72, 1000, 1792, 9216):
                for parts in (1, 2):
                    p = plan(M, N, K, parts, cut)
                    n = (K + 63) // 64 * parts
                    T_, slots = (256, 256) if p.large else (128, 512)
                    tiles = -(-M // T_) * -(-N // T_)
                    assert p.S >= 1 and (p.S - 1) * p.per < n <= p.S * p.per
                    if p.S > 1:
                        assert cut and 0 < tiles % slots * p.S <= slots
                        assert p.part_bytes == tiles % slots * p.S * T_ * T_ * 4 <= 64 << 20
                    else:
                        assert p.part_bytes == 0
