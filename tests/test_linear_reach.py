"""Which kernels the GPU tests' sizes reach, product by product, where their results are compared with 64 bits."""
import ctypes
import functools
import os
import subprocess
import tempfile

from tests import test_gemm_plan as P
from tests import test_gpu_feedforward as T
from tests import test_gpu_linear_edges as E
from tests import test_gpu_linear_wide as W

EVERY = {(t, c) for t in P.TILES for c in (False, True)}


@functools.lru_cache(None)
def _lib():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "r.cpp"), os.path.join(d, "r.so")
        with open(src, "w") as f:
            f.write('#include "plans.h"\nextern "C" int columns(int64_t N) { return mla::rows_columns(N); }\n')
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(P.ROOT, "transformer_amd", "csrc"), src,
                        "-o", out], check=True)
        return ctypes.CDLL(out)


def tiles(of, sizes):
    return {(p.tile, p.S > 1) for p in (of(*s) for s in sizes if s[0] > 64)}


def rows(of, sizes):
    """(blocks of 16 rows, columns of a workgroup) of the few-row kernels."""
    return {(1 if M <= 16 else 2 if M <= 32 else 4, _lib().columns(ctypes.c_int64(of(M, N, K)))) for M, N, K in sizes if M <= 64}


def test_results_are_compared_on_every_tile_of_every_product():
    results = T.SIZES + E.TILES + T.LARGE  # (the last by test_results_of_large_tiles)
    assert tiles(P.linear, results) == EVERY
    assert tiles(P.gated, results) == EVERY
    assert tiles(lambda M, H, D: P.plan(M, D, H), results) == EVERY  # the gated block's second product
    gradients = T.SIZES + T.LARGE + E.TILES
    for parts in (1, 2):
        assert tiles(lambda M, N, K: P.dx(M, N, K, parts), gradients) == EVERY


def test_results_are_compared_on_every_few_row_kernel():
    every = {(b, c) for b in (1, 2, 4) for c in (16, 32)}
    assert rows(lambda M, N, K: N, T.SIZES + W.ROWS) == every           # linear_act's, and the gated block's first products
    assert rows(lambda M, N, K: K, T.SIZES + W.ROWS + W.DOWN) == every  # its second one
    wide = [s for s in W.ROWS if s[1] > 4096]
    assert {s[1] % 32 for s in wide} == {0, 8, 16, 24} and any(s[2] > 2048 for s in wide) and any(s[2] % 256 for s in wide)
