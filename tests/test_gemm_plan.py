"""Which tiles the linear layers take by size (csrc/plans.h), so that the GPU tests' sizes are known to reach both."""
import ctypes
import functools
import os
import subprocess
import tempfile

from tests import test_gpu_feedforward as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@functools.lru_cache(None)
def _lib():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "p.cpp"), os.path.join(d, "p.so")
        with open(src, "w") as f:
            f.write('#include "plans.h"\nextern "C" int large(int64_t M, int64_t N, int64_t K, int64_t parts) '
                    "{ return mla::gemm_plan(M, N, K, parts).large; }\n")
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "transformer_amd", "csrc"), src,
                        "-o", out], check=True)
        return ctypes.CDLL(out)


def large(*sizes):
    return bool(_lib().large(*(ctypes.c_int64(s) for s in sizes)))


def test_the_gpu_tests_reach_both_tiles():
    for M, H, D in T.SIZES:
        assert not large(M, 2 * H, D, 1) and not large(M, D, H, 1) and not large(M, D, H, 2)
    for M, N, K in T.LARGE[:2]:
        assert large(M, N, K, 1) and large(M, 2 * N, K, 1), (M, N, K)  # linear_act and gated_linear_bwd; gated_linear
    M, N, K = T.LARGE[2]
    assert large(M, K, N, 1) and large(M, K, N, 2)  # linear_dx of one layer and of two
