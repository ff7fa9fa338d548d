"""linear_act and gated_ffn at sizes that the forward tests of test_gpu_feedforward.py leave out, with its bounds: few rows against
more than 4096 columns, results of 256 x 256 tiles whole and cut along k (tests/test_linear_reach.py asserts which kernels the sizes
reach)."""
import pytest

from tests import test_gpu_feedforward as T

pytestmark = pytest.mark.gpu

# rows, columns with remainders of 8, 16 and 24 of a workgroup's 32 and none, k below and past the ring's chunks of 256
ROWS = [(M, N, K) for M, K in ((1, 40), (7, 2312), (16, 264), (17, 1800), (32, 520), (33, 264), (50, 2568), (64, 1800))
        for N in (4104, 4112, 4120, 4608)] + [(1, 8200, 4616), (64, 9240, 72), (33, 20000, 264)]
# the gated block's second product with as many columns
DOWN = [(M, 264, D) for M in (1, 17, 64) for D in (4104, 4120, 4608)]


@pytest.mark.parametrize("M,N,K", ROWS)
def test_few_rows_against_many_columns(M, N, K):
    for act in ("none", "relu", "silu", "gelu_tanh"):
        T.test_linear_act_forward(M, N, K, True, act != "relu", act)
        T.test_linear_act_gradients(M, N, K, act)  # (they read what the forward kept)
        if act != "none":
            T.test_gated_ffn_forward(M, N, K, act != "relu", act)
            T.test_gated_ffn_gradients(M, N, K, act)


@pytest.mark.parametrize("M,H,D", DOWN)
def test_few_rows_back_to_many_columns(M, H, D):
    T.test_gated_ffn_forward(M, H, D, True, "silu")
    T.test_gated_ffn_gradients(M, H, D, "silu")


@pytest.mark.parametrize("M,N,K", T.LARGE)
def test_results_of_large_tiles(M, N, K):
    for act in ("none", "relu", "silu", "gelu_tanh"):
        T.test_linear_act_forward(M, N, K, True, True, act)
        if act != "none":
            T.test_gated_ffn_forward(M, N, K, True, act)
    T.test_linear_act_forward(M, N, K, False, False, "silu")
    T.test_gated_ffn_forward(M, N, K, False, "silu")
