"""The registered backward operators of the linear layers compare their operands before anything is launched.  CPU tensors: those
that belong together are refused for their device, all others for what does not fit."""
import pytest
import torch

import transformer_amd  # noqa: F401  (registers the operators)
from transformer_amd import linear_ops

ops = torch.ops.mla_mi355x
BF = torch.bfloat16
M, N, K = 40, 24, 16


def z(*shape, dt=BF):
    return torch.zeros(*shape, dtype=dt)


def saved(blocks=1, m=M, n=N, dt=torch.uint8):
    return z(blocks * linear_ops._saved_size(m, n), dt=dt)


LINEAR = dict(dy=z(M, N), x=z(M, K), weight=z(N, K), saved=saved(), activation="silu", need_dx=True, need_dw=True,
              db_dtype=torch.float32)
GATED = dict(dy=z(M, K), x=z(M, K), w_gate=z(N, K), w_up=z(N, K), w_down=z(K, N), h=z(M, N), saved=saved(2), activation="silu",
             need_dx=True, need_gate=True, need_up=True, need_down=True)
BAD_LINEAR = {
    "dy narrower": dict(dy=z(M, 8)), "dy wider": dict(dy=z(M, 32)), "dy of fewer rows": dict(dy=z(M - 1, N)),
    "dy of another leading shape": dict(dy=z(2, M // 2, N)), "x narrower": dict(x=z(M, 8)), "x wider": dict(x=z(M, 24)),
    "x of more rows": dict(x=z(M + 1, K)), "x of another type": dict(x=z(M, K, dt=torch.float32)), "x a number": dict(x=torch.zeros((), dtype=BF)),
    "weight of three dimensions": dict(weight=z(1, N, K)), "weight of another type": dict(weight=z(N, K, dt=torch.float16)),
    "nothing saved": dict(saved=saved(0)), "saved for fewer rows": dict(saved=saved(m=32)),
    "saved of another type": dict(saved=z(linear_ops._saved_size(M, N), dt=torch.int8)),
    "saved with gaps": dict(saved=z(linear_ops._saved_size(M, N), 2, dt=torch.uint8)[:, 0]),
    "bias gradient of another type": dict(db_dtype=torch.float16), "activation": dict(activation="swish"),
}
BAD_GATED = {
    "dy narrower": dict(dy=z(M, 8)), "dy of fewer rows": dict(dy=z(8, K)), "x narrower": dict(x=z(M, 8)),
    "x and dy narrower": dict(x=z(M, 8), dy=z(M, 8)), "x of another type": dict(x=z(M, K, dt=torch.float32)),
    "w_up of fewer rows": dict(w_up=z(8, K)), "w_up narrower": dict(w_up=z(N, 8)), "w_down smaller": dict(w_down=z(K, 8)),
    "w_down not turned": dict(w_down=z(N, K)), "w_gate of three dimensions": dict(w_gate=z(1, N, K)),
    "w_down of another type": dict(w_down=z(K, N, dt=torch.float64)), "h narrower": dict(h=z(M, 8)), "h of fewer rows": dict(h=z(8, N)),
    "h with gaps": dict(h=z(M, 2 * N)[:, :N]), "h of another type": dict(h=z(M, N, dt=torch.float32)),
    "one of two saved": dict(saved=saved(1)), "saved of another type": dict(saved=saved(2, dt=torch.int8)),
    "saved with gaps": dict(saved=z(2 * linear_ops._saved_size(M, N), 2, dt=torch.uint8)[:, 0]), "activation": dict(activation="none"),
}


@pytest.mark.parametrize("bad", sorted(BAD_LINEAR))
def test_linear_act_bwd_refuses(bad):
    with pytest.raises((ValueError, TypeError), match="linear_act_bwd"):
        ops.linear_act_bwd(*{**LINEAR, **BAD_LINEAR[bad]}.values())


@pytest.mark.parametrize("bad", sorted(BAD_GATED))
def test_gated_ffn_bwd_refuses(bad):
    with pytest.raises((ValueError, TypeError), match="gated_ffn_bwd"):
        ops.gated_ffn_bwd(*{**GATED, **BAD_GATED[bad]}.values())


def test_what_belongs_together_is_refused_for_its_device_alone():
    for change in ({}, dict(dy=z(5, 8, N), x=z(5, 8, K)), dict(dy=z(M, N, dt=torch.float32)), dict(weight=z(N, K, dt=torch.float32)),
                   dict(activation="none", saved=saved(0))):
        with pytest.raises(RuntimeError, match="GPU"):
            ops.linear_act_bwd(*{**LINEAR, **change}.values())
    for change in ({}, dict(dy=z(5, 8, K), x=z(5, 8, K)), dict(w_down=z(K, N, dt=torch.float32))):
        with pytest.raises(RuntimeError, match="GPU"):
            ops.gated_ffn_bwd(*{**GATED, **change}.values())


def test_parts_of_a_weight_lie_within_the_kernels_reach():
    for rows in (8, 264, 1 << 14, 1 << 15, (1 << 20) - 8):
        for cols in (8, 264, 1 << 15, (1 << 20) - 8):
            n = linear_ops._columns(rows, cols)
            assert (rows + 64) * n < linear_ops.REACH  # (as mla_linear_dx and mla_gated_linear_bwd ask of a contiguous one)
            assert n == cols or (n >= 256 and n % 256 == 0 and (rows + 64) * cols >= linear_ops.REACH)


def test_a_bias_is_refused_off_its_alignment_or_in_another_type():
    import ctypes
    from tests.test_linear_args import BASE
    from transformer_amd import _lib
    lib, (struct, good) = _lib.load(), BASE["mla_linear_act"]
    for change in (dict(bias=4096, bias_dtype=2), dict(bias=4096, bias_dtype=-1), dict(bias=4104, bias_dtype=1),
                   dict(bias=4100, bias_dtype=0), dict(bias=4100, bias_dtype=1)):
        assert lib.mla_linear_act(ctypes.byref(struct(**{**good, **change})), None) < 0, change
        assert b"bias" in lib.mla_last_error()
