"""Calls of the linear layers' operators that their documentation allows or refuses, beside the numerics of test_gpu_feedforward.py.
Bounds as derived there."""
import pytest
import torch

from tests import test_gpu_feedforward as T
from tests import test_linear_bwd_args as A

pytestmark = pytest.mark.gpu


def test_backward_operators_refuse_what_does_not_belong_together():
    ops = torch.ops.mla_mi355x
    cuda = lambda d: {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    for op, good, bad in ((ops.linear_act_bwd, A.LINEAR, A.BAD_LINEAR), (ops.gated_ffn_bwd, A.GATED, A.BAD_GATED)):
        want = op(*cuda(good).values())
        for name, change in bad.items():
            if name in ("saved with gaps", "h with gaps"):
                continue  # (a copy to the GPU has none)
            with pytest.raises((ValueError, TypeError)):
                op(*{**cuda(good), **cuda(change)}.values())
        for name in good:  # one of them elsewhere
            if isinstance(good[name], torch.Tensor):
                with pytest.raises(RuntimeError):
                    op(*{**cuda(good), name: good[name]}.values())
        assert all(torch.equal(a, c) for a, c in zip(op(*cuda(good).values()), want))
