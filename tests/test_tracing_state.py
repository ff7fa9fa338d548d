"""What decides between an operator's body and the registered operator sees torch.jit.trace: a body's launch is not recorded."""
import pytest
import torch

from transformer_amd import kernels


def test_a_jit_trace_is_not_a_plain_call():
    seen = []

    def f(t):
        seen.append((kernels._not_plain(()), kernels.dispatcher_needed(()), kernels.function_fits(())))
        return t + 1

    with torch.no_grad():
        torch.jit.trace(f, torch.zeros(2), check_trace=False)
    assert seen == [(True, True, False)]
    assert not kernels._not_plain(()) and kernels.function_fits(())


def test_the_clipping_refuses_a_jit_trace():
    from transformer_amd import clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(2))
    p.grad = torch.ones(2)
    for f in (lambda t: grad_norm([t]), lambda t: clip_grad_norm_([p], 1.0)):
        with pytest.raises(RuntimeError, match="jit.trace"):
            torch.jit.trace(f, torch.zeros(2), check_trace=False)
        with pytest.raises(RuntimeError, match="GPU"):
            f(torch.zeros(2))
    assert torch.equal(p.grad, torch.ones(2))
