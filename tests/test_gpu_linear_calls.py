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


class _Call(torch.nn.Module):
    def __init__(self, layer, f):
        super().__init__()
        self.layer, self.f = layer, f

    def forward(self, x):
        return self.f(self.layer, x)


def test_a_jit_trace_records_the_operators():
    """Replayed on other inputs, with what the trace's own outputs held overwritten, a trace gives the eager call's result."""
    from transformer_amd import MLA, ModelArgs, RMSNorm, SwiGLU, chunked_linear_cross_entropy, gated_ffn, linear_act
    torch.manual_seed(0)
    g = T.gen("trace")
    w, wd, b, r = T.bf16(g, 136, 72, std=0.1), T.bf16(g, 72, 136, std=0.1), T.bf16(g, 136), T.bf16(g, 40, 136)
    with torch.device("cuda"):
        ffn, norm = SwiGLU(72, 136).bfloat16().requires_grad_(False), RMSNorm(72).requires_grad_(False)
        mla = MLA(ModelArgs(d_model=256, n_heads=2, max_seq_len=128)).bfloat16().requires_grad_(False)
    vocab, targets = T.bf16(g, 64, 72), torch.randint(0, 64, (1, 40), generator=g, device="cuda")
    calls = [
        ("linear_act", None, lambda _, x: linear_act(x, w, b, r, "silu"), (40, 72)),
        ("gated_ffn", None, lambda _, x: gated_ffn(x, w, w, wd, x), (40, 72)),
        ("SwiGLU", ffn, lambda m, x: m(x), (40, 72)),
        ("RMSNorm", norm, lambda m, x: m(x), (40, 72)),
        ("loss", None, lambda _, x: chunked_linear_cross_entropy(x, vocab, targets, 32), (1, 40, 72)),
        ("MLA", mla, lambda m, x: m(x)[0], (1, 40, 256)),
        ("MLA, a chunk", mla, lambda m, x: m(x, None, True)[0], (1, 40, 256)),
        ("MLA, one token", mla, lambda m, x: m(x, None, True)[0], (2, 1, 256)),
    ]
    with torch.no_grad():
        for name, layer, f, shape in calls:
            call = _Call(layer, f)
            x = T.bf16(g, *shape)
            call(x)
            traced = torch.jit.trace(call, x, check_trace=False)
            for _ in range(2):
                x = T.bf16(g, *shape)
                junk = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 8, 1 << 12, 1 << 16, 1 << 20) for _ in range(4)]
                del junk
                got, want = traced(x), call(x)
                assert torch.equal(got, want), name
    # with gradients: the operators have their own under a trace
    x = T.bf16(g, 40, 72).requires_grad_()
    traced = torch.jit.trace(_Call(None, lambda _, t: gated_ffn(linear_act(t, wd @ w, None, t, "silu"), w, w, wd)), x, check_trace=False)
    y = T.bf16(g, 40, 72).requires_grad_()
    dy = T.bf16(g, 40, 72)
    want = torch.autograd.grad(gated_ffn(linear_act(y, wd @ w, None, y, "silu"), w, w, wd), y, dy)[0]
    assert torch.equal(torch.autograd.grad(traced(y), y, dy)[0], want)


@pytest.mark.parametrize("H", [(1 << 19) - 8, 1 << 19, (1 << 20) - 8])
def test_gradients_of_the_widest_hidden_layers(H):
    """From 2^19 on, both first weights' gradients are more rows than one weight gradient takes."""
    from transformer_amd import gated_ffn
    g = T.gen("wide", H)
    M, D = 5, 16
    t = [T.bf16(g, M, D), T.bf16(g, H, D, std=0.2), T.bf16(g, H, D, std=0.2), T.bf16(g, D, H, std=1e-3)]
    dy = T.bf16(g, M, D)
    leaves = [v.clone().requires_grad_() for v in t]
    got = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    x, wg, wu, wd = (v.double() for v in t)
    a, u, dh = T.act64(x @ wg.t(), "silu"), x @ wu.t(), dy.double() @ wd
    dg, du = dh * u * T.slope64(x @ wg.t(), "silu"), dh * a
    for name, v, ref in zip(("dx", "dw_gate", "dw_up", "dw_down"), got,
                            (dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.double().t() @ (a * u))):
        T.near(v, ref, name)
