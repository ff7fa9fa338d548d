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


def _gradients_of_few_rows(g, x, w, wg, wu, wd):
    """dx of both operators, and the gated block's first weight gradients, against 64 bits (in parts of the wide sizes)."""
    from transformer_amd import gated_ffn, linear_act
    x = x.detach().requires_grad_()
    y = linear_act(x, w, None, None, "relu")
    dy = T.bf16(g, *y.shape)
    dx, = torch.autograd.grad(y, x, dy)
    x6, ref = x.detach().double(), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for part, d in zip(w.split(4096), dy.split(4096, 1)):
        ref += (d.double() * (x6 @ part.double().t() > 0)) @ part.double()
    T.near(dx, ref, "dx")
    leaves = [x, wg.detach().requires_grad_()]
    y = gated_ffn(x, leaves[1], wu, wd, x)
    dy = T.bf16(g, *y.shape)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    ref = dy.double()
    for s in range(0, wg.size(0), 4096):
        a, b, c = wg[s:s + 4096].double(), wu[s:s + 4096].double(), wd[:, s:s + 4096].double()
        p, u, dh = x6 @ a.t(), x6 @ b.t(), dy.double() @ c
        dg = dh * u * T.slope64(p, "silu")
        ref = ref + dg @ a + (dh * T.act64(p, "silu")) @ b
        T.near(dw[s:s + 4096], dg.t() @ x6, "dw_gate")
    T.near(dx, ref, "gated dx")


@pytest.mark.parametrize("M,H,D", [(5, 520, 808), (200, 1032, 264), (300, 264, 1032)])
def test_gradients_through_weights_in_parts(M, H, D, monkeypatch):
    from transformer_amd import linear_ops
    g = T.gen("parts", M, H, D)
    t = [T.bf16(g, M, D), *(T.bf16(g, H, D, std=D ** -0.5) for _ in range(3)), T.bf16(g, D, H, std=H ** -0.5)]
    monkeypatch.setattr(linear_ops, "REACH", 257 * (max(H, D) + 64))
    launches = []
    launch = linear_ops._launch
    monkeypatch.setattr(linear_ops, "_launch", lambda entry, *a: launches.append(entry) or launch(entry, *a))
    _gradients_of_few_rows(g, *t)
    parts = {"mla_linear_dx": -(-D // linear_ops._columns(H, D)), "mla_gated_linear_bwd": -(-H // linear_ops._columns(D, H))}
    assert min(parts.values()) > 1
    assert launches.count("mla_linear_dx") == 2 * parts["mla_linear_dx"]  # (linear_act's and the gated block's)
    assert launches.count("mla_gated_linear_bwd") == parts["mla_gated_linear_bwd"]


def test_gradients_through_weights_whose_rows_lie_far_apart():
    g = T.gen("far weights")
    M, H, D = 40, 304, 264
    buf = torch.zeros(304, (1 << 22) - 8, dtype=torch.bfloat16, device="cuda")  # 2.6 GB
    w, wg, wd = buf[:, 64:64 + D], buf[:, 1024:1024 + D], buf[:D, 4096:4096 + H]
    for t in (w, wg, wd):
        t.copy_(T.bf16(g, *t.shape, std=0.06))
    _gradients_of_few_rows(g, T.bf16(g, M, D), w, wg, T.bf16(g, H, D, std=0.06), wd)


def test_gradients_through_weights_of_two_gib():
    g = T.gen("large weights")
    H, D = (1 << 15) + 8, 1 << 15
    make = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda").normal_(0, 2.0 ** -7, generator=g)
    wg = make(H, D)
    _gradients_of_few_rows(g, T.bf16(g, 3, D), wg, wg, make(H, D), make(D, H))


@pytest.mark.parametrize("shape", [(1, 1, 72), (72,), (3, 40, 1), (2, 3, 40, 72), (1, 40, 72), ()])
def test_residuals_of_another_shape_are_refused_in_every_type(shape):
    from transformer_amd import SwiGLU, gated_ffn, linear_act
    g = T.gen("residual")
    x, w, wd = T.bf16(g, 3, 40, 72), T.bf16(g, 72, 72, std=0.1), T.bf16(g, 72, 72, std=0.1)
    with torch.device("cuda"):
        ffn, hooked = SwiGLU(72, 72), SwiGLU(72, 72)
    hooked.w1.register_forward_hook(lambda *a: None)
    for dt in (torch.bfloat16, torch.float32):
        bad, good = torch.zeros(shape, dtype=dt, device="cuda"), torch.ones(3, 40, 72, dtype=dt, device="cuda")
        for call in (lambda r: linear_act(x, w, None, r, "silu"), lambda r: gated_ffn(x, w, w, wd, r), lambda r: ffn(x, r),
                     lambda r: hooked(x, r)):
            with torch.autocast("cuda", dtype=torch.bfloat16):
                with pytest.raises(ValueError, match="residual"):
                    call(bad)
                assert call(good).shape == x.shape and call(good).dtype == dt


@pytest.mark.parametrize("dims,weights,rows,amp", [
    ((72, 136), torch.float32, torch.float32, None), ((72, 136), torch.float16, torch.float16, None),
    ((20, 36), torch.bfloat16, torch.bfloat16, None), ((72, 140), torch.bfloat16, torch.bfloat16, None),
    ((72, 136), torch.float64, torch.float64, None), ((72, 136), torch.float32, torch.bfloat16, torch.float16),
    ((72, 136), torch.float32, torch.float32, torch.float16), ((20, 136), torch.float32, torch.float32, torch.bfloat16),
    ((72, 136), torch.float16, torch.float32, torch.bfloat16)])
def test_blocks_that_the_kernels_do_not_take_run_in_torch(dims, weights, rows, amp):
    import torch.nn.functional as F
    from transformer_amd import SwiGLU
    torch.manual_seed(6)
    with torch.device("cuda"):
        m = SwiGLU(*dims).to(weights)
    g = T.gen("torch", dims)
    x, r, dy = (torch.randn(2, 30, dims[0], generator=g, device="cuda").to(rows) for _ in range(3))

    def run(f):
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=amp or torch.bfloat16, enabled=amp is not None):
            y = f(leaf)
        return [y, *torch.autograd.grad(y, (leaf, *m.parameters()), dy.to(y.dtype))]

    for got, want in ((run(m), run(lambda t: m.w2(F.silu(m.w1(t)) * m.w3(t)))),
                      (run(lambda t: m(t, r)), run(lambda t: r + m.w2(F.silu(m.w1(t)) * m.w3(t))))):
        assert all(a.dtype == c.dtype and torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("M,N,K", [(1, 24, 40), (20, 264, 72), (64, 4104, 40), (65, 264, 128), (300, 1000, 64), (4090, 328, 4072),
                                   (4750, 3496, 3144)])
def test_an_fp32_bias_is_added_as_it_is(M, N, K):
    from transformer_amd import linear_act
    g = T.gen("fp32 bias", M, N, K)
    x, w, dy = T.bf16(g, M, K), T.bf16(g, N, K, std=K ** -0.5), T.bf16(g, M, N)
    b = torch.randn(N + 1, generator=g, device="cuda")[1:]  # (off 16 bytes)
    r = (-b).bfloat16().expand(M, N)
    # without a product: what is left of the bias once its own bf16 value is taken away, rounded once
    assert torch.equal(linear_act(torch.zeros_like(x), w, b, r), (b + r.float()).bfloat16())
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = linear_act(*leaves, r, "silu")
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    z = x.double() @ w.double().t() + b.double()
    mag = x.double().abs() @ w.double().abs().t() + b.double().abs()
    ref = T.act64(z, "silu") + r.double()
    T.within(y.detach(), ref, 1.13 * mag * (K + 8) * T.EPS32 + T.act_error(z) + ref.abs() * T.EPS32, "y")
    dz = dy.double() * T.slope64(z, "silu")
    assert db.dtype == torch.float32 and y.dtype == torch.bfloat16
    # (z kept to 24 bits, a slope's derivative below 1 / 2, fp32 sums)
    T.within(db, dz.sum(0), (dy.double().abs() * (z.abs() * 2.0 ** -16 + mag * (K + 8) * T.EPS32 + 16 * T.EPS32 * (1 + z.abs()) ** 2)
                             + dz.abs() * (M + 8) * T.EPS32).sum(0), "db")
    if min(M, N, K) >= 20:
        T.near(dx, dz @ w.double(), "dx")
        T.near(dw, dz.t() @ x.double(), "dw")


def test_a_compiled_block():
    from transformer_amd import SwiGLU
    torch.manual_seed(8)
    m = SwiGLU(72, 136).cuda().bfloat16()
    x, dy = T.bf16(T.gen("block"), 50, 72), T.bf16(T.gen("block dy"), 50, 72)
    compiled = torch.compile(m, backend="aot_eager", fullgraph=True)
    want, got = (torch.autograd.grad(f(x, x), tuple(m.parameters()), dy) for f in (m, compiled))
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_block_whose_last_layer_has_another_width_runs_in_torch():
    import torch.nn.functional as F
    from transformer_amd import SwiGLU
    torch.manual_seed(9)
    with torch.device("cuda"):
        m = SwiGLU(72, 136)
        m.w2 = torch.nn.Linear(136, 40, bias=False)
        m.bfloat16()
        x = torch.randn(30, 72).bfloat16()
    assert torch.equal(m(x), m.w2(F.silu(m.w1(x)) * m.w3(x)))


def test_the_operators_without_rows_and_without_what_they_keep():
    ops = torch.ops.mla_mi355x
    z = lambda *s: torch.zeros(*s, device="cuda").bfloat16().requires_grad_()
    for shape in ((0, 16), (2, 0, 16)):
        x, w, wd, b = z(*shape), z(24, 16), z(16, 24), z(24)
        for save in (False, True):
            for y, of in ((ops.gated_ffn(x, w, w, wd, None, "silu", save)[0], (x, w, wd)),
                          (ops.linear_act(x, w, b, None, "silu", save)[0], (x, w, b))):
                got = torch.autograd.grad(y, of, torch.zeros_like(y))
                assert all(t.shape == o.shape and not t.any() for t, o in zip(got, of))


def test_one_row_of_one_dimension():
    from transformer_amd import gated_ffn, linear_act
    g = T.gen("one row")
    x, w, wd, b, r = T.bf16(g, 72), T.bf16(g, 136, 72, std=0.1), T.bf16(g, 72, 136, std=0.1), T.bf16(g, 136), T.bf16(g, 136)
    for f, dy in ((lambda t: linear_act(t, w, b, r.view(*t.shape[:-1], 136), "silu"), T.bf16(g, 136)),
                  (lambda t: gated_ffn(t, w, w, wd, t), T.bf16(g, 72))):
        one, row = x.clone().requires_grad_(), x.view(1, 72).clone().requires_grad_()
        y, want = f(one), f(row)
        assert y.dim() == 1 and torch.equal(y, want[0])
        assert torch.equal(torch.autograd.grad(y, one, dy)[0], torch.autograd.grad(want, row, dy.view(1, -1))[0][0])
