"""linear_act, gated_ffn and clip_grad_norm_ where their memory, their graphs and their ranges end: what lies around the
operands, row counts around every change of kernel, outputs past 2^31 elements, second derivatives, batched gradients, calls
captured side by side.  Bounds as derived in test_gpu_feedforward.py."""
import ctypes

import pytest
import torch

from tests import test_gpu_feedforward as T

pytestmark = pytest.mark.gpu

NAN = float("nan")


# with test_gpu_feedforward's sizes: every tile of every product, whole and cut along k (tests/test_gemm_plan.py asserts it)
TILES = [(5924, 328, 672), (5558, 176, 4744), (3338, 3808, 600)]


@pytest.mark.parametrize("M,N,K", TILES)
def test_further_tiles(M, N, K):
    for act in ("silu", "gelu_tanh"):
        T.test_linear_act_forward(M, N, K, True, True, act)
        T.test_gated_ffn_forward(M, N, K, True, act)
        T.test_linear_act_gradients(M, N, K, act)
        T.test_gated_ffn_gradients(M, N, K, act)


def inside(t, rows=3, left=8, right=16):
    """A copy of ``t [M, N]`` as a window of a buffer of NaNs, and that buffer."""
    M, N = t.shape
    buf = torch.full((M + 2 * rows, left + N + right), NAN, dtype=t.dtype, device=t.device)
    view = buf[rows:rows + M, left:left + N]
    view.copy_(t)
    return view, buf


def untouched(view, buf, rows=3, left=8):
    """Whether everything of ``buf`` around ``view`` is still NaN."""
    M, N = view.shape
    out = torch.ones_like(buf, dtype=torch.bool)
    out[rows:rows + M, left:left + N] = False
    return bool(buf[out].isnan().all())


SIZES = [(1, 24, 40), (33, 136, 72), (64, 264, 328), (65, 136, 200), (200, 264, 136), (300, 1000, 72), (4090, 328, 4072), *TILES]


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_what_lies_around_the_operands_is_neither_read_into_results_nor_written(M, N, K, act):
    from transformer_amd import _lib, linear_ops
    g = T.gen("around", M, N, K, act)
    x, w, b, r, dy = T.bf16(g, M, K), T.bf16(g, N, K, std=K ** -0.5), T.bf16(g, N), T.bf16(g, M, N), T.bf16(g, M, N)
    w2, code = T.bf16(g, N, K, std=K ** -0.5), linear_ops.ACTIVATIONS[act]
    launch, size = linear_ops._launch, linear_ops._saved_size(M, N)
    runs = []
    for windows in (False, True):
        put = inside if windows else (lambda t: (t.clone(), None))
        (xv, _), (wv, _), (w2v, _), (rv, _), (dyv, _) = (put(t) for t in (x, w, w2, r, dy))
        new = lambda rows, cols: put(torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda"))
        saved = torch.zeros(2 * size, dtype=torch.uint8, device="cuda")  # (rows past the last are whatever they were)
        outs = []

        def out(rows, cols):
            outs.append(new(rows, cols))
            return outs[-1][0]

        def call(entry, a, like):
            ws = linear_ops._fit_workspace(entry + "_workspace_bytes", a, like) if hasattr(a, "workspace") else None
            launch(entry, a, like, entry)
            return ws

        y = out(M, N)
        call("mla_linear_act", _lib.LinearActArgs(xv.data_ptr(), wv.data_ptr(), b.data_ptr(), rv.data_ptr(), y.data_ptr(),
                                                  saved.data_ptr() if code else None, None, 0, M, N, K, xv.stride(0),
                                                  wv.stride(0), rv.stride(0), y.stride(0), code), y)
        dz = out(M, N)
        db = torch.full((N,), NAN, device="cuda")
        call("mla_act_grad", _lib.ActGradArgs(dyv.data_ptr(), saved.data_ptr() if code else None, dz.data_ptr(), db.data_ptr(),
                                              None, 0, M, N, dyv.stride(0), dz.stride(0), code, _lib.MLA_DTYPE_F32), y)
        dx = out(M, K)
        call("mla_linear_dx", _lib.LinearDxArgs(dyv.data_ptr(), wv.data_ptr(), None, dx.data_ptr(), None, 0, M, N, K,
                                                dyv.stride(0), wv.stride(0), 0, dx.stride(0)), y)
        if code:
            h = out(M, N)
            call("mla_gated_linear", _lib.GatedLinearArgs(xv.data_ptr(), wv.data_ptr(), w2v.data_ptr(), h.data_ptr(),
                                                          saved.data_ptr(), None, 0, M, N, K, xv.stride(0), wv.stride(0), w2v.stride(0),
                                                          h.stride(0), code), y)
            dgu = out(M, 2 * N)
            wd, _ = put(w.t().contiguous())
            dyk, _ = put(x)
            call("mla_gated_linear_bwd", _lib.GatedLinearBwdArgs(dyk.data_ptr(), wd.data_ptr(), saved.data_ptr(), dgu.data_ptr(),
                                                                 M, N, K, dyk.stride(0), wd.stride(0), dgu.stride(0), code), y)
        torch.cuda.synchronize()
        if windows:
            assert all(untouched(v, buf) for v, buf in outs)
        runs.append([db, *(v.clone() for v, _ in outs)])
    for i, (a, c) in enumerate(zip(*runs)):
        assert torch.equal(a, c), f"output {i}"


@pytest.mark.parametrize("M", [1, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 96, 127, 128, 129, 255, 256, 257])
def test_row_counts_around_every_change_of_kernel(M):
    """Every row of a long input has the same result whatever rows are with it (up to the order of the sums)."""
    from transformer_amd import gated_ffn, linear_act
    g = T.gen("rows")
    x, r = T.bf16(g, 300, 328), T.bf16(g, 300, 328)
    w, b, wg, wu, wd = T.bf16(g, 136, 328, std=0.06), T.bf16(g, 136), *(T.bf16(g, 136, 328, std=0.06) for _ in range(2)), \
        T.bf16(g, 328, 136, std=0.09)
    xm, rm = x[:M].double(), r[:M].double()
    z = xm @ w.double().t() + b.double()
    ez = (xm.abs() @ w.double().abs().t() + b.double().abs()) * (328 + 8) * T.EPS32
    T.within(linear_act(x[:M], w, b, None, "silu"), T.act64(z, "silu"), 1.13 * ez + T.act_error(z), "y")
    gg, uu = xm @ wg.double().t(), xm @ wu.double().t()
    eg, eu = (xm.abs() @ t.double().abs().t() * (328 + 8) * T.EPS32 for t in (wg, wu))
    a = T.act64(gg, "silu")
    h, d6 = a * uu, wd.double().abs()
    eh = (1.13 * eg + T.act_error(gg)) * (uu.abs() + eu) + a.abs() * eu + h.abs() * T.EPS32
    eh = eh + (h.abs() + eh) * T.EPS16
    ref = h @ wd.double().t() + rm
    T.within(gated_ffn(x[:M], wg, wu, wd, r[:M]), ref,
             eh @ d6.t() + (h.abs() + eh) @ d6.t() * (136 + 8) * T.EPS32 + ref.abs() * T.EPS32, "ffn")


def test_outputs_past_two_to_the_31_elements():
    from transformer_amd import linear_act
    M, N, K = 560_000, 4096, 64  # 2.29e9 outputs, 4.6 GB; 6.9 GB kept
    g = T.gen("long")
    x, w, b = T.bf16(g, M, K), T.bf16(g, N, K, std=K ** -0.5), T.bf16(g, N)
    for t in (x, w, b):
        t.requires_grad_()
    y = linear_act(x, w, b, None, "silu")
    dy = T.bf16(g, 1, N).expand(M, N)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy.contiguous())
    with torch.no_grad():
        at = torch.cat([torch.arange(s, s + 8, device="cuda") for s in (0, (1 << 30) // N - 4, (1 << 31) // N - 4, M - 8)])
        x6, w6 = x[at].double(), w.double()
        z = x6 @ w6.t() + b.double()
        ez = (x6.abs() @ w6.abs().t() + b.double().abs()) * (K + 8) * T.EPS32
        T.within(y[at], T.act64(z, "silu"), 1.13 * ez + T.act_error(z), "y")
        dz = dy[at].double() * T.slope64(z, "silu")
        T.near(dx[at], dz @ w6, "dx")
        sums, prod = torch.zeros(N, dtype=torch.float64, device="cuda"), torch.zeros(N, K, dtype=torch.float64, device="cuda")
        for s in range(0, M, 20_000):
            part = x[s:s + 20_000].double()
            dz = dy[:1].double() * T.slope64(part @ w6.t() + b.double(), "silu")
            sums += dz.sum(0)
            prod += dz.t() @ part
        T.near(dw, prod, "dw")
        T.near(db, sums, "db")


def test_more_rows_than_a_weight_gradient_takes_at_once():
    from transformer_amd import gated_ffn, linear_act
    M = (1 << 24) + 1000
    g = T.gen("many rows")
    x, w, b, dy = T.bf16(g, M, 8), T.bf16(g, 16, 8, std=0.3), T.bf16(g, 16), T.bf16(g, M, 16)
    for t in (x, w, b):
        t.requires_grad_()
    y = linear_act(x, w, b, None, "relu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        z = x.double() @ w.double().t() + b.double()
        dz = dy.double() * (z > 0)
        T.near(dx, dz @ w.double(), "dx")
        T.near(dw, dz.t() @ x.double(), "dw")
        T.near(db, dz.sum(0), "db")
        T.near(y, torch.relu(z), "y")
    wd = T.bf16(g, 8, 16, std=0.3).requires_grad_()
    y = gated_ffn(x, w, w, wd, None, "relu")
    got = torch.autograd.grad(y, (w, wd), x.detach())
    with torch.no_grad():
        z, d = x.double() @ w.double().t(), x.double()
        dh = d @ wd.double()
        T.near(got[0], (dh * 2 * torch.relu(z)).t() @ d, "dw of both")
        T.near(got[1], d.t() @ torch.relu(z).square(), "dwd")


def test_rows_that_lie_far_apart():
    from transformer_amd import linear_act
    g = T.gen("far apart")
    buf = torch.zeros(300, (1 << 22) - 8, dtype=torch.bfloat16, device="cuda")  # 2.5 GB
    x, w, dy = buf[:, 16:152], T.bf16(g, 72, 136, std=0.1).requires_grad_(), T.bf16(g, 300, 72)
    x.copy_(T.bf16(g, 300, 136))
    near, far = (linear_act(t, w, None, None, "silu") for t in (x.contiguous(), x))
    assert torch.equal(near, far)
    (a,), (c,) = (torch.autograd.grad(t, w, dy) for t in (near, far))
    T.near(c, a.double(), "dw")


def test_slopes_of_huge_pre_activations():
    """z up to 3e38: the slope is 0 or 1 there, and 0 times a square past the range is not formed."""
    from transformer_amd import gated_ffn, linear_act
    z = torch.tensor([1e10, 1e19, 3e19, 1e30, 2e38, -1e10, -1e19, -3e19, -1e30, -2e38], device="cuda").bfloat16()
    x = torch.zeros(10, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = z
    w = torch.zeros(8, 8, dtype=torch.bfloat16, device="cuda")
    w[:, 0] = 1
    for act in ("relu", "silu", "gelu_tanh"):
        leaf = x.clone().requires_grad_()
        y = linear_act(leaf, w, None, None, act)
        dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert torch.equal(y[:, 0], torch.where(z > 0, z, 0)), act
        assert torch.equal(dx[:, 0], torch.where(z > 0, 8, 0).bfloat16()), act
        up = torch.zeros(8, 8, dtype=torch.bfloat16, device="cuda")  # u = 0: dg = 0
        leaf = x.clone().requires_grad_()
        dx, = torch.autograd.grad(gated_ffn(leaf, w, up, w, None, act), leaf, torch.full_like(x, 0.0625))
        assert torch.equal(dx, torch.zeros_like(dx)), act


def leaves_of(g, M=40, H=72, D=136):
    return [t.requires_grad_() for t in (T.bf16(g, M, D), T.bf16(g, H, D, std=0.1), T.bf16(g, H, D, std=0.1),
                                         T.bf16(g, D, H, std=0.1), T.bf16(g, M, D), T.bf16(g, H))]


def test_second_derivatives_are_refused():
    from transformer_amd import gated_ffn, linear_act
    x, wg, wu, wd, r, b = leaves_of(T.gen("second"))
    for y in (gated_ffn(x, wg, wu, wd, r), linear_act(x, wg, b, None, "silu")):
        dx, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(dx.float().square().sum(), x)


def test_batched_gradients_equal_one_after_the_other():
    from transformer_amd import gated_ffn, linear_act
    g = T.gen("batched")
    x, wg, wu, wd, r, b = leaves_of(g)
    for y, of in ((gated_ffn(x, wg, wu, wd, r), (x, wg, wu, wd, r)), (linear_act(x, wg, b, None, "silu"), (x, wg, b))):
        dys = T.bf16(g, 3, *y.shape)
        together = torch.autograd.grad(y, of, dys, is_grads_batched=True, retain_graph=True)
        for i in range(3):
            one = torch.autograd.grad(y, of, dys[i], retain_graph=True)
            assert all(torch.equal(t[i], o) for t, o in zip(together, one))


def test_functional_transforms():
    """vmap runs through the registered operators; torch.func.grad, which torch's registered operators do not take, raises."""
    from transformer_amd import gated_ffn, linear_act
    g = T.gen("func")
    with torch.no_grad():
        xs, wg, wu, wd, b = T.bf16(g, 3, 40, 136), *(T.bf16(g, 72, 136, std=0.1) for _ in range(2)), T.bf16(g, 136, 72, std=0.1), \
            T.bf16(g, 72)
    for f, of in ((lambda x, w: gated_ffn(x, w, wu, wd), wg), (lambda x, w: linear_act(x, w, b, None, "silu"), wg)):
        got = torch.func.vmap(f, in_dims=(0, None))(xs, of)
        assert all(torch.equal(got[i], f(xs[i], of)) for i in range(3))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda x: f(x, of).float().square().sum())(xs[0])


def test_graphs_that_live_on():
    """A graph run twice with retain_graph, saved weights changed in place, hooks on saved tensors."""
    from transformer_amd import gated_ffn
    g = T.gen("live")
    x, wg, wu, wd, r, b = leaves_of(g)
    dy = T.bf16(g, *x.shape)
    y = gated_ffn(x, wg, wu, wd, r)
    one = torch.autograd.grad(y, (x, wg, wd), dy, retain_graph=True)
    assert all(torch.equal(a, c) for a, c in zip(one, torch.autograd.grad(y, (x, wg, wd), dy, retain_graph=True)))
    with torch.no_grad():
        wg.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        wg.div_(2)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.shape) or t.cpu(), lambda t: t.cuda()):
        y = gated_ffn(x, wg, wu, wd, r)
    assert len(kept) == 6
    assert all(torch.equal(a, c) for a, c in zip(one, torch.autograd.grad(y, (x, wg, wd), dy)))


def test_the_residual_may_be_the_output():
    from transformer_amd import _lib, linear_ops, linear_act
    for M, N, K in ((20, 72, 136), (300, 264, 72), (4090, 328, 4072)):  # few rows, tiles, tiles cut along k
        g = T.gen("alias", M)
        x, w, r = T.bf16(g, M, K), T.bf16(g, N, K, std=K ** -0.5), T.bf16(g, M, N)
        want, y = linear_act(x, w, None, r, "relu"), r.clone()
        a = _lib.LinearActArgs(x.data_ptr(), w.data_ptr(), None, y.data_ptr(), y.data_ptr(), None, None, 0, M, N, K, K, K, N, N,
                               linear_ops.ACTIVATIONS["relu"])
        ws = linear_ops._fit_workspace("mla_linear_act_workspace_bytes", a, y)  # noqa: F841
        linear_ops._launch("mla_linear_act", a, y, "linear_act")
        assert torch.equal(y, want)


def test_a_short_workspace_is_refused():
    from transformer_amd import _lib
    lib = _lib.load()
    M, N, K = 4090, 328, 4072
    z = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    a = _lib.LinearActArgs(z.data_ptr(), z.data_ptr(), None, None, z.data_ptr(), None, None, 0, M, N, K, K, K, 0, N, 0)
    need = lib.mla_linear_act_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    assert need > 0
    for at, size in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 16, need)):
        a.workspace, a.workspace_bytes = at, size
        assert lib.mla_linear_act(ctypes.byref(a), None) == _lib.MLA_ERR_WORKSPACE


def test_two_captured_graphs_replayed_together():
    """Two graphs, each with its own workspaces, on two streams at once: products cut along k, their backward and the clipping."""
    from transformer_amd import clip_grad_norm_, linear_act
    M, N, K = 4090, 328, 4072
    g = T.gen("two graphs")
    sets = [[T.bf16(g, M, K), T.bf16(g, N, K, std=K ** -0.5), T.bf16(g, N), T.bf16(g, M, N)] for _ in range(2)]

    def step(x, w, b, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = linear_act(*leaves, None, "gelu_tanh")
        grads = torch.autograd.grad(y, leaves, dy)
        for t, d in zip(leaves, grads):
            t.grad = d
        return [y.detach(), clip_grad_norm_(leaves, 1.0), *grads]

    want = [[t.clone() for t in step(*s)] for s in sets]
    graphs, outs = [], []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*s)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*s))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(a, c) for a, c in zip(out, w))
            for t in out:
                t.fill_(NAN)
        torch.cuda.synchronize()


def test_compiled_with_any_number_of_rows():
    from transformer_amd import gated_ffn, linear_act
    g = T.gen("dynamic")
    w = [T.bf16(g, 136, 72, std=0.1), T.bf16(g, 136, 72, std=0.1), T.bf16(g, 72, 136, std=0.1), T.bf16(g, 72)]

    def f(x, wg, wu, wd, b):
        return linear_act(gated_ffn(x, wg, wu, wd, x), wd[:, :72], b, None, "gelu_tanh")

    compiled = torch.compile(f, backend="aot_eager", dynamic=True, fullgraph=True)
    for M in (50, 51, 7, 200):
        leaves = [t.requires_grad_() for t in (T.bf16(g, M, 72), *(t.clone() for t in w))]
        dy = T.bf16(g, M, 72)
        got, want = compiled(*leaves), f(*leaves)
        assert torch.equal(got, want)
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)))


def test_registered_operators_hold_their_contract():
    """Schemas, fake kernels and autograd registration; without what the backward keeps, the operator forms it again."""
    from torch.library import opcheck
    ops = torch.ops.mla_mi355x
    g = T.gen("contract")
    x, wg, wu, wd, r, b = leaves_of(g)
    dy, dz = T.bf16(g, 40, 136), T.bf16(g, 40, 72)
    every = ("test_schema", "test_faketensor", "test_autograd_registration")
    for save in (False, True):
        opcheck(ops.gated_ffn, (x, wg, wu, wd, r, "silu", save), test_utils=every)
        opcheck(ops.linear_act, (x, wg, b, None, "silu", save), test_utils=every)
        opcheck(ops.linear_act, (x, wg, None, None, "none", save), test_utils=every)
    _, h, saved = ops.gated_ffn(x, wg, wu, wd, None, "silu", True)
    opcheck(ops.gated_ffn_bwd, (dy, *(t.detach() for t in (x, wg, wu, wd, h)), saved, "silu", True, True, False, True),
            test_utils=every[:2])
    saved = ops.linear_act(x, wg, b, None, "silu", True)[1]
    opcheck(ops.linear_act_bwd, (dz, x.detach(), wg.detach(), saved, "silu", True, True, torch.float32), test_utils=every[:2])
    for f, of, d in ((lambda save: ops.gated_ffn(x, wg, wu, wd, r, "silu", save)[0], (x, wg, wu, wd, r), dy),
                     (lambda save: ops.linear_act(x, wg, b, None, "silu", save)[0], (x, wg, b), dz)):
        kept, formed = (torch.autograd.grad(f(save), of, d) for save in (True, False))
        assert all(torch.equal(a, c) for a, c in zip(kept, formed))


def test_gradients_that_are_views_of_one_buffer_are_used_like_any_other():
    """The two first weights' gradients share an allocation: accumulated, changed in place, clipped and stepped apart."""
    from transformer_amd import SwiGLU, clip_grad_norm_
    torch.manual_seed(5)
    m = SwiGLU(136, 264).cuda().bfloat16()
    x = T.bf16(T.gen("views"), 40, 136)
    m(x, x).float().square().mean().backward()
    once = [p.grad.clone() for p in m.parameters()]
    m(x, x).float().square().mean().backward()
    assert all(torch.equal(p.grad, 2 * q) for p, q in zip(m.parameters(), once))  # (twice a bf16 value is one)
    m.w1.weight.grad.zero_()
    assert torch.equal(m.w3.weight.grad, 2 * once[2]) and not m.w1.weight.grad.any()
    norm = clip_grad_norm_(m.parameters(), 1e-3)
    left = torch.stack([p.grad.double().square().sum() for p in m.parameters()]).sum().sqrt()
    assert norm > 1e-3 and abs(float(left) - 1e-3) <= 1e-3 * (T.EPS16 + 1e-5)  # (a rounding to bf16 an element)
    torch.optim.SGD(m.parameters(), lr=0.1).step()


def test_gradients_without_elements():
    from transformer_amd import clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(0, 4, device="cuda"))
    p.grad = torch.zeros(0, 4, device="cuda")
    assert float(clip_grad_norm_([p], 1.0)) == 0 and float(grad_norm([p.grad], float("inf"))) == 0
