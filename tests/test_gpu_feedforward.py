"""linear_act and gated_ffn, forward and backward, against plain forms in 64 bits.

Tolerances.  A sum of K exact products in fp32 is off by at most (K + 8) 2^-24 of the sum of magnitudes; an activation's slope
is at most 1.13 and its own evaluation off by at most |z| (8 + 2 |z|) 2^-23 (an exponential of an argument rounded to fp32, a
reciprocal, two products); a rounding to bf16 is off by at most 2^-8 of the value.  Where a bf16 value enters a second product
(the hidden layer, the gradients of the first products), each of its roundings may count in full in the element-wise bound.
Over a whole tensor they do not line up: one rounding to bf16 has a relative rms error of at most 2^-8 / sqrt(3) = 2.26e-3,
and two independent ones 3.2e-3, which ``NORM`` allows (with 10 % for the spread of small samples).
"""
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS16, EPS32 = 2.0 ** -8, 2.0 ** -24
NORM = 3.2e-3 * 1.1
DEV = "cuda"


def act64(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    return torch.relu(z) if name == "relu" else z


def slope64(z, name):
    """The derivative, from autograd in 64 bits (relu'(0) = 0)."""
    z = z.detach().clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, name).sum(), z)[0]


def act_error(z):
    return z.abs() * (8 + 2 * z.abs()) * 2 * EPS32


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def bf16(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).bfloat16()


def within(got, ref, bound, what):
    d = (got.double() - ref).abs()
    assert got.dtype == torch.bfloat16 or got.dtype == torch.float32
    bound = bound + (ref.abs() + bound) * (EPS16 if got.dtype == torch.bfloat16 else EPS32)
    assert (d <= bound).all(), f"{what}: {(d - bound).max().item():.3g} over the bound at {int((d - bound).argmax())}"


def near(got, ref, what, tol=NORM):
    n = ref.norm()
    assert n == 0 or (got.double() - ref).norm() <= tol * n, f"{what}: {float((got.double() - ref).norm() / n):.3g}"


SIZES = [(1, 8, 8), (1, 1000, 520), (2, 24, 40), (31, 264, 72), (33, 8, 640), (64, 256, 64), (65, 264, 128), (127, 136, 1000),
         (129, 392, 200), (300, 1000, 64), (1000, 264, 1800)]
# 256 x 256 tiles, whole, ragged and cut along k, with a k tail (tests/test_gemm_plan.py asserts that these sizes take them)
LARGE = [(4096, 4096, 256), (4090, 4072, 328), (4090, 328, 4072), (1250, 4104, 3248), (4750, 3496, 3144)]


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_act_forward(M, N, K, bias, res, act):
    from transformer_amd import linear_act
    g = gen(M, N, K, bias, res, act)
    x, w = bf16(g, M, K), bf16(g, N, K, std=K ** -0.5)
    b, r = bf16(g, N) if bias else None, bf16(g, M, N) if res else None
    with torch.no_grad():
        y = linear_act(x, w, b, r, act)
        again = linear_act(x, w, b, r, act)
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias:
        z, mag = z + b.double(), mag + b.double().abs()
    ref = act64(z, act) + (r.double() if res else 0)
    err = 1.13 * mag * (K + 8) * EPS32 + act_error(z) + ref.abs() * EPS32
    assert y.dtype == torch.bfloat16 and y.shape == (M, N)
    within(y, ref, err, "y")
    assert torch.equal(y, again), "not bitwise reproducible"


def ffn64(x, wg, wu, wd, res, act):
    g, u = x @ wg.t(), x @ wu.t()
    y = (act64(g, act) * u) @ wd.t()
    return y if res is None else y + res


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("M,H,D", SIZES)
def test_gated_ffn_forward(M, H, D, res, act):
    from transformer_amd import gated_ffn
    g = gen(M, H, D, res, act)
    x, wg, wu, wd = bf16(g, M, D), bf16(g, H, D, std=D ** -0.5), bf16(g, H, D, std=D ** -0.5), bf16(g, D, H, std=H ** -0.5)
    r = bf16(g, M, D) if res else None
    with torch.no_grad():
        y = gated_ffn(x, wg, wu, wd, r, act)
        again = gated_ffn(x, wg, wu, wd, r, act)
    x6, g6, u6, d6 = (t.double() for t in (x, wg, wu, wd))
    gg, uu = x6 @ g6.t(), x6 @ u6.t()
    mg, mu = (x6.abs() @ t.abs().t() * (D + 8) * EPS32 for t in (g6, u6))
    a = act64(gg, act)
    h = a * uu
    eh = (1.13 * mg + act_error(gg)) * (uu.abs() + mu) + a.abs() * mu + h.abs() * EPS32
    eh = eh + (h.abs() + eh) * EPS16
    ref = ffn64(x6, g6, u6, d6, None if r is None else r.double(), act)
    err = eh @ d6.abs().t() + (h.abs() + eh) @ d6.abs().t() * (H + 8) * EPS32 + ref.abs() * EPS32
    assert y.shape == x.shape
    within(y, ref, err, "y")
    if M * D >= 1000 and H >= 64:
        near(y, ref, "y")
    assert torch.equal(y, again), "not bitwise reproducible"


def linear_grads64(x, w, b, r, act, dy):
    z = x @ w.t() + (0 if b is None else b)
    dz = dy * slope64(z, act)
    return {"x": dz @ w, "w": dz.t() @ x, "b": dz.sum(0), "r": dy}, dz


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", SIZES + LARGE)
def test_linear_act_gradients(M, N, K, act):
    from transformer_amd import linear_act
    g = gen(M, N, K, act)
    x, w, b, r, dy = bf16(g, M, K), bf16(g, N, K, std=K ** -0.5), bf16(g, N, std=0.5), bf16(g, M, N), bf16(g, M, N)
    for t in (x, w, b, r):
        t.requires_grad_()
    y = linear_act(x, w, b, r, act)
    got = dict(zip("xwbr", torch.autograd.grad(y, (x, w, b, r), dy)))
    again = torch.autograd.grad(linear_act(x, w, b, r, act), (x, w, b, r), dy)
    with torch.no_grad():
        ref, dz = linear_grads64(x.double(), w.double(), b.double(), r.double(), act, dy.double())
        for k in "xwbr":
            assert got[k].dtype == torch.bfloat16
            if ref[k].numel() >= 1000 and min(M, N) >= 24:  # (fewer terms: the bound below)
                near(got[k], ref[k], "d" + k)
        if act != "relu":  # (whose slope jumps where z is within a rounding of 0)
            # dz: the slope from z kept to 24 bits (2^-16) and its fp32 sum, then one rounding
            z = x.double() @ w.double().t() + b.double()
            ez = x.double().abs() @ w.double().abs().t() * (K + 8) * EPS32 + z.abs() * 2.0 ** -15
            edz = dy.double().abs() * (1.2 * ez + 16 * EPS32 * (1 + z.abs()) ** 2)
            edz16 = edz + (dz.abs() + edz) * EPS16 * (act != "none")
            within(got["x"], ref["x"], edz16 @ w.double().abs() + dz.abs() @ w.double().abs() * (N + 8) * EPS32, "dx")
            within(got["w"], ref["w"], edz16.t() @ x.double().abs() + dz.abs().t() @ x.double().abs() * (M + 8) * EPS32, "dw")
            within(got["b"], ref["b"], edz.sum(0) + dz.abs().sum(0) * (M + 8) * EPS32, "db")
    assert torch.equal(got["r"], dy)
    assert all(torch.equal(a, c) for a, c in zip(got.values(), again)), "not bitwise reproducible"


@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("M,H,D", SIZES + LARGE)
def test_gated_ffn_gradients(M, H, D, act):
    from transformer_amd import gated_ffn
    g = gen(M, H, D, act)
    t = {"x": bf16(g, M, D), "wg": bf16(g, H, D, std=D ** -0.5), "wu": bf16(g, H, D, std=D ** -0.5),
         "wd": bf16(g, D, H, std=H ** -0.5), "r": bf16(g, M, D)}
    dy = bf16(g, M, D)
    for v in t.values():
        v.requires_grad_()
    y = gated_ffn(*t.values(), act)
    got = dict(zip(t, torch.autograd.grad(y, tuple(t.values()), dy)))
    again = torch.autograd.grad(gated_ffn(*t.values(), act), tuple(t.values()), dy)
    with torch.no_grad():
        x, wg, wu, wd = (t[k].double() for k in ("x", "wg", "wu", "wd"))
        gg, uu, dh = x @ wg.t(), x @ wu.t(), dy.double() @ wd
        a, s = act64(gg, act), slope64(gg, act)
        h, dg, du = a * uu, dh * uu * s, dh * a
        ref = {"x": dg @ wg + du @ wu, "wg": dg.t() @ x, "wu": du.t() @ x, "wd": dy.double().t() @ h, "r": dy.double()}
        for k, v in got.items():
            assert v.dtype == torch.bfloat16 and v.shape == t[k].shape
            if ref[k].numel() >= 1000 and min(M, H, D) >= 24:
                near(v, ref[k], "d" + k)
        if act != "relu":
            eg, eu = (x.abs() @ w.abs().t() * (D + 8) * EPS32 + z.abs() * 2.0 ** -15 for w, z in ((wg, gg), (wu, uu)))
            edh = dy.double().abs() @ wd.abs() * (D + 8) * EPS32
            ea = 1.13 * eg + act_error(gg)
            es = 1.2 * eg + 16 * EPS32 * (1 + gg.abs()) ** 2
            eu1 = uu.abs() + eu
            edg = edh * eu1 * (s.abs() + es) + dh.abs() * (eu * (s.abs() + es) + uu.abs() * es) + dg.abs() * 2 * EPS32
            edu = edh * (a.abs() + ea) + dh.abs() * ea + du.abs() * EPS32
            edg, edu = (e + (v.abs() + e) * EPS16 for e, v in ((edg, dg), (edu, du)))
            eh = ea * eu1 + a.abs() * eu + h.abs() * EPS32
            eh = eh + (h.abs() + eh) * EPS16
            within(got["x"], ref["x"], edg @ wg.abs() + edu @ wu.abs()
                   + (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) * (2 * H + 8) * EPS32, "dx")
            within(got["wg"], ref["wg"], edg.t() @ x.abs() + dg.abs().t() @ x.abs() * (M + 8) * EPS32, "dw_gate")
            within(got["wu"], ref["wu"], edu.t() @ x.abs() + du.abs().t() @ x.abs() * (M + 8) * EPS32, "dw_up")
            within(got["wd"], ref["wd"], dy.double().abs().t() @ eh + dy.double().abs().t() @ h.abs() * (M + 8) * EPS32,
                   "dw_down")
    assert torch.equal(got["r"], dy)
    assert all(torch.equal(a_, c) for a_, c in zip(got.values(), again)), "not bitwise reproducible"


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradients_against_differences(act):
    """The directional derivative of the 64-bit form along random directions, by central differences, against the kernels'
    gradients: they differ by at most the gradients' own rounding, NORM of their norm times the direction's (in one random
    direction far less: 6 / sqrt(n) of that)."""
    from transformer_amd import gated_ffn, linear_act
    g = gen(act)
    M, H, D = 150, 264, 136
    t = [bf16(g, M, D), bf16(g, H, D, std=0.1), bf16(g, H, D, std=0.1), bf16(g, D, H, std=0.1)]
    b, w, dy, dz = bf16(g, H), bf16(g, H, D, std=0.1), bf16(g, M, D), bf16(g, M, H)
    cases = [(t, lambda *a: gated_ffn(*a, None, act), lambda *a: ffn64(*a, None, act), dy),
             ([t[0], w, b], lambda *a: linear_act(*a, None, act), lambda x, w, b: act64(x @ w.t() + b, act), dz)]
    for inputs, ours, plain, dout in cases:
        leaves = [v.clone().requires_grad_() for v in inputs]
        grads = torch.autograd.grad(ours(*leaves), leaves, dout)
        base = [v.double() for v in inputs]
        for i, grad in enumerate(grads):
            v = torch.randn(base[i].shape, generator=g, device=DEV, dtype=torch.float64)
            at = lambda e: (plain(*[p + e * v if k == i else p for k, p in enumerate(base)]) * dout.double()).sum()
            want = (at(1e-5) - at(-1e-5)) / 2e-5
            got = (grad.double() * v).sum()
            assert (got - want).abs() <= 6 * NORM * grad.double().norm(), f"{act} input {i}"


def test_strided_unaligned_and_batched_inputs_equal_contiguous_ones():
    # padding that holds NaN, odd offsets, transposes and broadcast rows: the results are those of plain copies, bit for bit
    from transformer_amd import gated_ffn, linear_act
    g = gen("strides")
    buf = torch.full((70, 300), float("nan"), device=DEV).bfloat16()
    views = {"window": buf[3:68, 16:16 + 72], "odd": buf[3:68, 17:17 + 72]}
    wbuf = torch.full((264, 200), float("nan"), device=DEV).bfloat16()
    w = wbuf[:, 8:80]
    w.copy_(bf16(g, 264, 72, std=0.1))
    wd = bf16(g, 264, 72, std=0.1).t()  # a transposed weight
    b = bf16(g, 265)[1:]                # off the alignment
    x0, r0 = bf16(g, 65, 72), bf16(g, 264)
    for name, x in views.items():
        x.copy_(x0)
        with torch.no_grad():
            assert torch.equal(linear_act(x, w, b, None, "silu"), linear_act(x0, w.contiguous(), b.clone(), None, "silu")), name
            assert torch.equal(gated_ffn(x, w, w, wd), gated_ffn(x0, w.contiguous(), w.contiguous(), wd.contiguous())), name
        x.fill_(float("nan"))
    with torch.no_grad():
        xb = x0.view(5, 13, 72).transpose(0, 1)
        rb = r0.expand(13, 5, 264)  # one row for all
        y = linear_act(xb, w, b, rb, "relu")
        assert torch.equal(y, linear_act(xb.contiguous(), w, b, rb.contiguous(), "relu")) and y.shape == (13, 5, 264)
        one = x0[:1].expand(9, 72)  # the same row nine times
        assert torch.equal(linear_act(one, w), linear_act(x0[:1], w).expand(9, 264))
        r = bf16(g, 65, 72)
        assert torch.equal(gated_ffn(x0, w, w, wd, r), gated_ffn(x0, w, w, wd, r.t().contiguous().t()))


def test_infinities_and_nans_stay_in_their_rows():
    from transformer_amd import gated_ffn, linear_act
    g = gen("nan")
    x, w, wd = bf16(g, 300, 136), bf16(g, 264, 136, std=0.1), bf16(g, 136, 264, std=0.1)
    clean = [linear_act(x, w), gated_ffn(x, w, w, wd)]
    x[37, 5], x[299, 135], x[128, 0] = float("nan"), float("inf"), float("-inf")
    rest = torch.ones(300, dtype=torch.bool)
    rest[[37, 299, 128]] = False
    for got, ref in zip([linear_act(x, w), gated_ffn(x, w, w, wd)], clean):
        assert torch.equal(got[rest], ref[rest]) and not torch.isfinite(got[~rest]).any()
    # the gradient of a bad row reaches every weight, and no other row's input gradient
    for fn in (lambda t: linear_act(t, w, None, None, "silu"), lambda t: gated_ffn(t, w, w, wd)):
        t = x.clone().requires_grad_()
        dx, = torch.autograd.grad(fn(t).sum(), t)
        assert torch.isfinite(dx[rest]).all() and torch.isnan(dx[~rest]).any(1).all()


def test_large_values_do_not_overflow_the_activations():
    from transformer_amd import linear_act
    x = torch.tensor([[1.0] + [0.0] * 7, [-1.0] + [0.0] * 7], device=DEV).bfloat16()
    w = torch.zeros(8, 8, device=DEV).bfloat16()
    w[:, 0] = torch.tensor([1e-30, 1.0, 30.0, 100.0, 1000.0, 1e5, 1e10, 1e12], device=DEV)
    for act in ("silu", "gelu_tanh", "relu"):
        xs = x.clone().requires_grad_()
        y = linear_act(xs, w, None, None, act)
        z = x.double() @ w.double().t()
        # (far below 0 a sigmoid underflows: its product with z is off by less than 2^-126 |z|)
        assert ((y.double() - act64(z, act)).abs() <= act64(z, act).abs() * EPS16 * 1.1 + z.abs() * 2.0 ** -60).all(), act
        dx, = torch.autograd.grad(y, xs, torch.ones_like(y))
        assert torch.isfinite(dx).all(), act


def test_no_rows():
    from transformer_amd import gated_ffn, linear_act
    z = lambda *s: torch.zeros(*s, device=DEV).bfloat16().requires_grad_()
    x, w, wd, b = z(0, 16), z(24, 16), z(16, 24), z(24)
    y = linear_act(x, w, b, None, "silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == (0, 24) and dx.shape == x.shape and not dw.any() and not db.any()
    y = gated_ffn(x, w, w, wd)
    assert y.shape == (0, 16)
    assert all(not t.any() for t in torch.autograd.grad(y, (w, wd), torch.zeros_like(y)))


@pytest.mark.parametrize("frozen", ["x", "wg", "wu", "wd", "all weights", "wg and x"])
def test_only_needed_gradients_are_formed(frozen):
    from transformer_amd import gated_ffn
    g = gen("frozen")
    t = {"x": bf16(g, 70, 72), "wg": bf16(g, 136, 72, std=0.1), "wu": bf16(g, 136, 72, std=0.1), "wd": bf16(g, 72, 136, std=0.1)}
    dy = bf16(g, 70, 72)
    full = torch.autograd.grad(gated_ffn(*[v.requires_grad_() for v in t.values()]), tuple(t.values()), dy)
    off = {"all weights": ("wg", "wu", "wd"), "wg and x": ("wg", "x")}.get(frozen, (frozen,))
    part = {k: v.detach().requires_grad_(k not in off) for k, v in t.items()}
    gated_ffn(*part.values()).backward(dy)
    for (k, v), f in zip(part.items(), full):
        assert (v.grad is None) if k in off else torch.equal(v.grad, f), k


def test_shared_weights_and_broadcast_inputs_sum_their_gradients():
    # one weight as gate and up projection, one residual row for all: their gradients are sums
    from transformer_amd import gated_ffn
    g = gen("shared")
    x, w, wd, r = bf16(g, 70, 72), bf16(g, 136, 72, std=0.1), bf16(g, 72, 136, std=0.1), bf16(g, 72)
    dy = bf16(g, 70, 72)
    w1, w2 = w.clone().requires_grad_(), w.clone().requires_grad_()
    a, b = torch.autograd.grad(gated_ffn(x, w1, w2, wd), (w1, w2), dy)
    w.requires_grad_(), r.requires_grad_()
    dw, dr = torch.autograd.grad(gated_ffn(x, w, w, wd, r.expand(70, 72)), (w, r), dy)
    assert torch.equal(dw, a + b)
    # torch's sum of 70 bf16 rows in fp32, rounded once
    assert ((dr.double() - dy.double().sum(0)).abs() <= dy.double().abs().sum(0) * 80 * EPS32 + dy.double().sum(0).abs() * EPS16).all()


def test_autocast_fp32_weights_and_residual_stream():
    from transformer_amd import SwiGLU, linear_act
    torch.manual_seed(3)
    with torch.device(DEV):
        m = SwiGLU(136, 264)
    x, r = torch.randn(3, 40, 136, device=DEV, requires_grad=True), torch.randn(3, 40, 136, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, r)
        z = linear_act(x, m.w1.weight, None, None, "silu")
    assert y.dtype == torch.float32 and z.dtype == torch.bfloat16  # the residual stream stays fp32, as torch's sum leaves it
    dy = torch.randn_like(y)
    y.backward(dy)
    w = [m.w1.weight, m.w3.weight, m.w2.weight]
    assert all(p.grad.dtype == torch.float32 for p in w) and x.grad.dtype == torch.float32
    x6, w6 = x.detach().bfloat16().double().view(-1, 136), [p.detach().bfloat16().double() for p in w]
    leaves = [t.requires_grad_() for t in (x6, *w6)]
    ref = ffn64(*leaves, r.detach().double().view(-1, 136), "silu")
    near(y.detach().view(-1, 136), ref.detach(), "y")
    grads = torch.autograd.grad(ref, leaves, dy.bfloat16().double().view(-1, 136))
    for got, want, k in zip((x.grad.view(-1, 136), *(p.grad for p in w)), grads, ("x", "w1", "w3", "w2")):
        near(got, want, k)
    assert torch.equal(r.grad, dy)


def test_module_layers_that_are_not_plain_run_as_they_are():
    from transformer_amd import SwiGLU
    torch.manual_seed(4)
    with torch.device(DEV):
        m = SwiGLU(72, 136).bfloat16()
    assert set(m.state_dict()) == {"w1.weight", "w2.weight", "w3.weight"}
    x, r = torch.randn(30, 72, device=DEV).bfloat16(), torch.randn(30, 72, device=DEV).bfloat16()
    with torch.no_grad():
        plain, calls = m(x, r), []
        h = m.w3.register_forward_hook(lambda *a: calls.append(1))
        hooked = m(x, r)
        h.remove()
        # torch rounds each product and the activation to bf16: five roundings of the hidden layer and the result
        assert calls and (hooked.double() - plain.double()).norm() <= 5 * 2.26e-3 * plain.double().norm()
        again = m(x, r)
        assert len(calls) == 1 and torch.equal(again, plain)


def test_replayed_graph_sees_new_inputs_and_weights():
    """Forward and backward captured into one graph, replayed with eager work between: each replay equals the eager result."""
    from transformer_amd import gated_ffn, linear_act
    g = gen("graph")
    M, H, D = 200, 264, 136
    make = lambda: [bf16(g, M, D), bf16(g, H, D, std=0.1), bf16(g, H, D, std=0.1), bf16(g, D, H, std=0.1), bf16(g, M, D),
                    bf16(g, H, std=0.5), bf16(g, M, D)]
    static = make()

    def step(x, wg, wu, wd, r, b, dy):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd, r, b)]
        x, wg, wu, wd, r, b = leaves
        y = gated_ffn(x, wg, wu, wd, r)
        z = linear_act(linear_act(y, wg, b, None, "gelu_tanh"), wd)
        return [y.detach(), *torch.autograd.grad(z, leaves, dy)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for _ in range(4):
        new = make()
        for t, v in zip(static, new):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step(*new)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_two_streams_at_once():
    from transformer_amd import gated_ffn
    g = gen("streams")
    sets = [[bf16(g, 700, 136), bf16(g, 264, 136, std=0.1), bf16(g, 264, 136, std=0.1), bf16(g, 136, 264, std=0.1)]
            for _ in range(2)]
    run = lambda t: gated_ffn(*t)
    want = [run(t) for t in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, t in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(run(t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_and_checkpointed_calls():
    from torch.utils.checkpoint import checkpoint
    from transformer_amd import gated_ffn, linear_act
    g = gen("compile")
    x, wg, wu, wd, b = (bf16(g, 50, 72), bf16(g, 136, 72, std=0.1), bf16(g, 136, 72, std=0.1), bf16(g, 72, 136, std=0.1),
                        bf16(g, 72))
    dy = bf16(g, 50, 72)

    def f(x, wg, wu, wd, b):
        return linear_act(gated_ffn(x, wg, wu, wd, x), wd[:, :72], b, None, "gelu_tanh")

    def grads(fn):
        leaves = [t.detach().clone().requires_grad_() for t in (x, wg, wu, wd, b)]
        y = fn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = grads(f)
    for fn in (lambda *a: checkpoint(f, *a, use_reentrant=False), torch.compile(f, backend="aot_eager", fullgraph=True)):
        assert all(torch.equal(a, c) for a, c in zip(grads(fn), want))


def test_refusals():
    from transformer_amd import gated_ffn, linear_act
    z = lambda *s, dt=torch.bfloat16, dev=DEV: torch.zeros(*s, dtype=dt, device=dev)
    x, w, wd = z(4, 16), z(24, 16), z(16, 24)
    for err, call in (
            (TypeError, lambda: linear_act(z(4, 16, dt=torch.float32), w)),
            (TypeError, lambda: linear_act(z(4, 16, dt=torch.float16), w)),
            (TypeError, lambda: linear_act(x, z(24, 16, dt=torch.float16))),
            (ValueError, lambda: linear_act(x, z(24, 24))),
            (ValueError, lambda: linear_act(x, z(20, 16))),
            (ValueError, lambda: linear_act(z(4, 12), z(24, 12))),
            (ValueError, lambda: linear_act(x, w, z(16))),
            (ValueError, lambda: linear_act(x, w, None, z(4, 16))),
            (TypeError, lambda: linear_act(x, w, None, z(4, 24, dt=torch.float32))),
            (ValueError, lambda: linear_act(x, w, None, None, "swish")),
            (RuntimeError, lambda: linear_act(x.cpu(), w)),
            (ValueError, lambda: gated_ffn(x, w, z(32, 16), wd)),
            (ValueError, lambda: gated_ffn(x, w, w, w)),
            (ValueError, lambda: gated_ffn(x, w, w, wd, None, "none")),
            (ValueError, lambda: gated_ffn(x, w, w, wd, z(4, 24))),
            (RuntimeError, lambda: gated_ffn(x.cpu(), w, w, wd))):
        with pytest.raises(err):
            call()
