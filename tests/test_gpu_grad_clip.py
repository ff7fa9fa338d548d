"""clip_grad_norm_ and grad_norm against 64 bits.

The squares are summed in fp64 and the norm rounded to fp32 once: off by 2^-24 of it (and n 2^-53, nothing).  The factor is
formed in fp64 and rounded to fp32, each product rounded once more to fp32 and, for bf16 gradients, once to bf16: off by at
most 2 x 2^-24, and 2^-8 more in bf16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS32, EPS16 = 2.0 ** -24, 2.0 ** -8


def params(grads):
    out = []
    for t in grads:
        p = torch.nn.Parameter(torch.empty(t.shape, dtype=t.dtype, device=t.device))
        p.grad = t
        out.append(p)
    return out


def norm64(grads, kind):
    flat = torch.cat([t.double().reshape(-1) for t in grads])
    return flat.abs().max() if kind == math.inf else flat.square().sum().sqrt()


def check(grads, max_norm, kind=2.0):
    from transformer_amd import clip_grad_norm_, grad_norm
    before = [t.clone() for t in grads]
    alone = grad_norm(grads, kind)
    norm = clip_grad_norm_(params(grads), max_norm, kind)
    want = norm64(before, kind)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and torch.equal(norm, alone)
    assert (norm.double() - want).abs() <= want * EPS32 * 1.01, (norm.item(), want.item())
    factor = min(1.0, max_norm / (want.item() + 1e-6))
    for got, b in zip(grads, before):
        ref = b.double() * factor
        tol = ref.abs() * (3 * EPS32 + (EPS16 * 1.01 if b.dtype == torch.bfloat16 else 0)) + 2.0 ** -149
        assert ((got.double() - ref).abs() <= tol).all()
        if factor == 1.0:
            assert torch.equal(got, b)
    return norm


def make(sizes, dtypes=(torch.float32,), seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("sizes", [[1], [3], [4, 5], [7, 8, 9], [0, 1, 0], [16384], [16385, 1], [16383, 32769, 100000],
                                   [1000003], [(1 << 20) + 5, 3, (1 << 18) - 1]])
def test_sizes_and_types(sizes, dtypes, kind):
    grads = make(sizes, dtypes)
    check(grads, 0.5 * norm64(grads, kind).item(), kind)
    check(make(sizes, dtypes, 1), 1e6, kind)  # not clipped: unchanged


@pytest.mark.parametrize("n", [127, 128, 129, 257, 400])
def test_many_tensors(n):
    # beyond a launch's 128, sizes and types mixed, some without elements
    check(make([(37 * i * i) % 5003 for i in range(n)], (torch.float32, torch.float32, torch.bfloat16), n), 1.0)


def test_views_at_every_alignment():
    g = torch.Generator(device=DEV).manual_seed(5)
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.randn(40000, generator=g, device=DEV).to(dt)
        keep = buf.clone()
        views, mask, at = [], torch.ones(40000, dtype=torch.bool, device=DEV), 0
        for i, n in enumerate([1, 2, 3, 5, 7, 8, 9, 15, 17, 33, 100, 1001, 4097, 16390]):
            views.append(buf[at:at + n])
            mask[at:at + n] = False
            at += n + 1 + i % 3  # gaps of one to three elements
        check(views, 2.0)
        assert torch.equal(buf[mask], keep[mask]), "elements between the gradients were changed"


def test_layouts():
    g = torch.Generator(device=DEV).manual_seed(6)
    base = torch.randn(64, 96, generator=g, device=DEV)
    check([base.t(), torch.randn(3, 4, 5, generator=g, device=DEV).permute(2, 0, 1), torch.randn(7, 40, generator=g, device=DEV)[:, 3:17],
           torch.randn((), generator=g, device=DEV)], 1.0)


def test_bucket_views_of_one_buffer():
    flat = make([10000])[0]
    check([flat[:4000].view(40, 100), flat[4000:4001], flat[4001:10000]], 3.0)


def test_large_and_small_values():
    # squares that overflow or vanish in fp32 do neither here
    big = [torch.tensor([3e30, -4e30], device=DEV), torch.tensor([1.0], device=DEV)]
    assert check(big, 1.0).item() == pytest.approx(5e30, rel=2e-7)
    small = [torch.full((1000,), 1e-30, device=DEV)]
    assert check(small, 1.0).item() == pytest.approx(1e-30 * 1000 ** 0.5, rel=2e-7)
    check([torch.zeros(100, device=DEV)], 1.0)
    zeroed = make([1000])
    check(zeroed, 0.0)
    assert not zeroed[0].any()


@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_nan_and_infinity(kind):
    from transformer_amd import clip_grad_norm_
    for bad in (float("nan"), float("inf"), float("-inf")):
        for at in (0, 777, 99999):
            grads = make([5, 100000, 8])
            before = [t.clone() for t in grads]
            grads[1][at] = bad
            with pytest.raises(RuntimeError, match="non-finite"):
                clip_grad_norm_(params(grads), 1.0, kind, error_if_nonfinite=True)
            assert torch.equal(grads[0], before[0])  # nothing was scaled
            norm = clip_grad_norm_(params(grads), 1.0, kind)
            if math.isnan(bad):
                assert torch.isnan(norm) and all(torch.isnan(t).all() for t in grads)
            else:  # a factor of 0: zeros, and 0 x inf
                assert torch.isinf(norm) and torch.isnan(grads[1][at]) and not grads[0].any() and not grads[2].any()


def test_results_repeat_and_equal_torchs():
    from transformer_amd import clip_grad_norm_
    a, b, c = (make([1000, 300001, 17], (torch.float32, torch.bfloat16), 9) for _ in range(3))
    na, nb = clip_grad_norm_(params(a), 1.0), clip_grad_norm_(params(b), 1.0)
    assert torch.equal(na, nb) and all(torch.equal(x, y) for x, y in zip(a, b))
    nc = torch.nn.utils.clip_grad_norm_(params([t.double() for t in c]), 1.0)
    assert (na.double() - nc).abs() <= nc * EPS32 * 1.01


def test_parameters_without_gradients_and_versions():
    from transformer_amd import clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(4, device=DEV))
    assert clip_grad_norm_([p], 1.0).item() == 0.0 and clip_grad_norm_([], 1.0).item() == 0.0 and grad_norm([]).item() == 0.0
    p.grad = torch.ones(4, device=DEV)
    v = p.grad._version
    assert clip_grad_norm_(p, 1.0).item() == 2.0 and p.grad._version > v
    assert clip_grad_norm_((q for q in [p]), 10.0, foreach=True).item() == pytest.approx(1.0, rel=1e-6)


def test_captured_and_replayed():
    from transformer_amd import clip_grad_norm_
    grads = make([5000, 33, 70000], (torch.float32, torch.bfloat16))
    ps = params(grads)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        clip_grad_norm_(ps, 1.0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ps, 1.0)
    for i in range(4):
        new = make([5000, 33, 70000], (torch.float32, torch.bfloat16), 20 + i, 0.5 + i)
        for t, v in zip(grads, new):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = norm.clone()
        want = clip_grad_norm_(params(new), 1.0)
        assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(grads, new))


def test_two_streams_at_once():
    from transformer_amd import clip_grad_norm_
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(3):
        sets = [make([200000, 77, 3000], seed=rep * 2 + i) for i in range(2)]
        copies = [[t.clone() for t in s] for s in sets]
        want = [clip_grad_norm_(params(s), 1.0) for s in copies]
        torch.cuda.synchronize()
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(clip_grad_norm_(params(s), 1.0))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(x, y) for a, b in zip(sets, copies) for x, y in zip(a, b))


def test_refusals():
    from transformer_amd import clip_grad_norm_, grad_norm
    one = torch.ones(8, device=DEV)
    for err, call in ((ValueError, lambda: clip_grad_norm_(params([one]), -1.0)),
                      (ValueError, lambda: clip_grad_norm_(params([one]), float("nan"))),
                      (ValueError, lambda: clip_grad_norm_(params([one]), 1.0, 1.0)),
                      (TypeError, lambda: clip_grad_norm_(params([one.half()]), 1.0)),
                      (ValueError, lambda: clip_grad_norm_(params([torch.ones(1, device=DEV).expand(8)]), 1.0)),
                      (RuntimeError, lambda: clip_grad_norm_(params([one.cpu()]), 1.0)),
                      (RuntimeError, lambda: clip_grad_norm_(params([one, one]), 1.0)),        # the same gradient twice
                      (RuntimeError, lambda: clip_grad_norm_(params([one[:5], one[4:]]), 1.0)),  # overlapping ones
                      (TypeError, lambda: grad_norm([one.double()]))):
        with pytest.raises(err):
            call()
    assert torch.equal(one, torch.ones(8, device=DEV))


def test_a_training_step_of_a_block():
    """The operators as a step uses them: norm, gated block with the residual stream, loss, backward, clipping of the whole
    list, against the same step in 64 bits.  Rounding to bf16 happens at the normalised rows, the hidden layer, the block's
    output, its gradients (2 passes) and the weights' gradients: at most 7 roundings that add up in quadrature for any of
    them, each 2.26e-3 of the norm."""
    from transformer_amd import RMSNorm, SwiGLU, clip_grad_norm_
    torch.manual_seed(11)
    with torch.device(DEV):
        norm, ffn = RMSNorm(136), SwiGLU(136, 264).bfloat16()
    x = torch.randn(90, 136, device=DEV).bfloat16()
    target = torch.randn(90, 136, device=DEV)
    y = ffn(norm(x), x)
    (y.float() - target).square().mean().backward()
    ps = [*norm.parameters(), *ffn.parameters()]
    raw = [p.grad.clone() for p in ps]
    total = clip_grad_norm_(ps, 0.01)

    w = [p.detach().double().requires_grad_() for p in ps]
    x6 = x.double()
    n = x6 * torch.rsqrt(x6.square().mean(-1, keepdim=True) + 1e-6) * w[0]
    g, u = n @ w[1].t(), n @ w[3].t()
    loss = ((g * torch.sigmoid(g) * u) @ w[2].t() + x6 - target.double()).square().mean()
    ref = torch.autograd.grad(loss, w)
    want = torch.cat([r.reshape(-1) for r in ref]).norm()
    bound = 7 ** 0.5 * 2.26e-3
    assert (total.double() - want).abs() <= bound * want
    for p, r, f in zip(ps, raw, ref):
        assert (r.double() - f).norm() <= bound * f.norm()
        assert ((p.grad.double() - r.double() * (0.01 / (total.double() + 1e-6))).abs()
                <= r.double().abs() * (0.01 / total.double()) * (4 * EPS32 + (EPS16 if r.dtype == torch.bfloat16 else 0))).all()


def test_sparse_and_overlapping_layouts_are_refused_before_anything_is_scaled():
    from transformer_amd import clip_grad_norm_
    one = torch.ones(4, 4, device=DEV)
    p = torch.nn.Parameter(torch.zeros(4, 4, device=DEV))
    p.grad = torch.eye(4, device=DEV).to_sparse()
    with pytest.raises(ValueError):
        clip_grad_norm_([*params([one]), p], 1.0)
    with pytest.raises(ValueError):
        clip_grad_norm_(params([one, torch.ones(4, device=DEV).expand(3, 4)]), 1.0)
    buf = torch.ones(6, device=DEV)
    with pytest.raises(ValueError):  # rows that overlap
        clip_grad_norm_(params([buf.as_strided((3, 4), (1, 1))]), 1.0)
    assert torch.equal(one, torch.ones(4, 4, device=DEV))
