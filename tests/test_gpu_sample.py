"""sample_tokens on the GPU against numpy in 64 bits.  Tokens have to be equal: a weight is off by at most 2^-39 of itself and 2^-45
of the largest, sums S of V of them by 2^-39 S + V 2^-45, and a border of the choice and what is compared with it by twice that;
a row is asked only where no border is that near (none of the rows here is)."""
import math

import numpy as np
import pytest
import torch

import transformer_amd as T
from tests import sample_util

pytestmark = pytest.mark.gpu


def check(x, u, settings, got, strict=True):
    """``settings``: (temperature, top_k, top_p, min_p), each a number or a list of rows."""
    tokens, logprobs = got[0].cpu(), got[1].double().cpu()
    B, V = x.shape
    xs, us = x.double().cpu().numpy(), u.double().cpu().numpy()
    for b in range(B):
        s = [float(np.float32(v[b] if isinstance(v, (list, tuple)) else v)) for v in settings]
        token, logprob, room = sample_util.draw(xs[b], us[b], s[0], int(s[1]), s[2], s[3])
        # (weights of 1 add up exactly on both sides: a border met exactly is met by both)
        assert room > 4 or (not strict and room == 0), (b, room)
        assert int(tokens[b]) == token, (b, int(tokens[b]), token, s)
        # one rounding to fp32; the sum, 1 or more, relative to itself
        tol = 2.0 ** -24 * abs(logprob) + 2.0 ** -38 + V * 2.0 ** -44 if token >= 0 else 0.0
        assert logprobs[b] == logprob or abs(float(logprobs[b]) - logprob) <= tol, (b, float(logprobs[b]), logprob)


def rows(t, dtype=torch.float32):
    return torch.tensor(t, dtype=dtype, device="cuda") if isinstance(t, (list, tuple)) else t


def ask(x, u, settings):
    t, k, p, m = settings
    return T.sample_tokens(x, u, temperature=rows(t), top_k=rows(k, torch.int32), top_p=rows(p), min_p=rows(m))


def logits(B, V, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, V, generator=g) * spread).to(dtype).cuda(), torch.rand(B, generator=g).cuda()


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (1.0, 1, 1.0, 0.0), (0.0, 0, 0.3, 0.0),
            (1.5, 400, 0.99, 0.001), (2.0, 5000, 1.0, 0.0), (0.3, 0, 0.999, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 7, 0.5, 0.5)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 63), (5, 1000), (3, 1024), (4, 4099), (2, 32768), (1, 50257), (1, 131071)])
def test_tokens_and_logprobs(dtype, B, V):
    for i, settings in enumerate(SETTINGS):
        x, u = logits(B, V, dtype, 31 * V + i)
        check(x, u, settings, ask(x, u, settings))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_each_row_with_its_own_settings(dtype):
    n = len(SETTINGS)
    x, u = logits(3 * n, 32768, dtype, 5)
    settings = [[s[i] for s in SETTINGS] * 3 for i in range(4)]
    check(x, u, settings, ask(x, u, settings))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_draws_cover_the_rows(dtype):
    """The whole range of u over one small distribution: each token where its part of the sum lies."""
    x, _ = logits(1, 40, dtype, 3)
    u = (torch.arange(512).float() + 0.37) / 512
    x = x.expand(512, 40)
    for settings in ((1.0, 0, 1.0, 0.0), (1.0, 9, 0.9, 0.0)):
        check(x, u, settings, ask(x, u.cuda(), settings))


def test_ties_go_to_the_lowest_index():
    V = 5000
    x = torch.zeros(6, V)
    x[1, 100:] = -1.0
    x[2, 7::11] = 2.0
    x[3] = -0.0
    x[3, 1::2] = 0.0  # equal to -0
    x[4, 4000:] = 5.0
    x[5, :] = -3e38
    u = torch.tensor([0.999, 0.5, 0.7, 0.9, 0.31, 0.6])
    for settings in ((1.0, 10, 1.0, 0.0), (1.0, 0, 0.3, 0.0), (1.0, 600, 0.501, 0.0), (1.0, 1, 1.0, 0.0), (0.0, 0, 1.0, 0.0),
                     (1.0, 4999, 0.9999, 0.0)):
        for dtype in (torch.float32, torch.bfloat16):
            check(x.to(dtype), u, settings, ask(x.to(dtype).cuda(), u.cuda(), settings), strict=False)


def test_masks_infinities_and_nans():
    V = 3000
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, V, generator=g) * 2
    x[0] = -math.inf  # nothing is left
    x[1] = -math.inf
    x[1, 2999] = -4.0  # one token
    x[2, ::2] = math.nan
    x[3, 5], x[3, 900] = math.inf, math.inf
    x[4, :] = math.nan
    x[5, 40:] = -math.inf
    x[6, 17] = math.nan
    x[7] = torch.finfo(torch.float32).min
    x[7, 3] = 1.0
    u = torch.tensor([0.3, 0.9, 0.44, 0.7, 0.1, 0.99, 0.5, 0.2])
    for settings in SETTINGS:
        for dtype in (torch.float32, torch.bfloat16):
            check(x.to(dtype), u, settings, ask(x.to(dtype).cuda(), u.cuda(), settings), strict=False)


def test_settings_at_their_ends():
    x, _ = logits(4, 700, torch.float32, 9)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 0.25, 0.75]).cuda()
    first = x.cpu().double().argmax(1)
    # u = 0 takes the first token kept; the last, the last one
    got, _ = T.sample_tokens(x, u, top_k=5)
    best = x.cpu().topk(5, 1).indices.sort(1).values
    assert int(got[0]) == int(best[0, 0]) and int(got[1]) == int(best[1, -1])
    for kw in (dict(min_p=1.0), dict(min_p=7.0), dict(top_p=-1.0), dict(top_k=1), dict(temperature=-2.0), dict(temperature=1e-30)):
        got, lp = T.sample_tokens(x, u, **kw)
        assert got.cpu().tolist() == first.tolist() and (lp == 0).all(), kw
    # a temperature without end: all alike
    got, lp = T.sample_tokens(x, u, temperature=math.inf)
    assert got.cpu().tolist() == [0, 699, 175, 525] and torch.allclose(lp, torch.full_like(lp, -math.log(700)), rtol=2.0 ** -23, atol=0)
    for a, b in ((dict(top_k=0), dict(top_k=-4)), (dict(top_k=700), dict(top_k=1 << 30)), (dict(top_p=1.0), dict(top_p=9.0))):
        one, two = T.sample_tokens(x, u, **a), T.sample_tokens(x, u, **b)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_rows_of_any_stride_and_alignment():
    full, u = logits(6, 2100, torch.bfloat16, 12)
    settings = (0.9, 40, 0.95, 0.0)
    for x in (full[:, 1:2000], full[:, 3:2000], full[::2, 8:1999], full[2:3, 5:70], full[:, :1000].flip(1), full.t()[:6, :6],
              full[:1, :900].expand(6, 900)):
        check(x, u[:x.size(0)], settings, ask(x, u[:x.size(0)], settings))


def test_the_same_again_in_a_graph_and_on_another_stream():
    x, u = logits(9, 32768, torch.bfloat16, 4)
    settings = (0.8, 50, 0.95, 0.0)
    ask(x, u, settings)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ask(x, u, settings)
    for i in range(3):
        nx, nu = logits(9, 32768, torch.bfloat16, 40 + i)
        x.copy_(nx)
        u.copy_(nu)
        graph.replay()
        check(nx, nu, settings, out)
        eager = ask(x, u, settings)
        assert torch.equal(eager[0], out[0]) and torch.equal(eager[1], out[1])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = ask(x, u, settings)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(eager[0], again[0]) and torch.equal(eager[1], again[1])


def test_operator_checks_and_empty_batches():
    x, u = logits(2, 300, torch.float32, 1)
    torch.library.opcheck(torch.ops.mla_mi355x.sample_tokens, (x, u, 1.0, 5, 0.9, 0.0, None, None, None, None),
                          test_utils=("test_schema", "test_faketensor"))
    tokens, logprobs = T.sample_tokens(x[:0], u[:0])
    assert tokens.shape == (0,) and tokens.dtype == torch.int64 and logprobs.shape == (0,)
