"""sample_tokens on rows that are no plain draw of numbers, in each of its kernels (up to 8192 logits, up to 32768, and longer ones that
every pass reads again): infinities, NaN, masks, ties across the border of a choice, rows so flat that a bin holds more than a list.
Compared as in tests/test_gpu_sample.py: tokens equal, wherever no border is so near that roundings decide, which each test shows of
nearly all its rows."""
import math

import numpy as np
import pytest
import torch

import transformer_amd as T
from tests import sample_util

pytestmark = pytest.mark.gpu
LENGTHS = [700, 4099, 20003, 32768, 32771, 100003]
SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (0.0, 0, 0.3, 0.0), (1.5, 400, 0.99, 0.001),
            (2.0, 600, 0.7, 0.0), (0.3, 0, 0.999, 0.0), (1.0, 7, 0.5, 0.5), (1.3, 0, 1.0, 0.05), (50.0, 0, 0.4, 0.0), (1e6, 5000, 0.6, 0.0),
            (math.inf, 0, 0.55, 0.0)]


def special_rows(V, g):
    """{name: row}"""
    n = lambda std=2.0: torch.randn(V, generator=g) * std
    rows = {}
    x = n()
    x[5], x[V // 2], x[V - 1] = math.inf, math.inf, math.inf
    rows["infinities"] = x
    x = n()
    x[1:] = torch.where(torch.rand(V - 1, generator=g) < 0.5, math.inf, x[1:])
    rows["infinities in half of it"] = x
    rows["nothing"] = torch.full((V,), -math.inf)
    rows["NaN alone"] = torch.full((V,), math.nan)
    x = torch.full((V,), -math.inf)
    x[V - 1] = -4.0
    rows["one token"] = x
    x = torch.full((V,), -math.inf)
    x[3], x[V - 2] = math.nan, math.inf
    rows["one infinity"] = x
    x = n()
    x[::2] = math.nan
    rows["NaN in every second place"] = x
    rows["masked"] = n().masked_fill(torch.rand(V, generator=g) < 0.98, -math.inf)
    x = torch.full((V,), torch.finfo(torch.float32).min)
    x[3], x[V - 3] = 1.0, 0.5
    rows["the lowest value as a mask"] = x
    rows["all equal"] = torch.full((V,), 2.5)
    x = torch.zeros(V)
    x[::2] = -0.0
    rows["zeros of both signs"] = x
    x = torch.full((V,), -1.0)
    x[7::11] = 2.0
    rows["two values"] = x
    rows["a few values"] = torch.randint(5, (V,), generator=g).float() / 4
    rows["flat"] = n(1e-3)
    rows["steep"] = n(30.0)
    x = n()
    x[V // 3] = 40.0
    rows["nearly certain"] = x
    rows["rising"] = torch.arange(V).float() / V
    rows["far below"] = n() - 3e38
    return rows


def ask(x, u, settings):
    t, k, p, m = settings
    return T.sample_tokens(x, u, temperature=t, top_k=k, top_p=p, min_p=m)


def check(x, u, settings, got, share=0.9):
    """A row whose border is met exactly (room 0) is compared where the weights are exact on both sides (all 1), and has a token with a
    weight otherwise."""
    tokens, logprobs = got[0].cpu(), got[1].double().cpu()
    xs, us, V = x.double().cpu().numpy(), u.double().cpu().numpy(), x.size(1)
    s = [float(np.float32(v)) for v in settings]
    if s[0] == math.inf:  # (the same weights, without the oracle's infinity over infinity: a difference of up to 2^129 over 1e300)
        s[0] = 1e300
    compared = 0
    for b in range(x.size(0)):
        token, logprob, room = sample_util.draw(xs[b], us[b], s[0], int(s[1]), s[2], s[3])
        got_token, got_logprob = int(tokens[b]), float(logprobs[b])
        if room <= 4:
            assert -1 <= got_token < V and (token < 0) == (got_token < 0), (b, settings)
            continue
        compared += 1
        assert got_token == token, (b, got_token, token, settings)
        # one rounding to fp32; the sum, 1 or more, relative to itself
        tol = 2.0 ** -24 * abs(logprob) + 2.0 ** -38 + V * 2.0 ** -44 if token >= 0 else 0.0
        assert got_logprob == logprob or abs(got_logprob - logprob) <= tol, (b, got_logprob, logprob)
    assert compared >= share * x.size(0), (compared, x.size(0), settings)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", LENGTHS)
def test_special_rows(V, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.stack(list(special_rows(V, g).values())).to(dtype)
    u = (torch.rand(x.size(0), generator=g) * 0.98 + 0.01)
    for settings in SETTINGS:
        check(x, u, settings, ask(x.cuda(), u.cuda(), settings))


@pytest.mark.parametrize("V", [4099, 20003, 40000])
def test_ties_across_a_border(V):
    """top_k and top_p end inside a run of equal logits, wherever it begins: the lower indices stay."""
    for values in ((3.0, 3.0), (1.0, 3.0)):
        x = torch.full((1, V), -50.0)
        x[0, V // 5::3] = values[0]
        x[0, V // 2::7] = values[1]
        top = (x[0] == x.max()).nonzero().flatten()
        for k in (2, 100, 513, 700, top.numel() - 1):
            if k > top.numel():  # (the run of equal ones is the border's)
                continue
            for u in (0.0, 0.37, 1 - 2.0 ** -24):
                token, logprob = ask(x.cuda(), torch.tensor([u]).cuda(), (1.0, k, 1.0, 0.0))
                assert int(token) == int(top[min(k - 1, int(np.float64(np.float32(u)) * k))]), (values, k, u)
                assert abs(float(logprob) + math.log(k)) <= 2.0 ** -23 * math.log(k)
        # the first of n equal ones that hold half of their weight: ceil(n / 2)
        token, _ = ask(x.cuda(), torch.tensor([1 - 2.0 ** -24]).cuda(), (0.01, 0, 0.5, 0.0))
        assert int(token) == int(top[(top.numel() + 1) // 2 - 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("head", [0, 1, 3])
def test_the_longest_rows_and_any_beginning(dtype, head):
    V = 1 << 19
    g = torch.Generator().manual_seed(13 + head)
    x = (torch.randn(2, V, generator=g) * 2).to(dtype)
    wide = torch.zeros(2, V + 5, dtype=dtype)
    wide[:, head:V + head] = x
    u = torch.tensor([0.3, 0.999])
    for settings in ((0.9, 0, 1.0, 0.0), (1.0, 3000, 0.8, 0.0), (1.5, 0, 0.99, 0.001), (1.0, 40, 0.9, 0.0)):
        check(x, u, settings, ask(wide.cuda()[:, head:V + head], u.cuda(), settings), share=1.0)


def test_a_flat_row_of_the_greatest_length():
    """2^19 weights of 2^44 add up to 2^63."""
    V = 1 << 19
    x = torch.full((3, V), 1.25, device="cuda")
    u = torch.tensor([0.0, 0.5, 1 - 2.0 ** -24], device="cuda")
    tokens, logprobs = ask(x, u, (1.0, 0, 1.0, 0.0))
    assert tokens.tolist() == [0, V // 2, V - 1] and (logprobs + math.log(V)).abs().max() <= 2.0 ** -20
    tokens, logprobs = ask(x, u, (1.0, 0, 0.25, 0.0))
    assert tokens.tolist() == [0, V // 8, V // 4 - 1] and (logprobs + math.log(V // 4)).abs().max() <= 2.0 ** -20
    tokens, _ = ask(x, u, (1.0, V - 1, 1.0, 0.0))
    assert tokens.tolist() == [0, int(0.5 * (V - 1)), V - 2]


@pytest.mark.parametrize("V", [700, 20003, 40000])
def test_logits_as_far_apart_as_fp32_has_them(V):
    """Differences past fp32's largest number, at temperatures at which they count."""
    g = torch.Generator().manual_seed(V)
    x = (torch.rand(4, V, generator=g) * 2 - 1) * 3.3e38
    x[1, 7:] = -3.3e38
    x[2] = torch.where(torch.rand(V, generator=g) < 0.5, 3.4e38, -3.4e38)
    x[3, 5] = math.nan
    u = torch.tensor([0.3, 0.6, 0.9, 0.5])
    for settings in ((1e38, 0, 0.9, 0.0), (3e38, 5, 1.0, 0.0), (3e38, V - 2, 0.7, 0.0), (2e38, 0, 1.0, 0.1), (math.inf, 0, 0.9, 0.0)):
        check(x, u, settings, ask(x.cuda(), u.cuda(), settings), share=0.75)  # (u = 0.5 of an even number of equal weights: a border)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 20003, 40000])
def test_rows_of_the_lowest_value(V, dtype):
    """A mask of the type's lowest value over everything, over all but a few, and with -inf beside it."""
    low = torch.finfo(dtype).min
    x = torch.full((4, V), low, dtype=dtype)
    x[1, V // 2:] = -math.inf
    x[2, 9] = 0.0
    x[3, ::3] = math.nan
    u = torch.tensor([0.71, 0.43, 0.9, 0.31])
    for settings in ((1.0, 0, 0.55, 0.0), (0.5, 600, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 30, 1.0, 0.0), (1.0, V - 1, 0.37, 0.2),
                     (math.inf, 0, 0.81, 0.0)):
        check(x, u, settings, ask(x.cuda(), u.cuda(), settings), share=0.75)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [8188, 8189, 8190, 8192, 8193, 32764, 32765, 32767, 32768, 32769, 65537])
@pytest.mark.parametrize("head", [0, 1, 2])
def test_lengths_about_the_kernels_ends(V, head, dtype):
    """Rows that begin in any place of a quad, where one kernel takes over from another; settings of each row's own."""
    g = torch.Generator().manual_seed(V + head)
    B = 6
    wide = torch.full((B, V + 6), 77.0).to(dtype)  # (what is read of it would win)
    x = (torch.randn(B, V, generator=g) * torch.tensor([0.05, 0.5, 1.0, 2.0, 4.0, 9.0])[:, None]).to(dtype)
    wide[:, head:head + V] = x
    u = torch.rand(B, generator=g)
    t, k = torch.rand(B, generator=g) * 1.5 + 0.1, torch.tensor([0, 3, 64, 300, 513, 5000], dtype=torch.int32)[torch.randperm(B, generator=g)]
    p, m = torch.rand(B, generator=g) * 0.6 + 0.4, torch.tensor([0.0, 0.0, 0.001, 0.02, 0.3, 1.0])[torch.randperm(B, generator=g)]
    got = T.sample_tokens(wide.cuda()[:, head:head + V], u.cuda(), t.cuda(), k.cuda(), p.cuda(), m.cuda())
    for b in range(B):
        check(x[b:b + 1], u[b:b + 1], (float(t[b]), int(k[b]), float(p[b]), float(m[b])), (got[0][b:b + 1], got[1][b:b + 1]), share=1.0)
