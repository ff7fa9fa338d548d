"""The serving operators as a program uses them together: prompts taken in parts, then a token a step for a changing set of
sequences, eagerly and in a recorded graph, against the plain operators in 64 bits (tests/paged_util.py, tests/sample_util.py)."""
import copy
import math

import numpy as np
import pytest
import torch

import transformer_amd as T
from tests import paged_util as U
from tests import sample_util
from tests.test_gpu_paged import LAYOUTS, check_cache, check_decode, i32, same_bits

pytestmark = pytest.mark.gpu
SCALE, VOCAB = 192 ** -0.5, 1000
OPS = torch.ops.mla_mi355x


class Model:
    """What lies around the operators: a token's rows from tables, logits from the first columns of a head's result."""

    def __init__(self, layout, bits, size, sequences, room, seed=0):
        self.H, self.Hr, self.DL = LAYOUTS[layout]
        g = torch.Generator().manual_seed(seed)
        self.cache = U.Cache(g, bits, self.DL, self.Hr, size, [room] * sequences)
        self.qk, self.c, self.ql = (U.normal(g, VOCAB, *s) for s in ((self.H + self.Hr, 64), (self.DL,), (self.H, self.DL)))
        self.out = U.normal(g, VOCAB, 128, std=0.5)
        self.cos, self.sin = U.tables(512)
        self.dev = self.cache.dev()
        for name in ("qk", "c", "ql", "out", "cos", "sin"):
            setattr(self, name + "_d", getattr(self, name).cuda())
        self.table = self.cache.table.cuda()

    def step(self, token, at, u, settings, dev=None):
        """One token of each sequence at position at: (q_rope, ctx, lse, logits, next token, its logprob)."""
        pages, scales = dev or self.dev
        q = T.paged_append(self.qk_d[token][:, None], self.c_d[token][:, None], pages, scales, self.cos_d, self.sin_d, self.table, at)
        ctx, lse = T.paged_decode(self.ql_d[token], q[:, 0], pages, scales, self.table, at + 1, SCALE)
        logits = OPS.linear_rows(ctx[:, 0, :128], self.out_d)
        return (q, ctx, lse, logits, *T.sample_tokens(logits, u, **settings))

    def check_step(self, token, at, got, u, settings):
        q, ctx, lse, logits, new, logprob = got
        token, at, B = token.tolist(), at.tolist(), len(token)
        want_q = U.append(self.cache, self.qk[token][:, None], self.c[token][:, None], self.cos, self.sin, at, None)
        assert same_bits(q, want_q)
        check_cache(self.dev, self.cache)
        check_decode(self.cache, self.ql[token], want_q[:, 0], [n + 1 for n in at], SCALE, (ctx, lse))
        x = logits.float().cpu().numpy()
        for b in range(B):
            s = {k: v if not isinstance(v, torch.Tensor) else v[b].item() for k, v in settings.items()}
            s = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **s}
            want, lp, room = sample_util.draw(x[b], np.float32(u[b].item()), np.float32(s["temperature"]), s["top_k"], np.float32(s["top_p"]),
                                              np.float32(s["min_p"]))
            if room > 1:
                assert int(new[b]) == want
                assert abs(float(logprob[b]) - lp) <= 2.0 ** -22 * max(1.0, abs(lp))


SETTINGS = [dict(temperature=0.8, top_k=50, top_p=0.95), dict(temperature=0.0), dict(min_p=0.05, top_p=0.9)]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout", ["baseline", "model", "one"])
def test_prompts_in_parts_and_then_token_by_token(bits, layout):
    m = Model(layout, bits, 16, 3, 96)
    g = torch.Generator().manual_seed(1)
    lens = [40, 17, 1]
    prompt = torch.randint(VOCAB, (3, 40), generator=g)
    for t0 in (0, 24):  # the prompts' first 24 tokens, then the others
        part = prompt[:, t0:t0 + 24]
        n = part.size(1)
        counts = [max(0, min(n, k - t0)) for k in lens]
        q = T.paged_append(m.qk_d[part.cuda()], m.c_d[part.cuda()], *m.dev, m.cos_d, m.sin_d, m.table, i32([t0] * 3), i32(counts))
        want = U.append(m.cache, m.qk[part], m.c[part], m.cos, m.sin, [t0] * 3, counts)
        assert same_bits(q, want)
        check_cache(m.dev, m.cache)
        # the attention of a part over all before it, of what paged_read takes out: row t sees positions up to t0 + t
        latent, k_rope = T.paged_read(*m.dev, m.table, m.DL, t0 + n, None, i32([t0 + c for c in counts]))
        rows = U.read(m.cache, t0 + n, None, [t0 + c for c in counts], 3)
        assert same_bits(latent, rows[0]) and same_bits(k_rope, rows[1])
        if m.Hr == 1 and m.DL in (128, 256, 384, 512):
            ctx, lse = OPS.prefill_cached(m.ql_d[part.cuda()], q, latent, k_rope, t0, SCALE)
            for t in (0, n - 1):  # a row of it is the decode of that many tokens
                one, one_lse = T.paged_decode(m.ql_d[part[:, t].cuda()], q[:, t], *m.dev, m.table, i32([t0 + t + 1] * 3), SCALE)
                full = torch.tensor([c > t for c in counts])
                check_decode(m.cache, m.ql[part[:, t]], want[:, t], [t0 + t + 1] * 3, SCALE, (one, one_lse))
                # both within bf16 roundings of p and of the result
                a, b = ctx[:, t].float().cpu()[full], one.float().cpu()[full]
                assert a.numel() == 0 or float((a - b).abs().max()) <= 4 * 2.0 ** -8 * float(b.abs().max())
    token, at = prompt[torch.arange(3), torch.tensor(lens) - 1], torch.tensor(lens, dtype=torch.int32)
    token = (token + 1) % VOCAB
    for i, settings in enumerate(SETTINGS * 2):
        u = torch.rand(3, generator=g)
        got = m.step(token.cuda(), at.cuda(), u.cuda(), settings)
        m.check_step(token, at, got, u, settings)
        token, at = got[4].cpu(), at + 1
        if i == 2:  # a sequence ends, and another takes its pages
            at[0] = 0
            order = torch.randperm(m.cache.table.size(1), generator=g)
            m.cache.table[0] = m.cache.table[0][order]
            m.table.copy_(m.cache.table)


@pytest.mark.parametrize("bits", [16, 4])
def test_two_recorded_loops_of_steps(bits):
    """Two graphs of a step, which share the memory pool of their workspaces, replayed in turn beside eager steps: the positions, tokens
    and settings of each replay are those in the buffers."""
    models = [Model("baseline", bits, 32, 4, 160, seed=s) for s in (3, 4)]
    buffers, graphs, outs, pool = [], [], [], None
    for m in models:
        b = dict(token=torch.zeros(4, dtype=torch.int64, device="cuda"), at=i32([0, 30, 64, 100]), u=torch.rand(4, device="cuda"))
        s = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.3], device="cuda"), top_k=i32([0, 50, 0, 3]),
                 top_p=torch.tensor([1.0, 0.9, 0.5, 1.0], device="cuda"), min_p=torch.tensor([0.0, 0.0, 0.05, 0.0], device="cuda"))
        scratch = [t if t is None else t.clone() for t in m.dev]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(b["token"], b["at"], b["u"], s, scratch)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(m.step(b["token"], b["at"], b["u"], s))
        pool = graph.pool()
        buffers.append((b, s))
        graphs.append(graph)
    g = torch.Generator().manual_seed(9)
    for i in range(4):
        for m, (b, s), graph, out in zip(models, buffers, graphs, outs):
            token, at, u = b["token"].cpu(), b["at"].cpu(), torch.rand(4, generator=g)
            b["u"].copy_(u)
            graph.replay()
            torch.cuda.synchronize()
            recorded = [t.clone() for t in out]
            eager = m.step(b["token"], b["at"], b["u"], s)  # the same token to the same place again
            for x, y in zip(recorded, eager):
                assert torch.equal(x, y)
            m.check_step(token, at, recorded, u, s)
            b["token"].copy_(recorded[4])
            b["at"].add_(1)
    for m in models:
        assert not math.isnan(float(m.dev[0].float().abs().max()))


def test_calls_on_two_streams_at_once():
    """Calls that may run at the same time have workspaces of their own."""
    m = Model("baseline", 4, 64, 6, 160, seed=5)
    lens = [150, 3, 0, 77, 64, 128]
    q = U.normal(torch.Generator().manual_seed(6), 2, 6, 16, 576).cuda()
    want = [T.paged_decode(q[i, ..., :512], q[i, ..., 512:], *m.dev, m.table, i32(lens), SCALE) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    n = i32(lens)
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, T.paged_decode(q[i, ..., :512], q[i, ..., 512:], *m.dev, m.table, n, SCALE)))
    torch.cuda.synchronize()
    for i, (c, l) in got:
        assert torch.equal(c, want[i][0]) and torch.equal(l, want[i][1])


def test_inputs_that_ask_for_gradients():
    """Nothing of a cache has a gradient: results of inputs that ask for one have none, or say so."""
    m = Model("baseline", 16, 16, 2, 32, seed=7)
    before = copy.deepcopy(m.cache)
    q = m.ql_d[:2].clone().requires_grad_()
    qr = m.qk_d[:2, :16].contiguous()
    ctx, _ = T.paged_decode(q, qr, *m.dev, m.table, i32([20, 3]), SCALE)
    plain, _ = T.paged_decode(q.detach(), qr, *m.dev, m.table, i32([20, 3]), SCALE)
    assert torch.equal(ctx.detach(), plain)
    if ctx.requires_grad:
        with pytest.raises(RuntimeError):
            ctx.float().sum().backward()
    assert q.grad is None
    check_cache(m.dev, before)
    # what was saved for a backward pass and is appended to since is noticed there
    pages = m.dev[0]
    x = torch.ones_like(pages, requires_grad=True)
    y = (x * pages).float().sum()
    with torch.no_grad():
        T.paged_append(m.qk_d[:2][:, None], m.c_d[:2][:, None], *m.dev, m.cos_d, m.sin_d, m.table, i32([20, 3]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("DL", [64, 128, 256, 384, 512])
@pytest.mark.parametrize("H,Hr", [(16, 1), (5, 5), (12, 12), (16, 16), (17, 17)])
def test_every_layout(H, Hr, DL, bits):
    """Each width with a shared key and with heads' own, fewer and more than a head group has."""
    lens = [200, 1, 64]
    g = torch.Generator().manual_seed(H + DL)
    cache = U.Cache(g, bits, DL, Hr, 48, lens)
    q_lat, q_rope = U.normal(g, 3, H, DL), U.normal(g, 3, H, 64)
    dev, table = cache.dev(), cache.table.cuda()
    got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *dev, table, i32(lens), SCALE)
    check_decode(cache, q_lat, q_rope, lens, SCALE, got)
    qk, c_new = U.normal(g, 3, 2, H + Hr, 64), U.normal(g, 3, 2, DL)
    cos, sin = U.tables(256)
    q = T.paged_append(qk.cuda(), c_new.cuda(), *dev, cos.cuda(), sin.cuda(), table, i32([5, 0, 40]))
    assert same_bits(q, U.append(cache, qk, c_new, cos, sin, [5, 0, 40], None))
    check_cache(dev, cache)


@pytest.mark.parametrize("bits", [16, 4])
def test_many_short_sequences(bits):
    """More sequences than workgroups, empty ones among them, several in a workgroup's run."""
    lens = [(7 * b * b + 3 * b) % 90 if b % 11 else 0 for b in range(1500)]
    g = torch.Generator().manual_seed(12)
    cache = U.Cache(g, bits, 64, 1, 32, lens)
    q_lat, q_rope = U.normal(g, 1500, 2, 64), U.normal(g, 1500, 2, 64)
    got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32(lens), SCALE)
    check_decode(cache, q_lat, q_rope, lens, SCALE, got)


def test_an_empty_cache_and_then_one_of_the_same_sizes():
    q = torch.ones(2, 16, 512, dtype=torch.bfloat16, device="cuda")
    for n in (0, 200):
        pages, scales = T.new_paged_cache(n, 64, 512, bits=4)
        table = torch.arange(200, dtype=torch.int32, device="cuda").view(2, 100)
        ctx, lse = T.paged_decode(q, q[..., :64], pages, scales, table, i32([6400, 100]), SCALE)
        assert not ctx.any()
        if n:  # rows of zeros: every token weighs the same
            want = torch.tensor([6400.0, 100.0]).log()[:, None].expand(2, 16)
            torch.testing.assert_close(lse.cpu(), want, rtol=0, atol=2.0 ** -18)
        else:
            assert (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_longest_rows(dtype):
    """2^19 logits, a row that begins off its alignment."""
    V = 1 << 19
    g = torch.Generator().manual_seed(13)
    x = (torch.randn(2, V, generator=g) * 2).to(dtype)
    wide = torch.zeros(2, V + 5, dtype=dtype)
    wide[:, 3:V + 3] = x
    u = torch.tensor([0.3, 0.999])
    for settings in (dict(temperature=0.9), dict(top_k=3000, top_p=0.8), dict(temperature=1.5, top_p=0.99, min_p=0.001)):
        token, logprob = T.sample_tokens(wide.cuda()[:, 3:V + 3], u.cuda(), **settings)
        s = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **settings}
        for b in range(2):
            want, lp, room = sample_util.draw(x[b].float().numpy(), np.float32(u[b].item()), np.float32(s["temperature"]), s["top_k"],
                                              np.float32(s["top_p"]), np.float32(s["min_p"]))
            if room > 1:
                assert int(token[b]) == want and abs(float(logprob[b]) - lp) <= 2.0 ** -22 * max(1.0, abs(lp))


@pytest.mark.parametrize("layout", ["baseline", "model"])
def test_a_single_tokens_score_in_four_bits(layout):
    """lse of one token is its score.  A run's sum of u q, u = 16 + code (24.4 root mean square) and queries of size 1, is sqrt(k) 24.4 after
    k products; rounded after each of the 64, by 2^-24 / sqrt(12) of it, it is 2^-24 / sqrt(12) 24.4 sqrt(2080) = 1.9e-5 off.  The run's
    share of the score is sqrt(64) 2.8 = 22 (code - 8 is 2.8: a scale is 0.36 of the values), so it is 8.6e-7 of that, as is the sum of
    all runs.  With 24 sum q, of the same size and rounded to 24 bits, and a spread of a sixth over 16 heads, 1.5e-6 bounds it; with 128 in
    place of 16 throughout it would be 4e-6."""
    H, Hr, DL = LAYOUTS[layout]
    g = torch.Generator().manual_seed(21)
    cache = U.Cache(g, 4, DL, Hr, 16, [1] * 24)
    q_lat, q_rope = U.normal(g, 24, H, DL), U.normal(g, 24, H, 64)
    _, lse = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32([1] * 24), SCALE)
    _, want, _, _ = U.decode(cache, q_lat, q_rope, [1] * 24, SCALE)
    off = (lse.double().cpu() - want).norm() / want.norm()
    assert float(off) <= 1.5e-6, float(off)
