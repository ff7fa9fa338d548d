"""The serving operators under torch's program transforms and from several threads."""
import threading

import pytest
import torch

import transformer_amd as T
from tests import paged_util as U
from tests.test_gpu_paged import LAYOUTS, i32

pytestmark = pytest.mark.gpu


def world(bits, lens=(20, 3, 47), layout="baseline", seed=5):
    H, Hr, DL = LAYOUTS[layout]
    g = torch.Generator().manual_seed(seed)
    cache = U.Cache(g, bits, DL, Hr, 16, [n + 8 for n in lens])
    B = len(lens)
    qk, c_new, q_lat = (t.cuda() for t in (U.normal(g, B, 1, H + Hr, 64), U.normal(g, B, 1, DL), U.normal(g, B, H, DL)))
    w = U.normal(g, 500, DL).cuda()
    cos, sin = (t.cuda() for t in U.tables(128))
    table, at, u = cache.table.cuda(), i32(list(lens)), torch.rand(B, generator=g).cuda()

    def step(pages, scales, qk, c_new, q_lat, at, u):
        q = T.paged_append(qk, c_new, pages, scales, cos, sin, table, at)
        ctx, lse = T.paged_decode(q_lat, q[:, 0], pages, scales, table, at + 1, 0.07)
        latent, k_rope = T.paged_read(pages, scales, table, DL, 5, starts=at - 2)
        tokens, logprobs = T.sample_tokens((ctx[:, 0] @ w.T).float(), u, temperature=0.7, top_k=30, top_p=0.9)
        return q, ctx, lse, latent, k_rope, tokens, logprobs

    return step, cache, (qk, c_new, q_lat, at, u)


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [16, 4])
def test_compiled(bits):
    """aot_eager: functionalized, so the pages' writes are seen only if the operator says what it writes."""
    step, cache, rest = world(bits)
    dev, again = cache.dev(), cache.dev()
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    for i in range(3):
        rest = (*rest[:3], rest[3] + (1 if i else 0), rest[4])
        assert same(compiled(*dev, *rest), step(*again, *rest))
        assert torch.equal(dev[0], again[0]) and (bits == 16 or torch.equal(dev[1], again[1]))


@pytest.mark.parametrize("bits", [16, 4])
def test_traced(bits):
    step, cache, rest = world(bits)
    if bits == 16:
        traced_of = lambda pages, *a: step(pages, None, *a)
        args = lambda dev: (dev[0], *rest)
    else:
        traced_of, args = step, lambda dev: (*dev, *rest)
    traced = torch.jit.trace(traced_of, args(cache.dev()), check_trace=False)
    dev, again = cache.dev(), cache.dev()
    assert same(traced(*args(dev)), step(*again, *rest)) and torch.equal(dev[0], again[0])


@pytest.mark.parametrize("bits", [16, 4])
def test_in_inference_mode(bits):
    step, cache, rest = world(bits)
    want = step(*cache.dev(), *rest)
    with torch.inference_mode():
        pages, scales = (t if t is None else t.clone() for t in cache.dev())
        assert same(step(pages, scales, *rest), want)
    assert same(step(pages, scales, *rest), want)  # and what was made there, outside it


@pytest.mark.parametrize("bits", [16, 4])
def test_many_threads(bits):
    """Each on a stream and a cache of its own, their calls in no order."""
    worlds = [world(bits, seed=s) for s in range(4)]
    want = [step(*cache.dev(), *rest) for step, cache, rest in worlds]
    torch.cuda.synchronize()
    wrong = []

    def loop(k):
        step, cache, rest = worlds[k]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            dev = cache.dev()
            for _ in range(40):
                got = step(*dev, *rest)
            stream.synchronize()
            if not same(got, want[k]):
                wrong.append(k)

    threads = [threading.Thread(target=loop, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_inputs_are_left_alone():
    """What a call only reads keeps its bits, the cache's rows beside the new ones among it."""
    step, cache, rest = world(4)
    dev = cache.dev()
    before = [t.clone() for t in (*dev, *rest)]
    step(*dev, *rest)
    for t, was in zip(rest, before[2:]):
        assert torch.equal(t, was)
    new = torch.zeros(cache.n, cache.size, dtype=torch.bool)
    for b, n in enumerate(rest[3].tolist()):
        new[cache.place(b, n)] = True
    assert torch.equal(dev[0].cpu()[~new], before[0].cpu()[~new])
    assert torch.equal(dev[1].cpu().transpose(1, 2)[~new], before[1].cpu().transpose(1, 2)[~new])


@pytest.mark.parametrize("bits", [16, 4])
def test_the_serving_tests_compare_their_tokens(bits, monkeypatch):
    """Those tests leave out a row whose border is within roundings: they have next to none."""
    from tests import sample_util
    from tests import test_gpu_serving as S

    rooms, draw = [], sample_util.draw

    def recorded(*args):
        out = draw(*args)
        rooms.append(out[2])
        return out

    monkeypatch.setattr(sample_util, "draw", recorded)
    S.test_prompts_in_parts_and_then_token_by_token(bits, "baseline")
    S.test_two_recorded_loops_of_steps(bits)
    assert len(rooms) >= 50 and sum(r > 1 for r in rooms) >= 0.98 * len(rooms), sorted(rooms)[:5]
    rooms.clear()
    S.test_the_longest_rows(torch.bfloat16 if bits == 16 else torch.float32)
    assert len(rooms) == 6 and min(rooms) > 4
