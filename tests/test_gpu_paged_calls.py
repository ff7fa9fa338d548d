"""Calls of the paged operators that a program makes and no other test does: layouts of one sequence, token or head."""
import pytest
import torch

import transformer_amd as T
from tests import paged_util as U
from tests.test_gpu_paged import LAYOUTS, check_cache, check_decode, i32, same_bits

pytestmark = pytest.mark.gpu


def odd(t, dims):
    """``t`` with strides 1, 3, 5 .. in its dimensions ``dims`` of size 1."""
    st = list(t.stride())
    for k, d in enumerate(dims):
        assert t.size(d) == 1
        st[d] = 2 * k + 1
    return t.as_strided(t.shape, st)


@pytest.mark.parametrize("bits", [16, 4])
def test_one_sequences_queries_as_a_product_leaves_them(bits):
    H, Hr, DL = LAYOUTS["baseline"]
    g = torch.Generator().manual_seed(3)
    cache = U.Cache(g, bits, DL, Hr, 16, [70])
    w, x = U.normal(g, H, DL, 64).cuda(), U.normal(g, H, 64, 1, std=0.1).cuda()
    q_lat = torch.matmul(w, x).permute(2, 0, 1)  # [1, H, DL], strides (1, DL, 1)
    assert q_lat.stride(0) % 8
    q_rope = U.normal(g, 1, H, 64)
    got = T.paged_decode(q_lat, odd(q_rope.cuda(), (0,)), *cache.dev(), cache.table.cuda(), i32([70]), 0.07)
    check_decode(cache, q_lat.cpu(), q_rope, [70], 0.07, got)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout,B,T_,dims", [("one", 4, 1, (1,)), ("one", 1, 3, (0,)), ("one", 1, 1, (0, 1)), ("model", 1, 1, (1, 0))])
def test_appended_rows_of_one_token_or_sequence(bits, layout, B, T_, dims):
    H, Hr, DL = LAYOUTS[layout]
    g = torch.Generator().manual_seed(4 + B)
    cache = U.Cache(g, bits, DL, Hr, 16, [40] * B)
    qk, c_new, starts = U.normal(g, B, T_, H + Hr, 64), U.normal(g, B, T_, DL), [5 * b for b in range(B)]
    cos, sin = U.tables(64)
    dev = cache.dev()
    q = T.paged_append(odd(qk.cuda(), dims), odd(c_new.cuda(), dims), *dev, cos.cuda(), sin.cuda(), cache.table.cuda(), i32(starts))
    assert same_bits(q, U.append(cache, qk, c_new, cos, sin, starts, None))
    check_cache(dev, cache)


@pytest.mark.parametrize("bits", [16, 4])
def test_one_head(bits):
    g = torch.Generator().manual_seed(6)
    cache = U.Cache(g, bits, 128, 1, 16, [33, 5])
    q_lat, q_rope = U.normal(g, 2, 1, 128), U.normal(g, 2, 1, 64)
    got = T.paged_decode(odd(q_lat.cuda(), (1,)), odd(q_rope.cuda(), (1,)), *cache.dev(), cache.table.cuda(), i32([33, 5]), 0.1)
    check_decode(cache, q_lat, q_rope, [33, 5], 0.1, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T_,heads,dims", [(1, 5, 3, (0,)), (4, 1, 3, (1,)), (2, 5, 1, (2,)), (1, 1, 1, (0, 1, 2))])
def test_rotation_of_one_sequence_token_or_head(dtype, B, T_, heads, dims):
    """The rotation that the append does, as an operator of its own."""
    g = torch.Generator().manual_seed(8)
    x = U.normal(g, B, T_, heads, 64).to(dtype).cuda()
    cos, sin = (t.cuda() for t in U.tables(16))
    ops = torch.ops.mla_mi355x
    want = ops.rope(x, cos, sin, 2, False)
    y = odd(x.clone(), dims)
    assert torch.equal(ops.rope(y, cos, sin, 2, False), want)
    ops.rope_(y, cos, sin, 2, False)
    assert torch.equal(y, want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H,Hr", [(16, 1), (33, 1), (5, 5)])
def test_as_many_sequences_as_the_entry_takes(bits, H, Hr):
    """2^20 - 1 sequences of up to a page, most of them empty: more workgroups of heads than 2^32 threads hold in one dimension (H = 16 and
    33), and the time of one look at all lengths, not of one a head."""
    B, n = (1 << 20) - 1, 251
    lens = [(b * 7) % 17 if b % 3 else 0 for b in range(n)]
    g = torch.Generator().manual_seed(31)
    cache = U.Cache(g, bits, 64, Hr, 16, lens)
    q_lat, q_rope, dev, table = U.normal(g, n, H, 64), U.normal(g, n, H, 64), cache.dev(), cache.table.cuda()
    some = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *dev, table, i32(lens), 0.2)
    check_decode(cache, q_lat, q_rope, lens, 0.2, some)
    at = torch.arange(B, device="cuda") % n
    ql, qr = q_lat.cuda()[at], q_rope.cuda()[at]
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    ctx, lse = T.paged_decode(ql, qr, *dev, table[at], i32(lens)[at], 0.2)
    end.record()
    torch.cuda.synchronize()
    assert torch.equal(ctx, some[0][at]) and torch.equal(lse, some[1][at])  # (one tile each: in one run whatever the batch)
    assert start.elapsed_time(end) < 2000, start.elapsed_time(end)


@pytest.mark.parametrize("bits", [16, 4])
def test_sequences_cut_into_many_runs_beside_short_and_empty_ones(bits):
    """Parts of one sequence in two runs and in many, heads in several groups."""
    g = torch.Generator().manual_seed(32)
    lens = [0, 6000, 1, 0, 64, 700, 0, 2500, 16, 0]
    cache = U.Cache(g, bits, 64, 1, 64, lens)
    for H in (3, 16, 40):
        q_lat, q_rope = U.normal(g, len(lens), H, 64), U.normal(g, len(lens), H, 64)
        got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32(lens), 0.1)
        check_decode(cache, q_lat, q_rope, lens, 0.1, got)
