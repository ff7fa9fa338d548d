"""The paged latent cache's operators on the GPU against plain ones in 64 bits: appending and reading bit for bit, attention
within the bounds that its roundings have (tests/paged_util.py)."""
import copy
import math

import pytest
import torch

import transformer_amd as T
from tests import paged_util as U

pytestmark = pytest.mark.gpu
LAYOUTS = {"model": (14, 14, 384), "baseline": (16, 1, 512), "tiny": (3, 3, 64), "one": (1, 1, 128), "wide": (33, 1, 256),
           "many": (20, 20, 128)}


def same_bits(a, b):
    """Equal, NaN where the other is."""
    a, b = a.cpu(), b.cpu()
    if a.dtype.is_floating_point:
        return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())
    return torch.equal(a, b)


def check_cache(dev, cache):
    pages, scales = dev
    assert same_bits(pages, cache.pages)
    assert scales is None or same_bits(scales, cache.scales)


def i32(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


APPENDS = [
    # layout, size, starts, counts, T
    ("model", 16, [0], None, 1),
    ("baseline", 64, [5, 0, 63, 64], None, 1),
    ("baseline", 16, [0, 15, 33, 7, 2], [37, 0, 1, 19, 16], 37),
    ("tiny", 48, [47, 1], [50, 7], 50),
    ("one", 32, [31], [2], 5),
    ("wide", 16, [3, 9], None, 21),
    ("many", 256, [250, 0, 17], [9, 12, 0], 12),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout,size,starts,counts,T_", APPENDS)
def test_append_and_read(bits, layout, size, starts, counts, T_):
    H, Hr, DL = LAYOUTS[layout]
    B = len(starts)
    g = torch.Generator().manual_seed(T_ + size)
    cache = U.Cache(g, bits, DL, Hr, size, [s + T_ for s in starts])
    # as columns of one product: rows of another stride, 16-byte aligned
    down = U.normal(g, B, T_, 8 + (H + Hr) * 64 + DL)
    qk, c_new = down[..., 8:8 + (H + Hr) * 64].unflatten(-1, (H + Hr, 64)), down[..., -DL:]
    cos, sin = U.tables(400)
    dev, down_d = cache.dev(), down.cuda()
    q = T.paged_append(down_d[..., 8:8 + (H + Hr) * 64].unflatten(-1, (H + Hr, 64)), down_d[..., -DL:], *dev, cos.cuda(), sin.cuda(),
                       cache.table.cuda(), i32(starts), None if counts is None else i32(counts))
    want = U.append(cache, qk, c_new, cos, sin, starts, counts)
    assert same_bits(q, want)
    check_cache(dev, cache)
    for at, n in ((starts, counts), (None, None), ([s - 3 for s in starts], [T_ + 5] * B)):
        latent, k_rope = T.paged_read(*dev, cache.table.cuda(), DL, T_ + 2, starts=None if at is None else i32(at),
                                      counts=None if n is None else i32(n))
        want_l, want_k = U.read(cache, T_ + 2, at, n, B)
        assert same_bits(latent, want_l) and same_bits(k_rope, want_k)


@pytest.mark.parametrize("bits", [16, 4])
def test_append_skips_what_has_no_place(bits):
    """Positions below 0 or past the tables, pages outside the cache, counts beyond T and below 0: nothing else is touched."""
    H, Hr, DL = LAYOUTS["baseline"]
    g = torch.Generator().manual_seed(3)
    cache = U.Cache(g, bits, DL, Hr, 16, [64] * 6)
    cache.table[1, 1], cache.table[2, 0], cache.table[3, 2] = -1, cache.n, -(1 << 31)
    starts, counts = [-3, 10, 0, 30, 60, 0], [9, 9, 20, 9, 40, -5]
    qk, c_new = U.normal(g, 6, 20, H + Hr, 64), U.normal(g, 6, 20, DL)
    for rows in (400, 50):  # tables that end before the pages do
        cos, sin = U.tables(rows)
        dev = cache.dev()
        q = T.paged_append(qk.cuda(), c_new.cuda(), *dev, cos.cuda(), sin.cuda(), cache.table.cuda(), i32(starts), i32(counts))
        kept = copy.deepcopy(cache)
        assert same_bits(q, U.append(kept, qk, c_new, cos, sin, starts, counts))
        check_cache(dev, kept)
        latent, k_rope = T.paged_read(*dev, cache.table.cuda(), DL, 70, starts=i32(starts), counts=i32([70] * 6))
        want = U.read(kept, 70, starts, [70] * 6, 6)
        assert same_bits(latent, want[0]) and same_bits(k_rope, want[1])


def test_four_bit_values_at_the_edges():
    """Runs of zeros, of one value, of the least and greatest magnitudes, halves that round to even, a NaN, infinities."""
    g = torch.Generator().manual_seed(1)
    DL = 512
    c_new = U.normal(g, 1, 8, DL)
    c_new[0, 0] = 0
    c_new[0, 1] = 3.0
    c_new[0, 2, :64] = 2.0 ** -133  # a subnormal
    c_new[0, 2, 64:128] = 3e38
    c_new[0, 3, :64] = torch.arange(64).float() / 4 - 8  # scale 8 / 7 in bf16
    c_new[0, 3, 64:128] = (torch.arange(64) % 15).float() * 0.5 - 3.5  # scale 0.5: whole and half codes
    c_new[0, 3, 128:192] = (torch.arange(64) % 29).float() * 0.25 - 3.5  # scale 0.5: quarters and halves
    c_new[0, 4, 70], c_new[0, 5, 3], c_new[0, 6, 511] = math.nan, math.inf, -math.inf
    c_new[0, 7, 5::7] *= 100
    cache = U.Cache(g, 4, DL, 1, 16, [16])
    qk = U.normal(g, 1, 8, 2, 64)
    qk[0, 4, 1, 7] = math.nan
    cos, sin = U.tables(32)
    dev = cache.dev()
    T.paged_append(qk.cuda(), c_new.cuda(), *dev, cos.cuda(), sin.cuda(), cache.table.cuda(), i32([2]))
    U.append(cache, qk, c_new, cos, sin, [2], None)
    check_cache(dev, cache)
    latent, k_rope = T.paged_read(*dev, cache.table.cuda(), DL, 12)
    want = U.read(cache, 12, None, None, 1)
    assert same_bits(latent, want[0]) and same_bits(k_rope, want[1])
    got = latent.cpu()
    assert got[0, 6, 64:128].isnan().all() and got[0, 7, :64].isnan().all() and not got[0, 6, :64].isnan().any()
    assert (got[0, 2] == 0).all()


DECODES = [
    # layout, size, lengths
    ("model", 16, [701]),
    ("baseline", 64, [1]),
    ("baseline", 16, [0, 1, 15, 16, 17, 31, 32, 33]),
    ("baseline", 128, [63, 64, 65, 127, 128, 129, 1000]),
    ("baseline", 48, [0, 0, 0]),
    ("model", 32, [5, 0, 64, 333, 47]),
    ("tiny", 16, [100, 7]),
    ("one", 4096, [4097, 20]),
    ("wide", 80, [161, 3, 250]),
    ("many", 16, [70, 0, 130]),
    ("baseline", 16, [17 * b % 211 for b in range(70)]),
    ("baseline", 64, [9000, 3, 2500]),
    ("model", 64, [40, 3000]),
]


def decode_inputs(bits, layout, size, lens, seed=0, room=None, std=1.0):
    H, Hr, DL = LAYOUTS[layout]
    g = torch.Generator().manual_seed(seed + sum(lens) + size)
    cache = U.Cache(g, bits, DL, Hr, size, room or lens, std=std)
    return cache, U.normal(g, len(lens), H, DL), U.normal(g, len(lens), H, 64)


def check_decode(cache, q_lat, q_rope, lens, scale, got, limit=None):
    ctx, lse, ctx_tol, lse_tol = U.decode(cache, q_lat, q_rope, lens if limit is None else limit, scale)
    c, l = got[0].double().cpu(), got[1].double().cpu()
    empty = lse == -math.inf
    assert (c[empty] == 0).all() and (l[empty] == -math.inf).all()
    e = (c - ctx).abs()
    # all roundings are independent: two of 2^-8 / sqrt(3) each (root mean square) make 0.82 x 2^-8 of the result's norm
    norm = float(ctx.norm())
    assert ctx.numel() < 2000 or float(e.norm()) <= 2.0 ** -8 * norm + 2 * float(ctx_tol.mean()) * 2.0 ** -8, float(e.norm()) / max(norm, 1e-30)
    assert bool((e <= ctx_tol).all()), ("ctx", float((e - ctx_tol).max()), float((e / ctx_tol.clamp(min=1e-30)).max()))
    e = (l - lse)[~empty].abs()
    assert bool((e <= lse_tol[~empty]).all()), ("lse", float(e.max()), float((e / lse_tol[~empty]).max()))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout,size,lens", DECODES)
def test_decode(bits, layout, size, lens):
    cache, q_lat, q_rope = decode_inputs(bits, layout, size, lens)
    scale = 192 ** -0.5
    got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32(lens), scale)
    check_decode(cache, q_lat, q_rope, lens, scale, got)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout", ["model", "baseline", "tiny"])
def test_decode_leaves_out_what_is_no_token(bits, layout):
    """Entries that are no page, lengths past the table and below 0, and NaN behind every sequence's end and in other pages."""
    lens = [200, 64, 37, 0, 500, -7]
    cache, q_lat, q_rope = decode_inputs(bits, layout, 16, [200, 64, 37, 0, 500, 0], seed=5)
    cache.table[0, 3], cache.table[0, 7], cache.table[1, :] = -1, cache.n + 5, -1
    clean = copy.deepcopy(cache)
    used = torch.zeros(cache.n, cache.size, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(max(0, n)):
            at = cache.place(b, p)
            if at is not None:
                used[at] = True
    if bits == 16:
        cache.pages[~used] = math.nan
    else:
        cache.pages[~used] = 0xF1
        cache.scales.transpose(1, 2)[~used] = math.nan
    asked = list(lens)
    asked[4] = 1 << 30  # past the table: all that it has
    limit = list(lens)
    limit[4] = cache.table.size(1) * cache.size
    lo = 500 // 16 * 16
    for p in range(lo, limit[4]):  # the last page's tokens behind the end are tokens now
        at = cache.place(4, p)
        if bits == 16:
            cache.pages[at] = clean.pages[at]
        else:
            cache.pages[at] = clean.pages[at]
            cache.scales[at[0], :, at[1]] = clean.scales[at[0], :, at[1]]
    got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32(asked), 0.07)
    check_decode(clean, q_lat, q_rope, asked, 0.07, got, limit)


def test_decode_agrees_with_the_contiguous_one():
    lens = [1, 130, 700, 64]
    cache, q_lat, q_rope = decode_inputs(16, "baseline", 64, lens)
    pages, _ = cache.dev()
    table = cache.table.cuda()
    latent, k_rope = T.paged_read(pages, None, table, 512, 700)
    want, want_lse = torch.ops.mla_mi355x.decode(q_lat.cuda(), q_rope.cuda(), latent, k_rope, i32(lens), 0.07, 0)
    got, lse = T.paged_decode(q_lat.cuda(), q_rope.cuda(), pages, None, table, i32(lens), 0.07)
    # both within bf16 roundings of p, of a partial and of the result
    assert float((got.float() - want.float()).abs().max()) <= 4 * 2.0 ** -8 * float(want.float().abs().max())
    torch.testing.assert_close(lse, want_lse, rtol=0, atol=1e-4)


@pytest.mark.parametrize("bits", [16, 4])
def test_peaked_and_large_scores(bits):
    """One token carries nearly all the weight; scores in the thousands."""
    cache, q_lat, q_rope = decode_inputs(bits, "baseline", 32, [700, 90], std=8.0)
    got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32([700, 90]), 1.0)
    check_decode(cache, q_lat, q_rope, [700, 90], 1.0, got)


@pytest.mark.parametrize("bits", [16, 4])
def test_strides_shared_pages_and_layers(bits):
    """Queries as columns of wider rows, a cache that is one layer of many, two sequences with the same first pages, a block table
    with more columns than are used."""
    H, Hr, DL = LAYOUTS["baseline"]
    lens = [150, 180, 16]
    cache, q_lat, q_rope = decode_inputs(bits, "baseline", 16, lens, seed=9)
    cache.table[1, :6] = cache.table[0, :6]
    q = torch.zeros(3, H, DL + 64 + 8, dtype=torch.bfloat16)
    q[..., :DL], q[..., DL:DL + 64] = q_lat, q_rope
    q = q.cuda()
    layers = torch.stack([torch.zeros_like(cache.pages), cache.pages, torch.zeros_like(cache.pages)], 1).cuda()
    scales = None if bits == 16 else torch.stack([torch.zeros_like(cache.scales), cache.scales], 1).cuda()[:, 1]
    wide = torch.full((3, 40), -1, dtype=torch.int32)
    wide[:, :cache.table.size(1)] = cache.table
    got = T.paged_decode(q[..., :DL], q[..., DL:DL + 64], layers[:, 1], scales, wide.cuda()[:, :33], i32(lens), 0.1)
    check_decode(cache, q_lat, q_rope, lens, 0.1, got)
    latent, k_rope = T.paged_read(layers[:, 1], scales, wide.cuda()[:, :33], DL, 150)
    want = U.read(cache, 150, None, None, 3)
    assert same_bits(latent, want[0]) and same_bits(k_rope, want[1])
    cos, sin = U.tables(256)
    qk, c_new = U.normal(torch.Generator().manual_seed(2), 3, 2, H + 1, 64), U.normal(torch.Generator().manual_seed(4), 3, 2, DL)
    T.paged_append(qk.cuda(), c_new.cuda(), layers[:, 1], scales, cos.cuda(), sin.cuda(), wide.cuda()[:, :33], i32(lens))
    U.append(cache, qk, c_new, cos, sin, lens, None)
    check_cache((layers[:, 1].contiguous(), scales), cache)
    assert not layers[:, 0].any() and not layers[:, 2].any()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_cache_past_4_gib(bits):
    """Pages whose byte offsets pass 32 bits."""
    H, Hr, DL = LAYOUTS["model"]
    small, q_lat, q_rope = decode_inputs(bits, "model", 64, [130, 70], seed=2)
    per = small.pages[0].numel() * small.pages.element_size()
    n = (9 << 29) // per + 4
    pages = torch.empty(n, *small.pages.shape[1:], dtype=small.pages.dtype, device="cuda")
    scales = None if bits == 16 else torch.empty(n, *small.scales.shape[1:], dtype=torch.bfloat16, device="cuda")
    shift = n - small.n
    pages[shift:] = small.pages.cuda()
    if bits == 4:
        scales[shift:] = small.scales.cuda()
    table = torch.where(small.table >= 0, small.table + shift, -1).to(torch.int32).cuda()
    cos, sin = U.tables(256)
    qk, c_new = U.normal(torch.Generator().manual_seed(1), 2, 3, H + Hr, 64), U.normal(torch.Generator().manual_seed(2), 2, 3, DL)
    T.paged_append(qk.cuda(), c_new.cuda(), pages, scales, cos.cuda(), sin.cuda(), table, i32([100, 60]))
    U.append(small, qk, c_new, cos, sin, [100, 60], None)
    assert same_bits(pages[shift:], small.pages)
    got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), pages, scales, table, i32([130, 70]), 0.07)
    check_decode(small, q_lat, q_rope, [130, 70], 0.07, got)
    latent, _ = T.paged_read(pages, scales, table, DL, 130)
    assert same_bits(latent, U.read(small, 130, None, None, 2)[0])


@pytest.mark.parametrize("bits", [16, 4])
def test_results_repeat_and_other_streams(bits):
    lens = [3000, 17, 900, 0, 2200]
    cache, q_lat, q_rope = decode_inputs(bits, "baseline", 64, lens)
    args = (q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32(lens), 0.07)
    first = T.paged_decode(*args)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = [T.paged_decode(*args) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(other)
    for c, l in again:
        assert torch.equal(c, first[0]) and torch.equal(l, first[1])


@pytest.mark.parametrize("bits", [16, 4])
def test_a_recorded_step_follows_the_lengths(bits):
    """Append, attention and what it reads from device buffers in a graph: replayed while the sequences grow, beside eager calls."""
    H, Hr, DL = LAYOUTS["baseline"]
    lens = [10, 63, 0, 300]
    cache, _, _ = decode_inputs(bits, "baseline", 16, lens, room=[400] * 4)
    cos, sin = U.tables(512)
    cos_d, sin_d, table = cos.cuda(), sin.cuda(), cache.table.cuda()
    dev = cache.dev()
    qk, c_new, q_lat = (torch.empty(4, 1, H + 1, 64, dtype=torch.bfloat16, device="cuda"),
                        torch.empty(4, 1, DL, dtype=torch.bfloat16, device="cuda"),
                        torch.empty(4, H, DL, dtype=torch.bfloat16, device="cuda"))
    for t in (qk, c_new, q_lat):
        t.zero_()
    start, after = i32(lens), i32([n + 1 for n in lens])
    scratch = [t if t is None else t.clone() for t in dev]

    def step(pages, scales):
        q = T.paged_append(qk, c_new, pages, scales, cos_d, sin_d, table, start)
        return T.paged_decode(q_lat, q[:, 0], pages, scales, table, after, 0.07)

    step(*scratch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*dev)
    g = torch.Generator().manual_seed(8)
    for i in range(4):
        new = U.normal(g, 4, 1, H + 1, 64), U.normal(g, 4, 1, DL), U.normal(g, 4, H, DL)
        for to, x in zip((qk, c_new, q_lat), new):
            to.copy_(x)
        start.copy_(i32(lens))
        after.copy_(i32([n + 1 for n in lens]))
        graph.replay()
        torch.cuda.synchronize()
        recorded = [t.clone() for t in out]
        eager = step(*dev)  # the same token to the same place again
        assert torch.equal(recorded[0], eager[0]) and torch.equal(recorded[1], eager[1])
        q = U.append(cache, new[0], new[1], cos, sin, lens, None)
        lens = [n + 1 for n in lens]
        check_decode(cache, new[2], q[:, 0], lens, 0.07, recorded)
        check_cache(dev, cache)


def test_operators_under_fake_tensors_and_opcheck():
    cache, q_lat, q_rope = decode_inputs(4, "baseline", 16, [20, 3])
    dev, table, lens = cache.dev(), cache.table.cuda(), i32([20, 3])
    cos, sin = (t.cuda() for t in U.tables(64))
    g = torch.Generator().manual_seed(0)
    ops = torch.ops.mla_mi355x
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.paged_decode, (q_lat.cuda(), q_rope.cuda(), *dev, table, lens, 0.1), test_utils=tests)
    torch.library.opcheck(ops.paged_read, (*dev, table, 512, 9, None, None), test_utils=tests)
    torch.library.opcheck(ops.paged_append, (U.normal(g, 2, 1, 17, 64).cuda(), U.normal(g, 2, 1, 512).cuda(), *dev, cos, sin, table,
                                             lens, None), test_utils=tests)


def test_nothing_to_do():
    pages, scales = T.new_paged_cache(4, 16, 512, bits=4)
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 16, 512, dtype=torch.bfloat16, device="cuda")
    ctx, lse = T.paged_decode(q, q[..., :64], pages, scales, none, i32([]), 0.1)
    assert ctx.shape == (0, 16, 512) and lse.shape == (0, 16)
    latent, k_rope = T.paged_read(pages, scales, i32([[1], [2]]), 512, 0)
    assert latent.shape == (2, 0, 512) and k_rope.shape == (2, 1, 0, 64)
    latent, k_rope = T.paged_read(pages, scales, i32([[1], [2]]), 512, 20)
    assert not latent.any() and not k_rope.any()
    # a table without columns: nobody has tokens
    q = torch.ones(2, 16, 512, dtype=torch.bfloat16, device="cuda")
    ctx, lse = T.paged_decode(q, q[..., :64], pages, scales, torch.empty(2, 0, dtype=torch.int32, device="cuda"), i32([5, 0]), 0.1)
    assert not ctx.any() and (lse == -math.inf).all()
