"""The paged operators over random layouts, and with infinities and NaN in rows and queries: what they do to their own sequence or head, and
that they do nothing to others."""
import math
import random

import pytest
import torch

import transformer_amd as T
from tests import paged_util as U
from tests.test_gpu_paged import LAYOUTS, check_cache, check_decode, i32, same_bits

pytestmark = pytest.mark.gpu


def random_layout(rng):
    H = rng.choice([1, 2, 5, 8, 14, 16, 17, 31, 40])
    return H, rng.choice([1, H]), rng.choice([64, 128, 256, 384, 512])


def spread(rng, hi):
    return max(0, min(hi, int(round(math.exp(rng.uniform(0, math.log(hi + 1)))) - 1)))


@pytest.mark.parametrize("seed", range(24))
def test_random_decodes(seed):
    rng, g = random.Random(900 + seed), torch.Generator().manual_seed(seed)
    H, Hr, DL = random_layout(rng)
    bits, size, B = rng.choice([16, 4]), 16 * rng.choice([1, 1, 2, 3, 5, 8, 64, 256]), rng.choice([1, 2, 3, 7, 20, 67])
    lens = [spread(rng, 6000 // B + 40) for _ in range(B)]
    cache = U.Cache(g, bits, DL, Hr, size, lens)
    for _ in range(rng.choice([0, 0, 2])):  # pages that are none
        if cache.table.numel():
            cache.table[rng.randrange(B), rng.randrange(cache.table.size(1))] = rng.choice([-1, cache.n, 1 << 30, -(1 << 31)])
    q_lat, q_rope = U.normal(g, B, H, DL), U.normal(g, B, H, 64)
    if rng.random() < 0.5:  # a slice of wider rows
        q = torch.cat([q_rope, q_lat, q_rope], -1).cuda()
        ql, qr = q[..., 64:64 + DL], q[..., :64]
    else:  # heads first
        ql, qr = (t.transpose(0, 1).contiguous().cuda().transpose(0, 1) for t in (q_lat, q_rope))
    scale = rng.choice([0.02, 192 ** -0.5, 0.3])
    got = T.paged_decode(ql, qr, *cache.dev(), cache.table.cuda(), i32(lens), scale)
    check_decode(cache, q_lat, q_rope, lens, scale, got)


@pytest.mark.parametrize("seed", range(24))
def test_random_appends_and_reads(seed):
    rng, g = random.Random(700 + seed), torch.Generator().manual_seed(seed)
    H, Hr, DL = random_layout(rng)
    if rng.random() < 0.2:
        H = Hr  # (as many query heads as keys)
    bits, size, B, T_ = rng.choice([16, 4]), 16 * rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 5, 9]), rng.choice([1, 2, 7, 33, 100])
    starts = [rng.randint(-3, 90) for _ in range(B)]
    counts = None if rng.random() < 0.4 else [rng.randint(-2, T_ + 3) for _ in range(B)]
    cache = U.Cache(g, bits, DL, Hr, size, [rng.randint(1, 200) for _ in range(B)])
    qk, c_new = U.normal(g, B, T_, H + Hr, 64, std=rng.choice([1e-3, 1.0, 300.0])), U.normal(g, B, T_, DL)
    cos, sin = U.tables(rng.choice([64, 120, 256]))
    dev = cache.dev()
    q = T.paged_append(qk.transpose(0, 1).contiguous().cuda().transpose(0, 1), c_new.cuda(), *dev, cos.cuda(), sin.cuda(), cache.table.cuda(),
                       i32(starts), None if counts is None else i32(counts))
    assert same_bits(q, U.append(cache, qk, c_new, cos, sin, starts, counts))
    check_cache(dev, cache)
    n = rng.choice([1, 50, 230])
    latent, k_rope = T.paged_read(*dev, cache.table.cuda(), DL, n, i32(starts), None if counts is None else i32(counts))
    want = U.read(cache, n, starts, counts, B)
    assert same_bits(latent, want[0]) and same_bits(k_rope, want[1])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout", ["baseline", "model", "one", "many"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_row_reaches_its_own_sequence_alone(bits, layout, bad):
    """Sequences that share workgroups, and ring slots, with one whose rows are all NaN or infinite; the others' ends lie inside tiles."""
    H, Hr, DL = LAYOUTS[layout]
    g = torch.Generator().manual_seed(50)
    lens = [(37 * b) % 150 + 1 for b in range(600)]
    cache = U.Cache(g, bits, DL, Hr, 16, lens)
    rotten = [b for b in range(600) if b % 5 == 2]
    q_lat, q_rope = U.normal(g, 600, H, DL), U.normal(g, 600, H, 64)
    table, args = cache.table.cuda(), (q_lat.cuda(), q_rope.cuda())
    clean = T.paged_decode(*args, *cache.dev(), table, i32(lens), 0.07)
    pages, scales = cache.dev()
    at = cache.table[rotten].flatten()
    at = at[at >= 0].long().cuda()
    if bits == 16:
        pages[at] = bad
    else:
        scales[at] = bad
    ctx, lse = T.paged_decode(*args, pages, scales, table, i32(lens), 0.07)
    ok = torch.ones(600, dtype=torch.bool)
    ok[rotten] = False
    ok = ok.cuda()
    assert torch.equal(ctx[ok], clean[0][ok]) and torch.equal(lse[ok], clean[1][ok])
    assert ctx[~ok].isnan().all() and not lse[~ok].isfinite().any()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("layout", ["baseline", "model", "tiny"])
def test_a_bad_query_reaches_its_own_head_alone(bits, layout):
    H, Hr, DL = LAYOUTS[layout]
    g = torch.Generator().manual_seed(51)
    lens = [700, 33, 5]
    cache = U.Cache(g, bits, DL, Hr, 32, lens)
    q_lat, q_rope = U.normal(g, 3, H, DL).cuda(), U.normal(g, 3, H, 64).cuda()
    rest = (*cache.dev(), cache.table.cuda(), i32(lens), 0.07)
    clean = T.paged_decode(q_lat, q_rope, *rest)
    q_lat[0, 1, 5], q_rope[1, 0, 63], q_lat[2, H - 1] = math.nan, math.inf, math.nan
    ctx, lse = T.paged_decode(q_lat, q_rope, *rest)
    ok = torch.ones(3, H, dtype=torch.bool)
    ok[0, 1] = ok[1, 0] = ok[2, H - 1] = False
    ok = ok.cuda()
    assert torch.equal(ctx[ok], clean[0][ok]) and torch.equal(lse[ok], clean[1][ok])
    assert ctx[~ok].isnan().any(-1).all()


def test_huge_and_tiny_values_in_16_bits():
    """Rows near bf16's ends whose scores stay finite."""
    g = torch.Generator().manual_seed(52)
    for std, qstd in ((1e15, 1e-15), (1e-20, 1.0), (3e18, 1e-19)):
        cache = U.Cache(g, 16, 512, 1, 16, [100, 9], std=std)
        q_lat, q_rope = U.normal(g, 2, 16, 512, std=qstd), U.normal(g, 2, 16, 64, std=qstd)
        got = T.paged_decode(q_lat.cuda(), q_rope.cuda(), *cache.dev(), cache.table.cuda(), i32([100, 9]), 0.07)
        check_decode(cache, q_lat, q_rope, [100, 9], 0.07, got)
