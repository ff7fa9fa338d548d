"""A paged latent cache and its operators in plain torch on the CPU, in 64 bits (what the paged tests compare with)."""
import math

import torch

BF16 = torch.bfloat16


def normal(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(BF16)


def quantise(rows):
    """bf16 [N, W] -> (codes int64 [N, W], scales bf16 [N, W / 64])."""
    x = rows.double().unflatten(-1, (-1, 64))
    scale = (x.abs().amax(-1) / 7).float().to(BF16)
    s = scale.double()[..., None]
    # the quotient of two bf16 values is nowhere near enough to a half for 64 bits to round differently
    q = torch.where(s > 0, (x / s).round().clamp(-7, 7), torch.zeros_like(x))
    return (torch.nan_to_num(q, nan=0.0) + 8).long().flatten(-2), scale


def values(codes, scales):
    return ((codes - 8).double().unflatten(-1, (-1, 64)) * scales.double()[..., None]).flatten(-2)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpack(pages):
    c = pages.long()
    return torch.stack([c & 15, c >> 4], -1).flatten(-2)


class Cache:
    """n pages of random rows and a table for B sequences with room for ``lengths`` tokens each."""

    def __init__(self, g, bits, DL, Hr, size, lengths, spare=3, std=1.0):
        self.bits, self.DL, self.Hr, self.size, self.W = bits, DL, Hr, size, DL + 64 * Hr
        need = [(n + size - 1) // size for n in lengths]
        self.n = sum(need) + spare
        order = torch.randperm(self.n, generator=g).tolist()
        self.table = torch.full((len(lengths), max(need) if need else 0), -1, dtype=torch.int32)
        for b, k in enumerate(need):
            for i in range(k):
                self.table[b, i] = order.pop()
        rows = normal(g, self.n * size, self.W, std=std)
        if bits == 16:
            self.pages, self.scales = rows.view(self.n, size, self.W), None
        else:
            codes, scales = quantise(rows)
            self.pages = pack(codes).view(self.n, size, self.W // 2)
            self.scales = scales.view(self.n, size, -1).transpose(1, 2).contiguous()

    def rows64(self):
        """float64 [n, size, W] of all pages."""
        if self.bits == 16:
            return self.pages.double()
        return values(unpack(self.pages), self.scales.transpose(1, 2))

    def dev(self):
        return self.pages.cuda(), None if self.scales is None else self.scales.cuda()

    def place(self, b, p):
        """(page, slot) of position p of sequence b, or None."""
        if p < 0 or p // self.size >= self.table.size(1):
            return None
        page = int(self.table[b, p // self.size])
        return (page, p % self.size) if 0 <= page < self.n else None


def tables(rows, theta=10000.0):
    a = torch.arange(rows).double()[:, None] * theta ** (-torch.arange(0, 64, 2).double() / 64)
    return a.cos().float().to(BF16), a.sin().float().to(BF16)


def rotate(x, c, s):
    """x bf16 [..., 64] with tables [32]: each product of two bf16 values is exact in fp32, so is rounded once, then to bf16."""
    a, b, c, s = x[..., :32].double(), x[..., 32:].double(), c.double(), s.double()
    return torch.cat([a * c - b * s, a * s + b * c], -1).float().to(BF16)


def append(cache, qk, c_new, cos, sin, starts, counts):
    """Writes into ``cache`` and returns the rotated queries."""
    B, T, heads, _ = qk.shape
    H = heads - cache.Hr
    q = torch.zeros(B, T, H, 64, dtype=BF16)
    limit = min(cos.size(0), cache.table.size(1) * cache.size)
    for b in range(B):
        for t in range(T if counts is None else min(T, max(0, int(counts[b])))):
            p = int(starts[b]) + t
            if not 0 <= p < limit:
                continue
            turned = rotate(qk[b, t], cos[p], sin[p])
            q[b, t] = turned[:H]
            at = cache.place(b, p)
            if at is None:
                continue
            row = torch.cat([c_new[b, t], turned[H:].flatten()])
            if cache.bits == 16:
                cache.pages[at] = row
            else:
                codes, scales = quantise(row[None])
                cache.pages[at] = pack(codes)[0]
                cache.scales[at[0], :, at[1]] = scales[0]
    return q


def read(cache, T, starts, counts, B):
    """bf16 (latent [B, T, DL], k_rope [B, Hr, T, 64])."""
    rows = torch.zeros(B, T, cache.W, dtype=torch.float64)
    all_rows = cache.rows64()
    for b in range(B):
        for t in range(T if counts is None else min(T, max(0, int(counts[b])))):
            at = cache.place(b, (0 if starts is None else int(starts[b])) + t)
            if at is not None:
                rows[b, t] = all_rows[at]
    rows = rows.float().to(BF16)  # (a code times a bf16 scale is exact in fp32)
    return rows[..., :cache.DL], rows[..., cache.DL:].unflatten(-1, (cache.Hr, 64)).transpose(1, 2)


def decode(cache, q_lat, q_rope, lens, scale):
    """float64 (ctx, lse) and the bounds of what bf16 and fp32 roundings can change of each.

    p is rounded to bf16 once (2^-8 of it), the result once (2^-8 of it).  A score is a sum of DL + 64 products in fp32; in 4 bits
    each run of 64 may be a sum of products with 16 + code, off which 24 times the queries' sum is taken, and the runs are added
    then: its error is at most 2^-24 (DL + 66) S, or 2^-24 (64 + DL / 64 + 6) S, with S the sum of the magnitudes added, which
    moves p by that much, and an exponential with the hardware's by 2^-22 (1 + the score's magnitude 2^-2 or so); sums over n
    tokens in fp32 add 2^-24 (n + 40) of the magnitudes added."""
    B, H, DL = q_lat.shape
    ctx, lse = torch.zeros(B, H, DL, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
    ctx_tol, lse_tol = torch.zeros_like(ctx), torch.zeros_like(lse)
    rows = cache.rows64()
    for b in range(B):
        at = [cache.place(b, p) for p in range(min(max(int(lens[b]), 0), cache.table.size(1) * cache.size))]
        at = [a for a in at if a is not None]
        if not at:
            continue
        page, slot = torch.tensor(at).T
        v = rows[page, slot]
        c, k = v[:, :DL], v[:, DL:].unflatten(-1, (cache.Hr, 64)).expand(-1, H, 64)
        ql, qr = q_lat[b].double(), q_rope[b].double()
        x = (c @ ql.T + (k * qr).sum(-1)) * scale  # [n, H]
        lse[b] = torch.logsumexp(x, 0)
        P = torch.softmax(x, 0)
        ctx[b] = P.T @ c
        ca, ka = c.abs(), k.abs()
        added = ca
        if cache.bits == 4:  # in scores 16 + code, at most 31, and 24; in ctx at most 128 + code, 143, and 136
            s = cache.scales.transpose(1, 2)[page, slot].double().repeat_interleave(64, -1)
            ca, ka = 55 * s[:, :DL], (55 * s[:, DL:]).unflatten(-1, (cache.Hr, 64)).expand(-1, H, 64)
            added = 279 * s[:, :DL]
        S = (ca @ ql.abs().T + (ka * qr.abs()).sum(-1)) * scale
        off = (2.0 ** -24 * (DL + 66 if cache.bits == 16 else DL // 64 + 70) * S + 2.0 ** -22 * (1 + x.abs() / 4)).amax(0)  # of a score, natural units
        A = P.T @ c.abs()
        n = len(at)
        ctx_tol[b] = 2.0 ** -8 * (ctx[b].abs() + 1.01 * A) + 2.1 * off[:, None] * A + 2.0 ** -24 * (n + 40) * (P.T @ added)
        lse_tol[b] = off + 2.0 ** -24 * (n + 40) + 2.0 ** -22 * lse[b].abs()
    return ctx, lse, ctx_tol, lse_tol
