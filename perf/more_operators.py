"""Operator cases: serving from a paged latent cache in 16 or 4 bits, and drawing the next tokens.

* ``append``: ``transformer_amd.paged_append``: new tokens' latents and rotated keys into pages, their rotated queries out;
* ``read``: ``transformer_amd.paged_read``: a prefix out of its pages, as the attention of a prompt's next chunk takes it;
* ``decode``: ``transformer_amd.paged_decode``: attention of one query token a sequence over its pages;
* ``sample``: ``transformer_amd.sample_tokens``: temperature, top-k, top-p, min-p and the draw, from given random numbers.

A cached row is ``[latent | rotated keys]``, W = d_latent + 64 Hr values.  In 16 bits ``pages`` is bf16 ``[n, size, W]`` and
``scales`` is None.  In 4 bits ``pages`` is uint8 ``[n, size, W / 2]`` (value 2 i in the low half of byte i) and ``scales`` bf16
``[n, W / 64, size]``: a run of 64 values of a row stands for ``(code - 8) scale``, ``scale = bf16(max |x| / 7)`` and
``code = 8 + rint(x / scale)`` within 1 .. 15 (8 where the scale is 0).

The head layouts are those of this package's ``ModelArgs``: "model" (14 heads, one rotated key each, latent 384) and
"baseline" (``mla_baseline``: 16 heads, one shared rotated key, latent 512).  Positions stay below ``mla_baseline``'s 16384.
"""
import math
import random

import torch

own = False
DEV = "cuda"
VOCAB, POSITIONS = 32768, 16384
LAYOUTS = {"model": (14, 14, 384), "baseline": (16, 1, 512)}  # query heads, rotated key heads, d_latent


def listed():
    return [
        # one user's reply, the trained model's heads: the smallest call, where latency counts
        {"name": "decode_reply", "kind": "decode", "layout": "model", "bits": 16, "B": 1, "L": 701, "size": 16},
        # a serving batch of sequences of any length, one slot of it empty
        {"name": "decode_serve", "kind": "decode", "layout": "baseline", "bits": 16, "B": 32, "L": 4096, "size": 64},
        # one user's long chat from a cache in 4 bits
        {"name": "decode4_reply", "kind": "decode", "layout": "baseline", "bits": 4, "B": 1, "L": 3001, "size": 32},
        # twice the batch for the same memory, every head with a rotated key of its own
        {"name": "decode4_serve", "kind": "decode", "layout": "model", "bits": 4, "B": 64, "L": 4000, "size": 16},
        # the largest: 64 documents up to the whole context
        {"name": "decode4_long", "kind": "decode", "layout": "baseline", "bits": 4, "B": 64, "L": 16384, "size": 128},
        # one user's next token into 16-bit pages: latency
        {"name": "append_token", "kind": "append", "layout": "model", "bits": 16, "B": 1, "T": 1, "size": 16},
        # a token of each sequence of a serving batch into 4-bit pages, and what these hold of it
        {"name": "append4_batch", "kind": "append", "layout": "baseline", "bits": 4, "B": 64, "T": 1, "size": 128},
        # eight prompts' chunks of any length into 4-bit pages, and what these hold of them
        {"name": "append4_prompts", "kind": "append", "layout": "baseline", "bits": 4, "B": 8, "T": 2048, "size": 64},
        # prompts in chunks: the prefix of each of four sequences, for the next chunk's attention
        {"name": "read_prefix", "kind": "read", "layout": "model", "bits": 16, "B": 4, "T": 8000, "size": 32},
        # one sequence's prefix out of 4-bit pages
        {"name": "read4_prefix", "kind": "read", "layout": "baseline", "bits": 4, "B": 1, "T": 5001, "size": 64},
        # one user's next token out of the trained model's vocabulary, the usual settings
        {"name": "sample_reply", "kind": "sample", "B": 1, "V": VOCAB, "dtype": "bf16", "mixed": False},
        # a large serving batch, each row with settings of its own, greedy and masked ones among them
        {"name": "sample_serve", "kind": "sample", "B": 256, "V": VOCAB, "dtype": "fp32", "mixed": True},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "append", "read", "sample", "sample"])
    if kind == "sample":
        V = _log(rng, 500, 4 * VOCAB)
        return {"kind": kind, "B": _log(rng, 1, min(256, 256 * VOCAB // V)), "V": V, "dtype": rng.choice(["bf16", "fp32"]),
                "mixed": rng.random() < 0.6}
    bits, layout, size = rng.choice([16, 4]), rng.choice(["model", "baseline"]), 16 * rng.choice([1, 1, 2, 3, 4, 8, 16])
    case = {"kind": kind, "layout": layout, "bits": bits, "size": size}
    if kind == "decode":
        L = _log(rng, 1, POSITIONS)
        # caches of up to 150 MB, which the largest listed case has too
        tokens = 150_000_000 // _row_bytes(case)
        return {**case, "B": _log(rng, 1, max(1, min(64, tokens // L))), "L": L}
    T = 1 if kind == "append" and rng.random() < 0.4 else _log(rng, 2, 8000)
    return {**case, "B": _log(rng, 1, min(64, max(1, 16384 // T))), "T": T}


# ------------------------------------------------------------------------------------------------ inputs

def _lens(case):
    """A length for each sequence: the first the longest, the others from an eighth of it on, a padded slot of a larger batch 0."""
    top, B = case.get("L") or case["T"], case["B"]
    rng = random.Random(1000003 * top + B)
    return [top] + [0 if b == B - 1 and B >= 8 else rng.randint((top + 7) // 8, top) for b in range(1, B)]


def _starts(case):
    """Positions that each sequence of an append or read begins at."""
    rng = random.Random(7 * case["T"] + case["B"])
    most = min(POSITIONS - case["T"], 4096, POSITIONS // case["B"])
    return [rng.randint(0, most) if case["kind"] == "append" else 0 for _ in range(case["B"])]


def _table(lengths, size, g):
    """(block table, number of pages): pages in any order, -1 where a sequence has none, one page in nine another user's."""
    need = torch.tensor([(n + size - 1) // size for n in lengths], device=DEV)
    width, used = max(1, int(need.max())), int(need.sum())
    total = used + used // 8 + 1
    held = torch.arange(width, device=DEV) < need[:, None]
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEV)
    table[held] = torch.randperm(total, generator=g, device=DEV)[:used].to(torch.int32)
    return table, total


def _quantised(x):
    """bf16 [..., W] -> (uint8 [..., W / 2], bf16 [..., W / 64])."""
    x = x.float().unflatten(-1, (-1, 64))
    scale = (x.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).float()
    code = torch.where(scale > 0, (x / scale).round().clamp(-7, 7), 0.0) + 8
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.squeeze(-1).to(torch.bfloat16)


def _rows(pages, scales, index):
    """fp32 [..., size, W] of the pages at ``index`` [...]."""
    if scales is None:
        return pages[index].float()
    c, s = pages[index], scales[index].float().transpose(-1, -2)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).float() - 8
    return (c.unflatten(-1, (-1, 64)) * s[..., None]).flatten(-2)


def _tables():
    angle = torch.arange(POSITIONS, device=DEV).float()[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, device=DEV).float() / 64)
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)

    if case["kind"] == "sample":
        return {"case": case, **_logits(case, g)}
    H, Hr, DL = LAYOUTS[case["layout"]]
    B, size, W = case["B"], case["size"], DL + 64 * Hr
    lens = _lens(case)
    starts = _starts(case) if case["kind"] != "decode" else [0] * B
    table, n = _table([a + c for a, c in zip(starts, lens)], size, g)
    pages, scales = normal(n, size, W), None
    if case["bits"] == 4:
        pages, scales = _quantised(pages)
        scales = scales.transpose(1, 2).contiguous()
    i32 = dict(dtype=torch.int32, device=DEV)
    s = {"case": case, "pages": pages, "scales": scales, "table": table, "lens": torch.tensor(lens, **i32)}
    if case["kind"] == "decode":
        return {**s, "q_lat": normal(B, H, DL), "q_rope": normal(B, H, 64), "scale": 192 ** -0.5}
    s["starts"] = torch.tensor(starts, **i32)
    if case["kind"] == "append":
        s["cos"], s["sin"] = _tables()
        s["qk"], s["c_new"] = normal(B, case["T"], H + Hr, 64), normal(B, case["T"], DL)
    return s


def _logits(case, g):
    """A model's logits: rows from flat to nearly certain; in a mixed batch some have a grammar's mask or a value out of range."""
    B, V = case["B"], case["V"]
    spread = 1 + 3 * torch.rand(B, 1, generator=g, device=DEV)
    x = torch.randn(B, V, generator=g, device=DEV) * spread
    s = {"u": torch.rand(B, generator=g, device=DEV)}
    if case["mixed"]:
        pick = torch.rand(B, generator=g, device=DEV)
        masked = (pick < 0.2)[:, None] & (torch.rand(B, V, generator=g, device=DEV) < 0.98)
        x = x.masked_fill(masked, -math.inf)

        def some(values, dtype):
            at = torch.randint(len(values), (B,), generator=g, device=DEV)
            return torch.tensor(values, dtype=dtype, device=DEV)[at]

        s.update(temperature=some([0.0, 0.5, 0.7, 1.0, 1.3], torch.float32), top_k=some([0, 0, 1, 20, 50, 400], torch.int32),
                 top_p=some([1.0, 0.95, 0.9, 0.5], torch.float32), min_p=some([0.0, 0.0, 0.02, 0.1], torch.float32))
    else:
        s.update(temperature=0.8, top_k=50, top_p=0.95, min_p=0.0)
    return {"logits": x.to(torch.bfloat16) if case["dtype"] == "bf16" else x, **s}


# ------------------------------------------------------------------------------------------------ plain forms

def _places(s, T):
    """(positions [B, T], page of each or 0, whether it is one of the sequence's tokens)."""
    t = torch.arange(T, device=DEV)
    at = s["starts"][:, None].long() + t
    inside = t < s["lens"][:, None]
    page = s["table"].long().gather(1, (at // s["case"]["size"]).clamp(max=s["table"].size(1) - 1))
    return at, page.clamp(min=0), inside


def _plain_read(s):
    _, Hr, DL = LAYOUTS[s["case"]["layout"]]
    size, T = s["case"]["size"], s["case"]["T"]
    at, page, inside = _places(s, T)
    if s["scales"] is None:
        rows = s["pages"][page, at % size].float()
    else:
        c, k = s["pages"][page, at % size], s["scales"][page, :, at % size].float()
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2).float() - 8
        rows = (c.unflatten(-1, (-1, 64)) * k[..., None]).flatten(-2)
    rows = torch.where(inside[..., None], rows, 0.0).to(torch.bfloat16)
    return {"latent": rows[..., :DL].contiguous(), "k_rope": rows[..., DL:].unflatten(-1, (Hr, 64)).transpose(1, 2).contiguous()}


def _plain_append(s):
    H, _, _ = LAYOUTS[s["case"]["layout"]]
    size, T = s["case"]["size"], s["case"]["T"]
    at, page, inside = _places(s, T)
    c, n = s["cos"][at].float()[:, :, None], s["sin"][at].float()[:, :, None]
    a, b = s["qk"].float().split(32, -1)
    turned = torch.cat([a * c - b * n, a * n + b * c], -1).to(torch.bfloat16)
    q = torch.where(inside[..., None, None], turned[:, :, :H], 0.0).to(torch.bfloat16)
    rows = torch.cat([s["c_new"], turned[:, :, H:].flatten(-2)], -1)[inside]
    page, slot = page[inside], (at % size)[inside]
    if s["scales"] is None:
        s["pages"][page, slot] = rows
        return {"q_rope": q, "pages": s["pages"]}
    code, scale = _quantised(rows)
    s["pages"][page, slot] = code
    s["scales"][page, :, slot] = scale
    return {"q_rope": q, **_plain_read(s)}


def _plain_decode(s):
    _, Hr, DL = LAYOUTS[s["case"]["layout"]]
    rows = _rows(s["pages"], s["scales"], s["table"].long().clamp(min=0)).flatten(1, 2)  # [B, L, W]
    lat, q = rows[..., :DL].contiguous(), s["q_rope"].float()
    x = torch.matmul(s["q_lat"].float(), lat.transpose(1, 2).contiguous())
    if Hr == 1:
        x = x + torch.matmul(q, rows[..., DL:].transpose(1, 2).contiguous())
    else:
        x = x + (rows[..., DL:].unflatten(-1, (Hr, 64)) * q[:, None]).sum(-1).transpose(1, 2)
    inside = torch.arange(rows.size(1), device=DEV) < s["lens"][:, None, None]
    x = (x * s["scale"]).masked_fill(~inside, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    ctx = torch.matmul(p / torch.where(total == 0, 1.0, total), lat)
    return {"ctx": ctx.to(torch.bfloat16), "lse": (top + total.log()).squeeze(-1)}


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape

    def column(name, dtype):
        return torch.as_tensor(s[name], device=DEV).to(dtype).expand(B)[:, None]

    temperature, top_p, min_p = (column(k, torch.float32).double() for k in ("temperature", "top_p", "min_p"))
    top_k, u = column("top_k", torch.int64), s["u"].double()[:, None]
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    greedy = temperature <= 0
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, temperature)))
    w = torch.where(x == -math.inf, 0.0, w)
    order = x.sort(dim=1, descending=True, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(V, device=DEV)
    keep = rank < torch.where(greedy, 1, torch.where(top_k <= 0, V, top_k))
    w = w * keep
    before = w.cumsum(1) - w
    keep = (rank == 0) | (top_p >= 1) | (before < top_p * w.sum(1, keepdim=True))
    w = w * keep * (w >= min_p)
    w = torch.zeros_like(w).scatter(1, order, w)
    run_up = w.cumsum(1)
    total = run_up[:, -1:]
    hit = run_up > u * total
    token = torch.where(hit.any(1), hit.byte().argmax(1), -1)
    weight = w.gather(1, token.clamp(min=0)[:, None])
    return {"token": token, "logprob": torch.where(token[:, None] < 0, -math.inf, (weight / total).log()).squeeze(1).float()}


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "sample": _plain_sample}[case["kind"]](state)
    import transformer_amd as T
    s = state
    if case["kind"] == "sample":
        token, logprob = T.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                         min_p=s["min_p"])
        return {"token": token, "logprob": logprob}
    if case["kind"] == "decode":
        ctx, lse = T.paged_decode(s["q_lat"], s["q_rope"], s["pages"], s["scales"], s["table"], s["lens"], s["scale"])
        return {"ctx": ctx, "lse": lse}
    out = {}
    if case["kind"] == "append":
        out["q_rope"] = T.paged_append(s["qk"], s["c_new"], s["pages"], s["scales"], s["cos"], s["sin"], s["table"], s["starts"],
                                       counts=s["lens"])
        if case["bits"] == 16:
            return {**out, "pages": s["pages"]}
    d_latent = LAYOUTS[case["layout"]][2]
    latent, k_rope = T.paged_read(s["pages"], s["scales"], s["table"], d_latent, case["T"], starts=s["starts"], counts=s["lens"])
    return {**out, "latent": latent, "k_rope": k_rope}


# ------------------------------------------------------------------------------------------------ the work of a pass

def _row_bytes(case):
    _, Hr, DL = LAYOUTS[case["layout"]]
    W = DL + 64 * Hr
    return 2 * W if case["bits"] == 16 else W // 2 + W // 32


def work(case):
    """Each input read once, each output written once; an append to 4-bit pages with what reads it back."""
    if case["kind"] == "sample":
        n = case["B"] * case["V"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 16 * case["B"], "flops": 4 * n}
    H, Hr, DL = LAYOUTS[case["layout"]]
    W, n, B = DL + 64 * Hr, sum(_lens(case)), case["B"]
    row = _row_bytes(case)
    if case["kind"] == "decode":
        return {"bytes": n * row + B * H * (2 * (2 * DL + 64) + 4), "flops": 2 * n * H * (2 * DL + 64)}
    read = n * row + 2 * B * case["T"] * W
    if case["kind"] == "read":
        return {"bytes": read, "flops": n * W}
    append = 2 * n * (64 * (H + Hr) + DL) + 2 * B * case["T"] * 64 * H + n * row
    return {"bytes": append + (read if case["bits"] == 4 else 0), "flops": 6 * n * (32 * (H + Hr)) + 4 * n * W}


# ------------------------------------------------------------------------------------------------ 64 bits

def _row64(s, b, length, first=0):
    """float64 [length, W]: the values that sequence b's tokens from ``first`` on stand for."""
    t = torch.arange(first, first + length, device=DEV)
    size = s["case"]["size"]
    page, slot = s["table"][b].long()[t // size], t % size
    if s["scales"] is None:
        return s["pages"][page, slot].double()
    byte = s["pages"][page, slot].int()
    v = torch.empty(length, 2 * byte.size(1), dtype=torch.float64, device=DEV)
    v[:, 0::2], v[:, 1::2] = (byte % 16 - 8).double(), (byte // 16 - 8).double()
    for k in range(v.size(1) // 64):
        v[:, 64 * k:64 * k + 64] *= s["scales"][page, k, slot].double()[:, None]
    return v


def _exact_append(s, case):
    H, Hr, DL = LAYOUTS[case["layout"]]
    T, size = case["T"], case["size"]
    W = DL + 64 * Hr
    q = torch.zeros(case["B"], T, H, 64, dtype=torch.float64, device=DEV)
    rows = torch.zeros(case["B"], T, W, dtype=torch.float64, device=DEV)
    pages = s["pages"].double() if case["bits"] == 16 else None
    for b, (first, n) in enumerate(zip(_starts(case), _lens(case))):
        z = torch.view_as_complex(torch.stack([s["qk"][b, :n, :, :32].double(), s["qk"][b, :n, :, 32:].double()], -1))
        at = slice(first, first + n)
        z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        z = torch.cat([z.real, z.imag], -1)
        q[b, :n] = z[:, :H]
        new = torch.cat([s["c_new"][b, :n].double(), z[:, H:].flatten(1)], 1)
        if case["bits"] == 16:
            t = torch.arange(first, first + n, device=DEV)
            pages[s["table"][b].long()[t // size], t % size] = new
            continue
        new[:, DL:] = new[:, DL:].float().to(torch.bfloat16).double()  # a cache holds the rotated key rounded to bf16
        for k in range(W // 64):
            x = new[:, 64 * k:64 * k + 64]
            step = (x.abs().max(1).values / 7).float().to(torch.bfloat16).double()[:, None]
            rows[b, :n, 64 * k:64 * k + 64] = torch.where(step > 0, (x / step).round().clamp(-7, 7), 0.0) * step
    if case["bits"] == 16:
        return {"q_rope": q, "pages": pages}
    return {"q_rope": q, "latent": rows[..., :DL], "k_rope": rows[..., DL:].reshape(case["B"], T, Hr, 64).permute(0, 2, 1, 3)}


def _exact_sample(s, case):
    B, V = case["B"], case["V"]
    token = torch.full((B,), -1, dtype=torch.int64, device=DEV)
    logprob = torch.full((B,), -math.inf, dtype=torch.float64, device=DEV)

    def at(name, b):
        v = s[name]
        return float(v[b]) if torch.is_tensor(v) else float(torch.tensor(v, dtype=torch.float32))

    for b in range(B):
        x = s["logits"][b].double()
        live = torch.nonzero(x > -math.inf).flatten()
        if not live.numel():
            continue
        # the living tokens, the likeliest first, of equal ones the lowest
        live = live[torch.argsort(x[live], descending=True, stable=True)]
        t, k = at("temperature", b), int(at("top_k", b))
        live = live[:1] if t <= 0 else live[:k] if k > 0 else live
        w = torch.exp((x[live] - x[live[0]]) / (t if t > 0 else 1.0))
        share = w / w.sum()
        if at("top_p", b) < 1:
            n = int((share.cumsum(0) - share < at("top_p", b)).sum())
            live, w = live[:max(1, n)], w[:max(1, n)]
        live, w = live[w >= at("min_p", b)], w[w >= at("min_p", b)]
        live, by = live.sort()
        w = w[by] / w.sum()
        i = min(int((w.cumsum(0) <= float(s["u"][b])).sum()), live.numel() - 1)
        token[b], logprob[b] = live[i], w[i].log()
    return {"token": token, "logprob": logprob}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s, case)
    if case["kind"] == "append":
        return _exact_append(s, case)
    H, Hr, DL = LAYOUTS[case["layout"]]
    if case["kind"] == "read":
        rows = torch.zeros(case["B"], case["T"], DL + 64 * Hr, dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lens(case)):
            rows[b, :n] = _row64(s, b, n)
        return {"latent": rows[..., :DL], "k_rope": rows[..., DL:].reshape(case["B"], case["T"], Hr, 64).permute(0, 2, 1, 3)}
    ctx = torch.zeros(case["B"], H, DL, dtype=torch.float64, device=DEV)
    lse = torch.full((case["B"], H), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(case)):
        if n:
            v = _row64(s, b, n)
            keys = v[:, DL:].reshape(n, Hr, 64).expand(n, H, 64)
            x = v[:, :DL] @ s["q_lat"][b].double().T + torch.einsum("nhd,hd->nh", keys, s["q_rope"][b].double())
            x = x * s["scale"]
            lse[b] = torch.logsumexp(x, 0)
            ctx[b] = torch.softmax(x, 0).T @ v[:, :DL]
    return {"ctx": ctx, "lse": lse}
