"""Operator cases: the feed-forward half of a block and the clipping of a step's gradients.

* ``ffn``: ``transformer_amd.gated_ffn``, ``y = residual + (act(x Wg^T) o (x Wu^T)) Wd^T``, with its backward where ``grad``;
* ``linear``: ``transformer_amd.linear_act``, ``y = act(x W^T + b) + residual``, with its backward where ``grad``;
* ``clip``: ``transformer_amd.clip_grad_norm_`` over a list of parameters' gradients.

Two widths occur throughout, both ``ModelArgs`` of this package: 1792 (the model that is trained) and 2048
(``ModelArgs.mla_baseline``), with a hidden layer of 4608.  Hidden states are N(0, 1), weights N(0, 0.02), all bf16.
"""
import math

import torch

own = False
DEV = "cuda"
VOCAB = 32768


def listed():
    return [
        # one user's reply, a token at a time: the smallest call, where latency counts
        {"name": "ffn_token", "kind": "ffn", "M": 1, "D": 1792, "H": 4608, "act": "silu", "residual": True, "grad": False},
        # a token of each sequence of a serving batch
        {"name": "ffn_decode", "kind": "ffn", "M": 32, "D": 2048, "H": 4608, "act": "silu", "residual": True, "grad": False},
        # a prompt of 1999 tokens
        {"name": "ffn_prompt", "kind": "ffn", "M": 1999, "D": 2048, "H": 4608, "act": "silu", "residual": True,
         "grad": False},
        # one block's step over the pretraining batch, 6 x 2048 tokens
        {"name": "ffn_train", "kind": "ffn", "M": 12288, "D": 1792, "H": 4608, "act": "silu", "residual": False,
         "grad": True},
        # the same fine-tuned on one long document of any length, with the other gate and a hidden layer of odd width
        {"name": "ffn_train_one", "kind": "ffn", "M": 3001, "D": 2048, "H": 5464, "act": "gelu_tanh", "residual": True,
         "grad": True},
        # the attention's output projection added to the residual stream, a token of each of 16 sequences
        {"name": "linear_decode", "kind": "linear", "M": 16, "K": 2048, "N": 2048, "act": "none", "bias": False,
         "residual": True, "grad": False},
        # an adapter's or a head's layer over a prompt: bias and activation, sizes that no tile divides
        {"name": "linear_prompt", "kind": "linear", "M": 2500, "K": 1800, "N": 1000, "act": "silu", "bias": True,
         "residual": False, "grad": False},
        # the first layer of an ungated feed-forward block over the pretraining batch, forward and backward
        {"name": "linear_train", "kind": "linear", "M": 12288, "K": 1792, "N": 4608, "act": "gelu_tanh", "bias": True,
         "residual": False, "grad": True},
        # the gradients of a small model: many small tensors, where latency counts
        {"name": "clip_small", "kind": "clip", "D": 256, "H": 640, "latent": 128, "layers": 4, "vocab": 1000,
         "dtype": "fp32"},
        # a bf16 model of the trained widths, fewer layers
        {"name": "clip_bf16", "kind": "clip", "D": 1792, "H": 4608, "latent": 384, "layers": 4, "vocab": VOCAB,
         "dtype": "bf16"},
        # fp32 gradients of the trained model itself, all layers
        {"name": "clip_model", "kind": "clip", "D": 1792, "H": 4608, "latent": 384, "layers": 28, "vocab": VOCAB,
         "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "linear", "linear", "clip"])
    if kind == "clip":
        return {"kind": kind, "D": 64 * _log(rng, 2, 28), "H": 8 * _log(rng, 50, 576), "latent": 8 * _log(rng, 8, 48),
                "layers": _log(rng, 1, 28), "vocab": _log(rng, 300, VOCAB), "dtype": rng.choice(["fp32", "bf16"])}
    grad = rng.random() < 0.5
    M = _log(rng, 1, 12000)
    if kind == "ffn":
        return {"kind": kind, "M": M, "D": 8 * _log(rng, 64, 224), "H": 8 * _log(rng, 128, 576),
                "act": rng.choice(["silu", "silu", "gelu_tanh", "relu"]), "residual": rng.random() < 0.5, "grad": grad}
    return {"kind": kind, "M": M, "K": 8 * _log(rng, 32, 576), "N": 8 * _log(rng, 32, 576),
            "act": rng.choice(["none", "silu", "gelu_tanh", "relu"]), "bias": rng.random() < 0.5,
            "residual": rng.random() < 0.5, "grad": grad}


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bf16(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _product_inputs(case, seed):
    """The inputs of a ffn or linear case by name, bf16; None where the case has none."""
    g = _gen(seed)
    M, res, grad = case["M"], case["residual"], case["grad"]
    if case["kind"] == "ffn":
        D, H = case["D"], case["H"]
        t = {"x": _bf16(g, M, D), "w_gate": _bf16(g, H, D, std=0.02), "w_up": _bf16(g, H, D, std=0.02),
             "w_down": _bf16(g, D, H, std=0.02)}
        out = D
    else:
        K, out = case["K"], case["N"]
        t = {"x": _bf16(g, M, K), "w": _bf16(g, out, K, std=0.02),
             "bias": _bf16(g, out, std=0.5) if case["bias"] else None}
    t["residual"] = _bf16(g, M, out) if res else None
    t["dy"] = _bf16(g, M, out) if grad else None
    return t


def _gradient_shapes(case):
    """The shapes of a model's parameters by layer: attention, feed-forward and norms of each, then embedding and norm."""
    D, H, dl = case["D"], case["H"], case["latent"]
    n = D // 64  # heads of 64 + 64, one rotated key a head
    layer = [(dl, D), (n * 64, dl), (2 * n * 64, D), (dl, D), (n * 64, dl), (n * 128, dl), (D, n * 128), (D,), (D,),
             (H, D), (H, D), (D, H)]
    return [layer] * case["layers"] + [[(case["vocab"], D), (D,)]]


def _buckets(case, seed):
    """One flat buffer of gradients for each layer, as a data-parallel step keeps them; layers differ in scale."""
    g = _gen(seed)
    dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    flat = []
    for i, shapes in enumerate(_gradient_shapes(case)):
        n = sum(math.prod(s) for s in shapes)
        flat.append((torch.randn(n, generator=g, device=DEV) * (0.02 / (1 + i))).to(dt))
    return flat


def prepare(case, seed):
    if case["kind"] != "clip":
        s = dict(_product_inputs(case, seed), case=case)
        if case["grad"]:
            s["leaves"] = [k for k in ("x", "w_gate", "w_up", "w_down", "w", "bias", "residual") if s.get(k) is not None]
            for k in s["leaves"]:
                s[k].requires_grad_()
        return s
    buckets, params = _buckets(case, seed), []
    for flat, shapes in zip(buckets, _gradient_shapes(case)):
        for part, shape in zip(flat.split([math.prod(s) for s in shapes]), shapes):
            p = torch.nn.Parameter(torch.empty(shape, dtype=flat.dtype, device=DEV))
            p.grad = part.view(shape)
            params.append(p)
    return {"case": case, "buckets": buckets, "params": params, "max_norm": 1.0}


# ------------------------------------------------------------------------------------------------ plain forms

def _act(z, name):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    return z.clamp_min(0) if name == "relu" else z


def _act_slope(z, name):
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * z * z)
    return (z > 0).to(z.dtype) if name == "relu" else torch.ones_like(z)


def _plain_ffn(s):
    act, dt = s["case"]["act"], torch.bfloat16
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    a = _act(g, act)
    y = (a * u) @ wd.t()
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    if s["dy"] is None:
        return {"y": y.to(dt)}
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * _act_slope(g, act), dh * a
    grads = {"x": dg @ wg + du @ wu, "w_gate": dg.t() @ x, "w_up": du.t() @ x, "w_down": dy.t() @ (a * u), "residual": dy}
    return {"y": y.to(dt), **{"d" + k: grads[k].to(dt) for k in s["leaves"]}}


def _plain_linear(s):
    act, dt = s["case"]["act"], torch.bfloat16
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, act)
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    if s["dy"] is None:
        return {"y": y.to(dt)}
    dy = s["dy"].float()
    dz = dy * _act_slope(z, act)
    grads = {"x": dz @ w, "w": dz.t() @ x, "bias": dz.sum(0), "residual": dy}
    return {"y": y.to(dt), **{"d" + k: grads[k].to(dt) for k in s["leaves"]}}


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()
    factor = (s["max_norm"] / (total + 1e-6)).clamp(max=1.0).float()
    [g.copy_(g.float() * factor) for g in grads]
    return {"norm": total.float(), "grads": s["buckets"]}


def run(state):
    case = state["case"]
    if not own:
        return {"ffn": _plain_ffn, "linear": _plain_linear, "clip": _plain_clip}[case["kind"]](state)
    import transformer_amd as T
    if case["kind"] == "clip":
        norm = T.clip_grad_norm_(state["params"], state["max_norm"])
        return {"norm": norm, "grads": state["buckets"]}
    with torch.set_grad_enabled(case["grad"]):
        if case["kind"] == "ffn":
            y = T.gated_ffn(state["x"], state["w_gate"], state["w_up"], state["w_down"], residual=state["residual"],
                            activation=case["act"])
        else:
            y = T.linear_act(state["x"], state["w"], bias=state["bias"], residual=state["residual"],
                             activation=case["act"])
    if not case["grad"]:
        return {"y": y}
    got = torch.autograd.grad(y, [state[k] for k in state["leaves"]], state["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(state["leaves"], got)}}


# ------------------------------------------------------------------------------------------------ the work of a pass

def work(case):
    """Each input read once, each output written once."""
    if case["kind"] == "clip":
        n = sum(math.prod(s) for shapes in _gradient_shapes(case) for s in shapes)
        return {"bytes": 2 * n * (4 if case["dtype"] == "fp32" else 2), "flops": 3 * n}
    M, grad = case["M"], case["grad"]
    K, N = (case["D"], case["D"]) if case["kind"] == "ffn" else (case["K"], case["N"])
    w = 3 * case["D"] * case["H"] if case["kind"] == "ffn" else K * N + (N if case["bias"] else 0)
    rows = M * (K + N + (N if case["residual"] else 0))
    values = rows + w
    flops = 2 * M * (3 * case["D"] * case["H"] if case["kind"] == "ffn" else K * N)
    if grad:
        values += rows + w  # dy in place of y, and each gradient
        flops *= 3
    return {"bytes": 2 * values, "flops": flops}


# ------------------------------------------------------------------------------------------------ 64 bits

def _slope64(z, name):
    """(act(z), act'(z)) from the definitions."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), torch.where(z > 0, 1.0, 0.0).double()
    if name == "silu":
        e = torch.exp(-z)
        return z / (1 + e), (1 + e + z * e) / (1 + e) ** 2
    c = math.sqrt(2 / math.pi)
    v = c * (z + 0.044715 * z ** 3)
    sech2 = 1 / torch.cosh(v) ** 2
    return z / 2 * (1 + torch.tanh(v)), (1 + torch.tanh(v)) / 2 + z / 2 * sech2 * c * (1 + 0.134145 * z ** 2)


def exact(case, seed):
    if case["kind"] == "clip":
        flat = [b.double() for b in _buckets(case, seed)]
        norm = math.sqrt(sum(float(torch.dot(b, b)) for b in flat))
        factor = min(1.0, 1.0 / (norm + 1e-6))
        return {"norm": norm, "grads": [b.mul_(factor) for b in flat]}
    t = {k: v.double() if v is not None else None for k, v in _product_inputs(case, seed).items()}
    x, dy, res = t["x"], t["dy"], t["residual"]
    out = {}
    if case["kind"] == "ffn":
        g, u = torch.mm(x, t["w_gate"].T), torch.mm(x, t["w_up"].T)
        a, slope = _slope64(g, case["act"])
        h = a * u
        y = torch.mm(h, t["w_down"].T)
        if dy is not None:
            dh = torch.mm(dy, t["w_down"])
            dg, du = dh * u * slope, dh * a
            out = {"dx": torch.mm(dg, t["w_gate"]) + torch.mm(du, t["w_up"]), "dw_gate": torch.mm(dg.T, x),
                   "dw_up": torch.mm(du.T, x), "dw_down": torch.mm(dy.T, h)}
    else:
        z = torch.mm(x, t["w"].T)
        if t["bias"] is not None:
            z = z + t["bias"]
        y, slope = _slope64(z, case["act"])
        if dy is not None:
            dz = dy * slope
            out = {"dx": torch.mm(dz, t["w"]), "dw": torch.mm(dz.T, x)}
            if t["bias"] is not None:
                out["dbias"] = dz.sum(0)
    if res is not None:
        y = y + res
        if dy is not None:
            out["dresidual"] = dy
    return {"y": y, **out}
