"""The linear layers' operators (``torch.ops.mla_mi355x.linear_act``, ``gated_ffn`` and their backwards).

They are registered as those of ``kernels`` are.  ``linear`` and ``gated`` are what eager callers take: the same bodies without
the dispatcher where nothing needs it, with an autograd.Function where a gradient is all that is needed.  There is no CPU path:
a CPU tensor, or a missing library, raises.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib, kernels
from ._lib import ACTIVATIONS
from .kernels import _alloc_workspace, _dt_code, _op, _register_autograd

LINEAR_MAX_STRIDE = 1 << 22
REACH = 1 << 30  # elements that a weight read across its rows, and 64 rows more, lie within (mla_linear_dx, mla_gated_linear_bwd)
ROWS_MAX = 64  # rows up to which mla_linear_act and mla_gated_linear need no workspace
_BF16, _F32 = torch.bfloat16, torch.float32
_byref, _current_device, _raw_stream = ctypes.byref, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


# ----------------------------------------------------------------- helpers

def _launch(entry: str, args, like: Tensor, op: str) -> None:
    """Call a C entry point on ``like``'s device and its current stream, whichever device is the current one."""
    fn, dev = _lib.entry(entry), like.get_device()
    if dev == _current_device():
        rc = fn(_byref(args), _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(_byref(args), _raw_stream(dev))
    if rc:
        _lib.check(rc, op)


def _fit_workspace(entry: str, args, like: Tensor) -> Optional[Tensor]:
    """The workspace that ``entry`` (a ``*_workspace_bytes`` function) asks for, set in ``args``; keep it until the call."""
    nbytes = _lib.entry(entry)(_byref(args))
    if not nbytes:
        return None
    ws = _alloc_workspace(nbytes, like.device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _rows(t: Tensor, K: int, one_row: bool = False) -> Tuple[Tensor, int]:
    """``t [..., K]`` as rows the linear kernels take, and their stride: unit inner stride, 16-byte aligned, a row stride that is
    a multiple of 8 and covers a row (``one_row``: or 0, the same row for all); copied where its layout is another."""
    if t.dim() != 2:
        t = t.reshape(-1, K)
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, K
        s, inner = t.stride()
        if inner == 1:
            if t.size(0) <= 1:
                return t, K
            if s % 8 == 0 and s < LINEAR_MAX_STRIDE and (s >= K or (one_row and s == 0)):
                return t, s
    return t.clone(memory_format=torch.contiguous_format), K


def _weight_rows(w: Tensor, K: int) -> Tuple[Tensor, int]:  # (and a gradient's)
    return _rows(w if w.dtype == _BF16 else w.to(_BF16), K)


def _activation(op: str, name: str, gate: bool = False) -> int:
    code = ACTIVATIONS.get(name)
    if code is None or (gate and code == 0):
        raise ValueError(f"{op}: activation {name!r} is not one of {[a for a in ACTIVATIONS if not (gate and a == 'none')]}")
    return code


def _check(op: str, x: Tensor, weights, names, residual: Optional[Tensor], n_out: int) -> None:
    """Types, devices and sizes of the inputs (their shapes were compared already)."""
    dev, ok = x.get_device(), x.dtype == _BF16 and x.is_cuda
    for t in weights:
        if t is not None:
            ok = ok and (t.dtype == _BF16 or t.dtype == _F32) and t.get_device() == dev
            if ok and t.dim() == 2:
                n, k = t.shape
                ok = not (n % 8 or k % 8) and n * k > 0
    if residual is not None:
        ok = ok and residual.dtype == _BF16 and residual.get_device() == dev \
            and residual.shape[:-1] == x.shape[:-1] and residual.shape[-1:] == (n_out,)
    if not ok:
        _refuse(op, x, weights, names, residual, n_out)


def _refuse(op: str, x: Tensor, weights, names, residual: Optional[Tensor], n_out: int) -> None:
    """The error of inputs that :func:`_check` did not pass."""
    kernels._require_gpu(op, x, residual, *weights)
    if x.dtype != _BF16:
        raise TypeError(f"{op}: x must be bfloat16, got {x.dtype}")
    for t, name in zip(weights, names):
        if t is None:
            continue
        if t.dtype != _BF16 and t.dtype != _F32:
            raise TypeError(f"{op}: {name} must be bfloat16 or float32, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{op}: {name} is on {t.device}, x on {x.device}")
        if t.dim() == 2 and (t.size(0) % 8 or t.size(1) % 8 or not t.numel()):
            raise ValueError(f"{op}: {name} {tuple(t.shape)}: both sizes must be positive multiples of 8")
    if residual.dtype != _BF16:
        raise TypeError(f"{op}: residual must be bfloat16, got {residual.dtype}")
    raise ValueError(f"{op}: residual must be {(*x.shape[:-1], n_out)} on {x.device}, got {tuple(residual.shape)} on "
                     f"{residual.device}")


def _refuse_bwd(op: str, fits: bool, x: Tensor, dy: Tensor, weights, saved: Optional[Tensor], h: Optional[Tensor] = None) -> None:
    """The error of a backward's operands that its launches must not see; ``fits``: whether the shapes belong together."""
    if not fits:
        raise ValueError(f"{op}: dy {tuple(dy.shape)}, x {tuple(x.shape)}, weights {[tuple(w.shape) for w in weights]}"
                         f"{'' if h is None else f', h {tuple(h.shape)}'} and saved "
                         f"{'(none)' if saved is None else tuple(saved.shape)} do not belong together")
    if x.dtype != _BF16 or (h is not None and h.dtype != _BF16) or (saved is not None and saved.dtype != torch.uint8) \
            or any(w.dtype != _BF16 and w.dtype != _F32 for w in weights):
        raise TypeError(f"{op}: x and h must be bfloat16, weights bfloat16 or float32 and saved uint8")
    if any(t is not None and not t.is_contiguous() for t in (h, saved)):
        raise ValueError(f"{op}: h and saved must be contiguous")
    kernels._require_gpu(op, x, dy, *weights, h, saved)
    raise ValueError(f"{op}: all tensors must be on one device")


def _saved_size(M: int, N: int) -> int:
    return (3 << 10) * ((M + 31) // 32) * ((N + 31) // 32)  # mla_linear_saved_size


def _linear_run(op, x2, x_stride, weight, bias, residual, code, saved, y, M, N, K):
    """``y = act(x2 weight^T + bias) + residual`` on bf16 rows as :func:`_rows` leaves them; bias contiguous, aligned to four of
    its elements."""
    w, w_stride = _weight_rows(weight, K)
    res2, r_stride = (None, 0) if residual is None else _rows(residual, N, True)
    args = _lib.LinearActArgs(
        x2.data_ptr(), w.data_ptr(), None if bias is None else bias.data_ptr(), None if res2 is None else res2.data_ptr(),
        y.data_ptr(), None if saved is None else saved.data_ptr(), None, 0, M, N, K, x_stride, w_stride, r_stride, N, code,
        0 if bias is None else _dt_code(bias))
    ws = _fit_workspace("mla_linear_act_workspace_bytes", args, y) if M > ROWS_MAX else None  # noqa: F841  (kept until the launch)
    _launch("mla_linear_act", args, y, op)


# ----------------------------------------------------------------- linear layer with its epilogue

def _linear_act(x, weight, bias, residual, activation, save):
    """``(y, saved or None)``; see :func:`linear_act`."""
    op = "mla_mi355x::linear_act"
    code = _activation(op, activation)
    if weight.dim() != 2 or x.dim() < 1 or x.size(-1) != weight.size(1) or (bias is not None
                                                                            and bias.shape != (weight.size(0),)):
        raise ValueError(f"{op}: expected x [..., K], weight [N, K], bias [N]; got {tuple(x.shape)}, {tuple(weight.shape)}, "
                         f"{None if bias is None else tuple(bias.shape)}")
    N, K = weight.shape
    _check(op, x, (weight, bias), ("weight", "bias"), residual, N)
    x2, x_stride = _rows(x, K)
    M = x2.size(0)
    y = x.new_empty((*x.shape[:-1], N))
    saved = x.new_empty(_saved_size(M, N), dtype=torch.uint8) if save and code else None
    if M:
        b = bias
        if b is not None:
            b = b.contiguous()
            if b.data_ptr() % (4 * b.element_size()):
                b = b.clone()
        _linear_run(op, x2, x_stride, weight, b, residual, code, saved, y, M, N, K)
    return y, saved


@_op("linear_act", mutates_args=())
def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], activation: str,
               save: bool) -> Tuple[Tensor, Tensor]:
    """``y = act(x W^T + bias) + residual`` for bf16 ``x [..., K]``, ``weight [N, K]`` (bf16, or fp32 read as bf16), ``bias
    [N]`` (bf16 or fp32), ``residual [..., N]`` bf16: fp32 sums and epilogue, one rounding.  ``activation``: none, relu, silu,
    gelu_tanh.  Returns ``y`` and, with ``save`` and an activation, what the backward keeps of the pre-activation (else an empty
    tensor).  K and N multiples of 8."""
    y, saved = _linear_act(x, weight, bias, residual, activation, save)
    return y, x.new_empty(0, dtype=torch.uint8) if saved is None else saved


def _saved_fake(x, K, N, blocks, wanted):
    return x.new_empty(blocks * _saved_size(x.numel() // K, N) if wanted else 0, dtype=torch.uint8)


@linear_act.register_fake
def _(x, weight, bias, residual, activation, save):
    N, K = weight.shape
    return x.new_empty(*x.shape[:-1], N), _saved_fake(x, K, N, 1, save and activation != "none")


def _weight_grad(dy: Tensor, sy: int, x: Tensor, sx: int, dtype: torch.dtype) -> Tensor:
    """``dy^T x`` in ``dtype`` for rows of strides ``sy`` and ``sx`` as :func:`_rows` leaves them, any number of them: those beyond
    the kernel's reach in several parts, added in fp32."""
    (M, N), K = dy.shape, x.size(1)
    if M == 0:
        return torch.zeros(N, K, dtype=dtype, device=dy.device)
    if kernels.weight_grad_fits(M, N, K, sy, sx):
        dw = torch.empty((N, K), dtype=dtype, device=dy.device)
        args = _lib.WeightGradArgs(dy.data_ptr(), x.data_ptr(), dw.data_ptr(), None, 0, M, N, K, sy, sx, K, _dt_code(dw))
        ws = _fit_workspace("mla_weight_grad_workspace_bytes", args, dw)  # noqa: F841  (kept until the launch)
        _launch("mla_weight_grad", args, dw, "mla_mi355x::weight_grad")
        return dw
    if max(sy, sx) > 1 << 20:  # (few rows would be within reach: closer together)
        dy, x, sy, sx = dy.contiguous(), x.contiguous(), N, K
    rows = min((1 << 30) // max(sy, sx) - 257, (1 << 24) - 1)
    dw = None
    for r in range(0, M, rows):
        part = kernels.weight_grad(dy[r:r + rows], x[r:r + rows], True)
        dw = part if dw is None else dw.add_(part)
    return dw.to(dtype)


def _columns(rows: int, cols: int) -> int:
    """How many of the columns of a weight that is read across its rows one call takes from a copy: all of them, or whole
    blocks of 256 within its reach."""
    return cols if (rows + 64) * cols < REACH else (REACH - 1) // (rows + 64) // 256 * 256


def _linear_dx(op: str, dy: Tensor, sy: int, weights, shape) -> Tensor:
    """``sum_p dy_p W_p`` for bf16 rows ``dy [M, P N]`` of stride ``sy`` and P = 1 or 2 weights ``[N, K]``, as ``shape``."""
    (N, K), M = weights[0].shape, dy.size(0)
    dx = dy.new_empty(shape)
    if not M:
        return dx
    w0, s0 = _weight_rows(weights[0], K)
    w1, s1 = _weight_rows(weights[1], K) if len(weights) > 1 else (None, s0)
    as_they_lie = s1 == s0 and (N + 64) * s0 < REACH  # (one stride for both)
    cols = K if as_they_lie else _columns(N, K)
    for c in range(0, K, cols):
        n, s, p0, p1 = min(cols, K - c), s0, w0, w1
        if not as_they_lie:
            s, p0, p1 = n, w0[:, c:c + n].contiguous(), None if w1 is None else w1[:, c:c + n].contiguous()
        args = _lib.LinearDxArgs(dy.data_ptr(), p0.data_ptr(), None if p1 is None else p1.data_ptr(), dx.data_ptr() + 2 * c, None, 0,
                                 M, N, n, sy, s, 0 if p1 is None else s, K)
        ws = _fit_workspace("mla_linear_dx_workspace_bytes", args, dx)  # noqa: F841  (kept until the launch)
        _launch("mla_linear_dx", args, dx, op)
    return dx


def _linear_act_bwd(dy, x, weight, saved, activation, need_dx, need_dw, db_dtype):
    """``(dx, dw, db)``, None where not needed; see :func:`linear_act_bwd`."""
    op = "mla_mi355x::linear_act_bwd"
    code = _activation(op, activation)
    if db_dtype is not None and db_dtype != _BF16 and db_dtype != _F32:
        raise TypeError(f"{op}: db_dtype must be bfloat16 or float32, got {db_dtype}")
    N, K = weight.shape if weight.dim() == 2 else (0, 0)
    M, dev = x.numel() // K if K else 0, x.get_device()
    # (without generators: a training pass of few rows is bound by the host)
    fits = N > 0 and x.dim() > 0 and x.size(-1) == K and dy.shape == (*x.shape[:-1], N) \
        and (not code or saved.numel() == _saved_size(M, N))
    if not (fits and x.dtype == _BF16 and (weight.dtype == _BF16 or weight.dtype == _F32)
            and 0 <= dev == dy.get_device() == weight.get_device()
            and (not code or (saved.dtype == torch.uint8 and saved.is_contiguous() and saved.get_device() == dev))):
        _refuse_bwd(op, fits, x, dy, (weight,), saved if code else None)
    (dy2, sy), (x2, sx) = _weight_rows(dy, N), _rows(x, K)
    dz, db = dy2, None
    if db_dtype is not None:
        db = (torch.empty if M else torch.zeros)(N, dtype=db_dtype, device=x.device)
    if M and (code or db is not None):
        if code:
            dz = x.new_empty((M, N))
        args = _lib.ActGradArgs(dy2.data_ptr(), saved.data_ptr() if code else None, dz.data_ptr() if code else None,
                                None if db is None else db.data_ptr(), None, 0, M, N, sy, N, code,
                                0 if db is None else _dt_code(db))
        ws = None if db is None else _fit_workspace("mla_act_grad_workspace_bytes", args, dy2)  # noqa: F841
        _launch("mla_act_grad", args, dy2, op)
    sz = N if code else sy
    return (_linear_dx(op, dz, sz, (weight,), x.shape) if need_dx else None,
            _weight_grad(dz, sz, x2, sx, weight.dtype) if need_dw else None, db)


@_op("linear_act_bwd", mutates_args=())
def linear_act_bwd(dy: Tensor, x: Tensor, weight: Tensor, saved: Tensor, activation: str, need_dx: bool, need_dw: bool,
                   db_dtype: Optional[torch.dtype]) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients ``(dx, dw, db)`` of :func:`linear_act` from ``dy`` and what it saved; ``dw`` in the weight's dtype, ``db`` in
    ``db_dtype`` (None: no bias).  Empty tensors where a gradient is not needed."""
    got = _linear_act_bwd(dy, x, weight, saved, activation, need_dx, need_dw, db_dtype)
    return tuple(x.new_empty(0) if t is None else t for t in got)


@linear_act_bwd.register_fake
def _(dy, x, weight, saved, activation, need_dx, need_dw, db_dtype):
    return (x.new_empty(x.shape if need_dx else 0), weight.new_empty(weight.shape) if need_dw else x.new_empty(0),
            x.new_empty(0) if db_dtype is None else x.new_empty(weight.size(0), dtype=db_dtype))


def _plain_backward(dy: Tensor) -> bool:
    """Whether a backward may run the bodies: it is not itself differentiated, batched, traced or under a dispatch mode."""
    return not (torch.is_grad_enabled() or type(dy) is not Tensor or kernels.batched_grad(dy)
                or torch._C._get_tracing_state() is not None or torch._C._len_torch_dispatch_stack() > 0
                or torch._C._functorch.peek_interpreter_stack() is not None)


def _linear_act_grads(ctx, dy, need):
    """The gradients for (x, weight, bias) from the saved tensors of either autograd path."""
    x, weight, bias, saved = ctx.saved_tensors
    plain = _plain_backward(dy)
    if ctx.activation != "none" and (saved is None or not saved.numel()) and x.numel():  # not kept: the product again
        saved = torch.ops.mla_mi355x.linear_act(x.detach(), weight.detach(), None if bias is None else bias.detach(), None,
                                                ctx.activation, True)[1]
    if saved is None:
        saved = x.new_empty(0, dtype=torch.uint8)
    run = _linear_act_bwd if plain else torch.ops.mla_mi355x.linear_act_bwd
    got = run(dy, x, weight, saved, ctx.activation, need[0], need[1], bias.dtype if bias is not None and need[2] else None)
    return tuple(g if n else None for g, n in zip(got, (need[0], need[1], bias is not None and need[2])))


def _linear_act_setup(ctx, inputs, output):
    x, weight, bias, residual, activation, _ = inputs
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1])


def _linear_act_backward(ctx, dy, dsaved):
    need = ctx.needs_input_grad
    grads = _linear_act_grads(ctx, dy, need) if any(need[:3]) else (None,) * 3
    return (*grads, dy if need[3] else None, None, None)


_register_autograd(linear_act, "linear_act", _linear_act_setup, _linear_act_backward)


class _LinearAct(torch.autograd.Function):
    """The operator's body and formula without its dispatch (60 to 80 us of host time a call)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        with kernels.below_autograd():
            y, saved = _linear_act(x, weight, bias, residual, activation, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        grads = _linear_act_grads(ctx, dy, need) if any(need[:3]) else (None,) * 3
        return (*grads, dy if need[3] else None, None)


def linear(x, weight, bias, residual, activation) -> Tensor:
    """:func:`linear_act`'s ``y`` for eager callers."""
    args = (x, weight, bias, residual)
    if kernels._needs_grad(args):
        if kernels.function_fits(args):
            return _LinearAct.apply(x, weight, bias, residual, activation)
        return torch.ops.mla_mi355x.linear_act(x, weight, bias, residual, activation, True)[0]
    if kernels._not_plain(args):
        return torch.ops.mla_mi355x.linear_act(x, weight, bias, residual, activation, False)[0]
    return _linear_act(x, weight, bias, residual, activation, False)[0]


# ----------------------------------------------------------------- gated feed-forward block

def _gated_ffn(x, w_gate, w_up, w_down, residual, activation, save):
    """``(y, h, saved or None)``; see :func:`gated_ffn`."""
    op = "mla_mi355x::gated_ffn"
    code = _activation(op, activation, gate=True)
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1] or x.dim() < 1 \
            or x.size(-1) != w_gate.size(1):
        raise ValueError(f"{op}: expected x [..., D], w_gate and w_up [H, D], w_down [D, H]; got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    H, D = w_gate.shape
    _check(op, x, (w_gate, w_up, w_down), ("w_gate", "w_up", "w_down"), residual, D)
    x2, x_stride = _rows(x, D)
    M = x2.size(0)
    y = x.new_empty(x.shape)
    h = x.new_empty((M, H))
    saved = x.new_empty(2 * _saved_size(M, H), dtype=torch.uint8) if save else None
    if M:
        (wg, sg), (wu, su) = _weight_rows(w_gate, D), _weight_rows(w_up, D)
        args = _lib.GatedLinearArgs(
            x2.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), None if saved is None else saved.data_ptr(), None, 0,
            M, H, D, x_stride, sg, su, H, code)
        ws = _fit_workspace("mla_gated_linear_workspace_bytes", args, h) if M > ROWS_MAX else None  # noqa: F841
        _launch("mla_gated_linear", args, h, op)
        _linear_run(op, h, H, w_down, None, residual, 0, None, y, M, D, H)
    return y, h, saved


@_op("gated_ffn", mutates_args=())
def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, residual: Optional[Tensor], activation: str,
              save: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """``y = residual + (act(x Wg^T) o (x Wu^T)) Wd^T`` for bf16 ``x [..., D]``, ``w_gate`` and ``w_up [H, D]``, ``w_down [D,
    H]`` (bf16, or fp32 read as bf16): silu(w1 x) * w3 x through w2 (transformer.py:117-125).  ``activation``: relu, silu,
    gelu_tanh.  The hidden layer is rounded to bf16 once, between the products.  Returns ``y`` and, with ``save``, the
    hidden layer and what the backward keeps of the two products (else empty tensors).  D and H multiples of 8."""
    y, h, saved = _gated_ffn(x, w_gate, w_up, w_down, residual, activation, save)
    return (y, h, saved) if save else (y, x.new_empty(0), x.new_empty(0, dtype=torch.uint8))


@gated_ffn.register_fake
def _(x, w_gate, w_up, w_down, residual, activation, save):
    H, D = w_gate.shape
    return (x.new_empty(x.shape), x.new_empty((x.numel() // D, H) if save else 0), _saved_fake(x, D, H, 2, save))


def _gated_grads(op, dy, sy, w_down, saved, dgu, code):
    """The gradients ``dgu [M, 2 H]`` of both first products from bf16 rows ``dy [M, D]`` of stride ``sy`` and what they saved."""
    (D, H), M = w_down.shape, dy.size(0)
    wd, sd = _weight_rows(w_down, H)
    as_it_lies = (D + 64) * sd < REACH
    cols = H if as_it_lies else _columns(D, H)
    for c in range(0, H, cols):
        n, w, s, kept, out = min(cols, H - c), wd, sd, saved, dgu
        if not as_it_lies:
            w, s = wd[:, c:c + n].contiguous(), n
        if n < H:  # (the blocks of the kept values that lie in these columns)
            out = dgu.new_empty((M, 2 * n))
            kept = saved.view((M + 31) // 32, (H + 31) // 32, -1)[:, c // 32:(c + n + 31) // 32].contiguous()
        args = _lib.GatedLinearBwdArgs(dy.data_ptr(), w.data_ptr(), kept.data_ptr(), out.data_ptr(), M, n, D, sy, s, 2 * n, code)
        _launch("mla_gated_linear_bwd", args, out, op)
        if n < H:
            dgu[:, c:c + n], dgu[:, H + c:H + c + n] = out[:, :n], out[:, n:]


def _gated_ffn_bwd(dy, x, w_gate, w_up, w_down, h, saved, activation, need_dx, need_gate, need_up, need_down):
    """``(dx, dw_gate, dw_up, dw_down)``, None where not needed; see :func:`gated_ffn_bwd`."""
    op = "mla_mi355x::gated_ffn_bwd"
    code = _activation(op, activation, gate=True)
    H, D = w_gate.shape if w_gate.dim() == 2 else (0, 0)
    M, dev = x.numel() // D if D else 0, x.get_device()
    fits = H > 0 and x.dim() > 0 and x.size(-1) == D and dy.shape == x.shape and w_up.shape == w_gate.shape \
        and w_down.shape == (D, H) and h.shape == (M, H) and saved.numel() == 2 * _saved_size(M, H)
    if not (fits and x.dtype == _BF16 and h.dtype == _BF16 and saved.dtype == torch.uint8 and h.is_contiguous()
            and saved.is_contiguous() and (w_gate.dtype == _BF16 or w_gate.dtype == _F32)
            and (w_up.dtype == _BF16 or w_up.dtype == _F32) and (w_down.dtype == _BF16 or w_down.dtype == _F32)
            and 0 <= dev == dy.get_device() == w_gate.get_device() == w_up.get_device() == w_down.get_device()
            == h.get_device() == saved.get_device()):
        _refuse_bwd(op, fits, x, dy, (w_gate, w_up, w_down), saved, h)
    (dy2, sy), (x2, sx) = _weight_rows(dy, D), _rows(x, D)
    dx = dwg = dwu = None
    dwd = _weight_grad(dy2, sy, h, H, w_down.dtype) if need_down else None
    if need_dx or need_gate or need_up:
        dgu = x.new_empty((M, 2 * H))
        if M:
            _gated_grads(op, dy2, sy, w_down, saved, dgu, code)
        if need_dx:
            dx = _linear_dx(op, dgu, 2 * H, (w_gate, w_up), x.shape)
        # one product, its rows the two gradients (which a weight gradient takes below 2^20 of)
        if need_gate and need_up and w_gate.dtype == w_up.dtype and 2 * H < 1 << 20:
            dwg, dwu = _weight_grad(dgu, 2 * H, x2, sx, w_gate.dtype).split(H)
        else:
            dwg = _weight_grad(dgu[:, :H], 2 * H, x2, sx, w_gate.dtype) if need_gate else None
            dwu = _weight_grad(dgu[:, H:], 2 * H, x2, sx, w_up.dtype) if need_up else None
    return dx, dwg, dwu, dwd


@_op("gated_ffn_bwd", mutates_args=())
def gated_ffn_bwd(dy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, h: Tensor, saved: Tensor,
                  activation: str, need_dx: bool, need_gate: bool, need_up: bool,
                  need_down: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients ``(dx, dw_gate, dw_up, dw_down)`` of :func:`gated_ffn` from ``dy`` and what it saved, the weights' in their
    dtypes.  Empty tensors where a gradient is not needed."""
    dx, dwg, dwu, dwd = _gated_ffn_bwd(dy, x, w_gate, w_up, w_down, h, saved, activation, need_dx, need_gate, need_up, need_down)
    if dwg is not None and dwu is not None and dwu.untyped_storage().data_ptr() == dwg.untyped_storage().data_ptr():
        dwu = dwu.clone()  # (an operator's outputs share no memory)
    return tuple(x.new_empty(0) if t is None else t for t in (dx, dwg, dwu, dwd))


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, h, saved, activation, need_dx, need_gate, need_up, need_down):
    return tuple(t.new_empty(t.shape) if n else x.new_empty(0)
                 for t, n in ((x, need_dx), (w_gate, need_gate), (w_up, need_up), (w_down, need_down)))


def _gated_ffn_grads(ctx, dy, need):
    """The gradients for (x, w_gate, w_up, w_down) from the saved tensors of either autograd path."""
    x, w_gate, w_up, w_down, h, saved = ctx.saved_tensors
    plain = _plain_backward(dy)
    if not saved.numel():  # not kept: the first half again (without rows: h's shape)
        _, h, saved = torch.ops.mla_mi355x.gated_ffn(x.detach(), w_gate.detach(), w_up.detach(), w_down.detach(), None,
                                                     ctx.activation, True)
    run = _gated_ffn_bwd if plain else torch.ops.mla_mi355x.gated_ffn_bwd
    got = run(dy, x, w_gate, w_up, w_down, h, saved, ctx.activation, *need[:4])
    return tuple(g if n else None for g, n in zip(got, need))


def _gated_ffn_setup(ctx, inputs, output):
    x, w_gate, w_up, w_down, residual, activation, _ = inputs
    ctx.save_for_backward(x, w_gate, w_up, w_down, output[1], output[2])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1], output[2])


def _gated_ffn_backward(ctx, dy, dh, dsaved):
    need = ctx.needs_input_grad
    grads = _gated_ffn_grads(ctx, dy, need) if any(need[:4]) else (None,) * 4
    return (*grads, dy if need[4] else None, None, None)


_register_autograd(gated_ffn, "gated_ffn", _gated_ffn_setup, _gated_ffn_backward)


class _GatedFfn(torch.autograd.Function):
    """The operator's body and formula without its dispatch."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, activation):
        save = any(ctx.needs_input_grad[:4])
        with kernels.below_autograd():
            y, h, saved = _gated_ffn(x, w_gate, w_up, w_down, residual, activation, save)
        if save:
            ctx.save_for_backward(x, w_gate, w_up, w_down, h, saved)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        grads = _gated_ffn_grads(ctx, dy, need) if any(need[:4]) else (None,) * 4
        return (*grads, dy if need[4] else None, None)


def gated(x, w_gate, w_up, w_down, residual, activation) -> Tensor:
    """:func:`gated_ffn`'s ``y`` for eager callers."""
    args = (x, w_gate, w_up, w_down, residual)
    if kernels._needs_grad(args):
        if kernels.function_fits(args):
            return _GatedFfn.apply(x, w_gate, w_up, w_down, residual, activation)
        return torch.ops.mla_mi355x.gated_ffn(x, w_gate, w_up, w_down, residual, activation, True)[0]
    if kernels._not_plain(args):
        return torch.ops.mla_mi355x.gated_ffn(x, w_gate, w_up, w_down, residual, activation, False)[0]
    return _gated_ffn(x, w_gate, w_up, w_down, residual, activation, False)[0]
