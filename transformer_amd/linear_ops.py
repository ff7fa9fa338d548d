"""The linear layers' operators (``torch.ops.mla_mi355x.linear_act``, ``gated_ffn`` and their backwards).

They are registered as those of ``kernels`` are; ``eager`` runs their bodies without the dispatcher where nothing needs it.
There is no CPU path: a CPU tensor, or a missing library, raises.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from .kernels import (_alloc_workspace, _bf16, _dt_code, _EagerOps, _op, _ptr, _register_autograd, _require_gpu, _stream,
                      batched_grad, weight_grad, weight_grad_or_none)

LINEAR_MAX_STRIDE = 1 << 22


def _launch(entry: str, args, like: Tensor, op: str) -> None:
    """Call a C entry point on ``like``'s device and its current stream, whichever device is the current one."""
    fn, dev = _lib.entry(entry), like.get_device()
    if dev == torch._C._cuda_getDevice():
        rc = fn(ctypes.byref(args), _stream(like))
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), _stream(like))
    _lib.check(rc, op)


def _fit_workspace(entry: str, args, like: Tensor) -> Optional[Tensor]:
    """The workspace that ``entry`` (a ``*_workspace_bytes`` function) asks for, set in ``args``; keep it until the call."""
    nbytes = int(_lib.entry(entry)(ctypes.byref(args)))
    if not nbytes:
        return None
    ws = _alloc_workspace(nbytes, like.device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _matrix(t: Tensor, K: int, one_row: bool = False) -> Tensor:
    """``t [..., K]`` as rows the linear kernels take: unit inner stride, 16-byte aligned, a row stride that is a multiple of
    8 and covers a row (``one_row``: or 0, the same row for all); copied where its layout is another."""
    t = t.reshape(-1, K)
    if t.size(0) <= 1:
        ok = t.stride(1) == 1 or K == 1
    else:
        s = t.stride(0)
        ok = t.stride(1) == 1 and s % 8 == 0 and s < LINEAR_MAX_STRIDE and (s >= K or (one_row and s == 0))
    if ok and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _row_stride(t: Tensor) -> int:
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _weight_bf16(w: Tensor) -> Tensor:
    return _matrix(w.detach().to(torch.bfloat16), w.size(1))


def _activation(op: str, name: str, gate: bool = False) -> int:
    code = _lib.ACTIVATIONS.get(name)
    if code is None or (gate and name == "none"):
        raise ValueError(f"{op}: activation {name!r} is not one of "
                         f"{[a for a in _lib.ACTIVATIONS if not (gate and a == 'none')]}")
    return code


def _linear_check(op: str, x: Tensor, weights, residual: Optional[Tensor], n_out: int) -> None:
    _require_gpu(op, x, residual, *weights.values())
    _bf16(op, x=x)
    for name, w in weights.items():
        if w.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{op}: {name} must be bfloat16 or float32, got {w.dtype}")
        if w.device != x.device:
            raise ValueError(f"{op}: {name} is on {w.device}, x on {x.device}")
        if w.dim() == 2 and (w.size(0) % 8 or w.size(1) % 8 or not w.numel()):
            raise ValueError(f"{op}: {name} {tuple(w.shape)}: both sizes must be positive multiples of 8")
    if residual is not None:
        _bf16(op, residual=residual)
        if residual.shape != (*x.shape[:-1], n_out) or residual.device != x.device:
            raise ValueError(f"{op}: residual must be {(*x.shape[:-1], n_out)} on {x.device}, got {tuple(residual.shape)} "
                             f"on {residual.device}")


def _saved_buffer(M: int, N: int, blocks: int, like: Tensor) -> Tensor:
    return torch.empty(blocks * int(_lib.entry("mla_linear_saved_size")(M, N)), dtype=torch.uint8, device=like.device)


def _linear_act_run(op, x2, w, bias, res2, code, saved, out):
    """``out = act(x2 w^T + bias) + res2`` on bf16 matrices as :func:`_matrix` leaves them."""
    (M, K), N = x2.shape, w.size(0)
    args = _lib.LinearActArgs(
        x=x2.data_ptr(), w=w.data_ptr(), bias=_ptr(bias), residual=_ptr(res2), y=out.data_ptr(), saved=_ptr(saved),
        workspace=None, workspace_bytes=0, M=M, N=N, K=K, x_stride=_row_stride(x2), w_stride=_row_stride(w),
        residual_stride=0 if res2 is None else _row_stride(res2), y_stride=N, activation=code)
    ws = _fit_workspace("mla_linear_act_workspace_bytes", args, out)  # noqa: F841  (kept until the launch)
    _launch("mla_linear_act", args, out, op)


@_op("linear_act", mutates_args=())
def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], activation: str,
               save: bool) -> Tuple[Tensor, Tensor]:
    """``y = act(x W^T + bias) + residual`` for bf16 ``x [..., K]``, ``weight [N, K]`` (bf16, or fp32 read as bf16), ``bias
    [N]``, ``residual [..., N]`` bf16: fp32 sums and epilogue, one rounding.  ``activation``: none, relu, silu, gelu_tanh.
    Returns ``y`` and, with ``save`` and an activation, what the backward keeps of the pre-activation (else an empty
    tensor).  K and N multiples of 8."""
    op = "mla_mi355x::linear_act"
    code = _activation(op, activation)
    if weight.dim() != 2 or x.dim() < 1 or x.size(-1) != weight.size(1) or (bias is not None
                                                                            and bias.shape != (weight.size(0),)):
        raise ValueError(f"{op}: expected x [..., K], weight [N, K], bias [N]; got {tuple(x.shape)}, {tuple(weight.shape)}, "
                         f"{None if bias is None else tuple(bias.shape)}")
    N, K = weight.shape
    _linear_check(op, x, {"weight": weight, **({} if bias is None else {"bias": bias})}, residual, N)
    x2 = _matrix(x, K)
    M = x2.size(0)
    y = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    saved = _saved_buffer(M if save and code else 0, N, 1, x)
    if M:
        b = None if bias is None else bias.detach().to(torch.bfloat16).contiguous()
        if b is not None and b.data_ptr() % 8:
            b = b.clone()
        _linear_act_run(op, x2, _weight_bf16(weight), b, None if residual is None else _matrix(residual, N, True), code,
                        saved if saved.numel() else None, y)
    return y.view(*x.shape[:-1], N), saved


def _saved_fake(x, K, N, blocks, wanted):
    M = x.numel() // K
    return x.new_empty(blocks * 3072 * ((M + 31) // 32) * ((N + 31) // 32) if wanted else 0, dtype=torch.uint8)


@linear_act.register_fake
def _(x, weight, bias, residual, activation, save):
    N, K = weight.shape
    return x.new_empty(*x.shape[:-1], N), _saved_fake(x, K, N, 1, save and activation != "none")


def _weight_grad_rows_any(dy: Tensor, x: Tensor, dtype: torch.dtype) -> Tensor:
    """``dy^T x`` in ``dtype`` for any number of rows: those beyond the kernel's 32-bit reach in several parts, added in fp32."""
    if dy.size(0) == 0:
        return torch.zeros(dy.size(1), x.size(1), dtype=dtype, device=dy.device)
    dw = weight_grad_or_none(dy, x, dtype == torch.float32)
    if dw is None:
        rows = (1 << 30) // max(_row_stride(dy), _row_stride(x)) - 257
        if rows < 32:
            raise ValueError(f"mla_mi355x::weight_grad: rows of {dy.size(1)} and {x.size(1)} are too wide")
        for r in range(0, dy.size(0), rows):
            part = weight_grad(dy[r:r + rows], x[r:r + rows], True)
            dw = part if dw is None else dw.add_(part)
    return dw.to(dtype)


def _linear_dx(op: str, dy: Tensor, weights, shape) -> Tensor:
    """``sum_p dy_p W_p`` for bf16 rows ``dy [M, P N]`` and P = 1 or 2 weights ``[N, K]``, as ``shape``."""
    w = [_weight_bf16(t) for t in weights]
    (N, K), M = w[0].shape, dy.size(0)
    dx = torch.empty(M, K, dtype=torch.bfloat16, device=dy.device)
    if M:
        args = _lib.LinearDxArgs(
            dy=dy.data_ptr(), w0=w[0].data_ptr(), w1=w[1].data_ptr() if len(w) > 1 else None, dx=dx.data_ptr(),
            workspace=None, workspace_bytes=0, M=M, N=N, K=K, dy_stride=_row_stride(dy), w0_stride=_row_stride(w[0]),
            w1_stride=_row_stride(w[1]) if len(w) > 1 else 0, dx_stride=K)
        ws = _fit_workspace("mla_linear_dx_workspace_bytes", args, dx)  # noqa: F841
        _launch("mla_linear_dx", args, dx, op)
    return dx.view(shape)


@_op("linear_act_bwd", mutates_args=())
def linear_act_bwd(dy: Tensor, x: Tensor, weight: Tensor, saved: Tensor, activation: str, need_dx: bool, need_dw: bool,
                   db_dtype: Optional[torch.dtype]) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients ``(dx, dw, db)`` of :func:`linear_act` from ``dy`` and what it saved; ``dw`` in the weight's dtype, ``db`` in
    ``db_dtype`` (None: no bias).  Empty tensors where a gradient is not needed."""
    op = "mla_mi355x::linear_act_bwd"
    code = _activation(op, activation)
    _require_gpu(op, dy, x, weight, saved)
    _bf16(op, x=x)
    N, K = weight.shape
    dy2, x2 = _matrix(dy.to(torch.bfloat16), N), _matrix(x, K)
    M = x2.size(0)
    if dy2.size(0) != M:
        raise ValueError(f"{op}: dy {tuple(dy.shape)} does not match x {tuple(x.shape)}")
    none = x.new_empty(0)
    dz, db = dy2, none
    if db_dtype is not None:
        db = torch.zeros(N, dtype=db_dtype, device=x.device) if M == 0 else torch.empty(N, dtype=db_dtype, device=x.device)
    if M and (code or db_dtype is not None):
        if code:
            if saved.numel() != int(_lib.entry("mla_linear_saved_size")(M, N)):
                raise ValueError(f"{op}: saved does not belong to x {tuple(x.shape)} and weight {tuple(weight.shape)}")
            dz = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
        args = _lib.ActGradArgs(
            dy=dy2.data_ptr(), saved=_ptr(saved) if code else None, dz=dz.data_ptr() if code else None,
            db=db.data_ptr() if db_dtype is not None else None, workspace=None, workspace_bytes=0, M=M, N=N,
            dy_stride=_row_stride(dy2), dz_stride=N, activation=code, db_dtype=_dt_code(db))
        ws = _fit_workspace("mla_act_grad_workspace_bytes", args, dy2)  # noqa: F841
        _launch("mla_act_grad", args, dy2, op)
    dx = _linear_dx(op, dz, (weight,), x.shape) if need_dx else none
    dw = _weight_grad_rows_any(dz, x2, weight.dtype) if need_dw else none
    return dx, dw, db


@linear_act_bwd.register_fake
def _(dy, x, weight, saved, activation, need_dx, need_dw, db_dtype):
    return (x.new_empty(x.shape if need_dx else 0), weight.new_empty(weight.shape if need_dw else 0),
            x.new_empty(0) if db_dtype is None else x.new_empty(weight.size(0), dtype=db_dtype))


def _linear_act_setup(ctx, inputs, output):
    x, weight, bias, residual, activation, _ = inputs
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1])


def _linear_act_backward(ctx, dy, dsaved):
    x, weight, bias, saved = ctx.saved_tensors
    need = ctx.needs_input_grad
    ops = _ops_for(dy)
    dx = dw = db = None
    if any(need[:3]):
        if ctx.activation != "none" and not saved.numel() and x.numel():  # not kept: the product again
            saved = ops.linear_act(x, weight, bias, None, ctx.activation, True)[1]
        dx, dw, db = ops.linear_act_bwd(dy, x, weight, saved, ctx.activation, need[0], need[1],
                                        bias.dtype if bias is not None and need[2] else None)
    return (dx if need[0] else None, dw if need[1] else None, db if bias is not None and need[2] else None,
            dy if need[3] else None, None, None)


_register_autograd(linear_act, "linear_act", _linear_act_setup, _linear_act_backward)


# ----------------------------------------------------------------- gated feed-forward block

@_op("gated_ffn", mutates_args=())
def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, residual: Optional[Tensor], activation: str,
              save: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """``y = residual + (act(x Wg^T) o (x Wu^T)) Wd^T`` for bf16 ``x [..., D]``, ``w_gate`` and ``w_up [H, D]``, ``w_down [D,
    H]`` (bf16, or fp32 read as bf16): silu(w1 x) * w3 x through w2 (transformer.py:117-125).  ``activation``: relu, silu,
    gelu_tanh.  The hidden layer is rounded to bf16 once, between the products.  Returns ``y`` and, with ``save``, the
    hidden layer and what the backward keeps of the two products (else empty tensors).  D and H multiples of 8."""
    op = "mla_mi355x::gated_ffn"
    code = _activation(op, activation, gate=True)
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1] or x.dim() < 1 \
            or x.size(-1) != w_gate.size(1):
        raise ValueError(f"{op}: expected x [..., D], w_gate and w_up [H, D], w_down [D, H]; got {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    H, D = w_gate.shape
    _linear_check(op, x, {"w_gate": w_gate, "w_up": w_up, "w_down": w_down}, residual, D)
    x2 = _matrix(x, D)
    M = x2.size(0)
    y = torch.empty(M, D, dtype=torch.bfloat16, device=x.device)
    h = torch.empty(M, H, dtype=torch.bfloat16, device=x.device)
    saved = _saved_buffer(M if save else 0, H, 2, x)
    if M:
        wg, wu = _weight_bf16(w_gate), _weight_bf16(w_up)
        args = _lib.GatedLinearArgs(
            x=x2.data_ptr(), w_gate=wg.data_ptr(), w_up=wu.data_ptr(), h=h.data_ptr(),
            saved=saved.data_ptr() if save else None, workspace=None, workspace_bytes=0, M=M, N=H, K=D,
            x_stride=_row_stride(x2), w_gate_stride=_row_stride(wg), w_up_stride=_row_stride(wu), h_stride=H, activation=code)
        ws = _fit_workspace("mla_gated_linear_workspace_bytes", args, h)  # noqa: F841
        _launch("mla_gated_linear", args, h, op)
        _linear_act_run(op, h, _weight_bf16(w_down), None, None if residual is None else _matrix(residual, D, True), 0, None, y)
    return y.view(x.shape), h if save else h.new_empty(0), saved


@gated_ffn.register_fake
def _(x, w_gate, w_up, w_down, residual, activation, save):
    H, D = w_gate.shape
    return (x.new_empty(x.shape), x.new_empty((x.numel() // D, H) if save else 0), _saved_fake(x, D, H, 2, save))


@_op("gated_ffn_bwd", mutates_args=())
def gated_ffn_bwd(dy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, h: Tensor, saved: Tensor,
                  activation: str, need_dx: bool, need_gate: bool, need_up: bool,
                  need_down: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients ``(dx, dw_gate, dw_up, dw_down)`` of :func:`gated_ffn` from ``dy`` and what it saved, the weights' in their
    dtypes.  Empty tensors where a gradient is not needed."""
    op = "mla_mi355x::gated_ffn_bwd"
    code = _activation(op, activation, gate=True)
    _require_gpu(op, dy, x, w_gate, w_up, w_down, h, saved)
    _bf16(op, x=x, h=h)
    H, D = w_gate.shape
    dy2, x2 = _matrix(dy.to(torch.bfloat16), D), _matrix(x, D)
    M = x2.size(0)
    if dy2.size(0) != M or tuple(h.shape) != (M, H) or not h.is_contiguous() \
            or saved.numel() != 2 * int(_lib.entry("mla_linear_saved_size")(M, H)):
        raise ValueError(f"{op}: dy {tuple(dy.shape)}, h {tuple(h.shape)} and saved do not belong to x {tuple(x.shape)}")
    none = x.new_empty(0)
    dx, dwg, dwu, dwd = none, none, none, none
    if need_down:
        dwd = _weight_grad_rows_any(dy2, h, w_down.dtype)
    if need_dx or need_gate or need_up:
        dgu = torch.empty(M, 2 * H, dtype=torch.bfloat16, device=x.device)
        if M:
            wd = _weight_bf16(w_down)
            args = _lib.GatedLinearBwdArgs(
                dy=dy2.data_ptr(), w_down=wd.data_ptr(), saved=saved.data_ptr(), dgu=dgu.data_ptr(), M=M, N=H, K=D,
                dy_stride=_row_stride(dy2), w_stride=_row_stride(wd), dgu_stride=2 * H, activation=code)
            _launch("mla_gated_linear_bwd", args, dgu, op)
        if need_dx:
            dx = _linear_dx(op, dgu, (w_gate, w_up), x.shape)
        if need_gate and need_up and w_gate.dtype == w_up.dtype:  # one product, its rows the two gradients
            dwg, dwu = _weight_grad_rows_any(dgu, x2, w_gate.dtype).split(H)
            dwu = dwu.clone()  # (an operator's outputs share no memory)
        else:
            dwg = _weight_grad_rows_any(dgu[:, :H], x2, w_gate.dtype) if need_gate else none
            dwu = _weight_grad_rows_any(dgu[:, H:], x2, w_up.dtype) if need_up else none
    return dx, dwg, dwu, dwd


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, h, saved, activation, need_dx, need_gate, need_up, need_down):
    return (x.new_empty(x.shape if need_dx else 0), w_gate.new_empty(w_gate.shape if need_gate else 0),
            w_up.new_empty(w_up.shape if need_up else 0), w_down.new_empty(w_down.shape if need_down else 0))


def _gated_ffn_setup(ctx, inputs, output):
    x, w_gate, w_up, w_down, residual, activation, _ = inputs
    ctx.save_for_backward(x, w_gate, w_up, w_down, output[1], output[2])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1], output[2])


def _gated_ffn_backward(ctx, dy, dh, dsaved):
    x, w_gate, w_up, w_down, h, saved = ctx.saved_tensors
    need = ctx.needs_input_grad
    ops = _ops_for(dy)
    grads = [None] * 4
    if any(need[:4]):
        if not saved.numel() and x.numel():  # not kept: the first half again
            _, h, saved = ops.gated_ffn(x, w_gate, w_up, w_down, None, ctx.activation, True)
        grads = ops.gated_ffn_bwd(dy, x, w_gate, w_up, w_down, h, saved, ctx.activation, *need[:4])
    return (*(g if n else None for g, n in zip(grads, need)), dy if need[4] else None, None, None)


_register_autograd(gated_ffn, "gated_ffn", _gated_ffn_setup, _gated_ffn_backward)


eager = _EagerOps(("linear_act", "linear_act_bwd", "gated_ffn", "gated_ffn_bwd"))


def _ops_for(grad: Tensor):
    """The operators that a backward formula runs on ``grad``."""
    return torch.ops.mla_mi355x if batched_grad(grad) else eager
