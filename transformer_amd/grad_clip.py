"""The norm of a training step's gradients and their clipping on the MI355X, with no host synchronisation.

``clip_grad_norm_(parameters, max_norm)`` is a drop-in for ``torch.nn.utils.clip_grad_norm_`` as the reference's step calls it
(train.py:454): two passes over all gradients, a HIP launch each for up to 128 tensors.  ``grad_norm(tensors)`` is the first
pass alone.
"""
from __future__ import annotations

import math
from array import array
from typing import Iterable, List, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from .linear_ops import _fit_workspace, _launch

_CODES = {torch.float32: _lib.MLA_DTYPE_F32, torch.bfloat16: _lib.MLA_DTYPE_BF16}


def _dense(t: Tensor) -> bool:
    """Whether ``t``'s elements fill its memory without gaps, in any order of the dimensions."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _shares(t: Tensor) -> bool:
    """Whether elements of ``t`` may share memory (a stride shorter than what lies below it)."""
    reach = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride < reach:
            return t.numel() > 0
        reach += stride * (size - 1)
    return False


def _layout(t: Tensor) -> Tuple[int, tuple]:
    """Where ``t``'s bytes lie: their first address, and (stride, count) of each dimension in bytes, the longest first and
    the last one a run."""
    dims = [(1, t.element_size())]
    for stride, size in sorted((s * t.element_size(), n) for s, n in zip(t.stride(), t.shape) if n != 1):
        below, count = dims[-1]
        if stride == below * count:
            dims[-1] = below, count * size
        else:
            dims.append((stride, size))
    return t.data_ptr(), tuple(reversed(dims))


def _reach(dims: tuple) -> int:
    return 1 + sum(s * (n - 1) for s, n in dims)


def _meet(a: int, da: tuple, b: int, db: tuple) -> bool:
    """Whether two layouts of :func:`_layout` share a byte."""
    if a + _reach(da) <= b or b + _reach(db) <= a:
        return False
    if len(da) == len(db) == 1:
        return True
    if da[0][0] < db[0][0]:
        a, da, b, db = b, db, a, da
    (s, n), inner = da[0], da[1:]
    if s == db[0][0]:  # rows of one stride: which of them meet goes by their distance alone
        first, other, within = 1 - db[0][1], db[1:], _reach(db[1:])
    else:              # the rows of the one with the longer stride, against all of the other
        first, other, within = 0, db, _reach(db)
    lo, hi = max(first, (b - a - _reach(inner)) // s + 1), min(n - 1, (b - a + within - 1) // s)
    return any(_meet(a + i * s, inner, b, other) for i in range(lo, hi + 1))


def _refuse_shared(op: str, grads: List[Tensor]) -> None:
    """An error where an element of ``grads`` lies in the memory of another one."""
    for g in grads:
        if _shares(g):
            raise ValueError(f"{op}: a gradient with strides {g.stride()} shares memory between its elements")
    near: List[Tuple[int, tuple]] = []  # those that reach past the start of the next one
    for at, dims in sorted(_layout(g) for g in grads if g.numel()):
        near = [o for o in near if o[0] + _reach(o[1]) > at]
        if any(_meet(*o, at, dims) for o in near):
            raise ValueError(f"{op}: two gradients share memory")
        near.append((at, dims))


def _is_max(op: str, norm_type: float) -> bool:
    """Whether the norm is the largest magnitude (else the 2-norm)."""
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"{op}: norm_type {norm_type} is not built (2 or inf)")
    return norm_type == math.inf


def _refuse(op: str, tensors: List[Tensor]) -> None:
    """The error of a list that the kernels do not take."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"transformer_amd.{op} is no registered operator: torch.jit.trace would not record its launches")
    for t in tensors:
        if t.layout != torch.strided:
            raise ValueError(f"{op}: sparse gradients are not built")
        if not t.is_cuda:
            raise RuntimeError(f"transformer_amd.{op} runs on a ROCm GPU only (no CPU path); got a tensor on {t.device}")
        if t.dtype not in _CODES:
            raise TypeError(f"{op}: gradients must be float32 or bfloat16, got {t.dtype}")
    raise ValueError(f"{op}: gradients on {sorted({str(t.device) for t in tensors})}: one device is needed")


def _laid_out(op: str, tensors: List[Tensor]) -> Tuple[List[Tensor], array]:
    """``tensors`` without gaps in memory (those with gaps copied) and their types.  (Few look-ups a tensor: they are the host's
    cost.)"""
    try:
        devices, whole = {t.get_device() for t in tensors}, [t.is_contiguous() for t in tensors]
        codes = array("i", [_CODES[t.dtype] for t in tensors])
    except (RuntimeError, KeyError):  # (of a compressed sparse tensor is_contiguous raises)
        _refuse(op, tensors)
    if len(devices) != 1 or -1 in devices or torch._C._get_tracing_state() is not None:
        _refuse(op, tensors)
    if not all(whole):
        if not all(t.layout == torch.strided for t in tensors):
            _refuse(op, tensors)
        tensors = [t if w or _dense(t) else t.detach().contiguous() for t, w in zip(tensors, whole)]
    return tensors, codes


def _run(op: str, entry: str, tensors: List[Tensor], codes: array, is_max: bool, max_norm: float) -> Tensor:
    n, like = len(tensors), tensors[0]
    norm = torch.empty((), dtype=torch.float32, device=like.device)
    # host tables, read before the entry point returns
    ptrs, numels = array("Q", [t.data_ptr() for t in tensors]), array("q", [t.numel() for t in tensors])
    args = _lib.GradNormArgs(ptrs.buffer_info()[0], numels.buffer_info()[0], codes.buffer_info()[0], n, norm.data_ptr(), None, 0,
                             max_norm, int(is_max))
    ws = _fit_workspace("mla_grad_norm_workspace_bytes", args, like)  # noqa: F841  (kept until the launch)
    _launch(entry, args, like, op)
    return norm


def grad_norm(tensors: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0) -> Tensor:
    """The norm (2, or inf: the largest magnitude) of all elements of ``tensors`` together, an fp32 scalar on their device.
    Tensors are fp32 or bf16, of any layout, on one device; squares are summed in fp64.  A NaN anywhere gives NaN."""
    tensors = [tensors] if isinstance(tensors, Tensor) else list(tensors)
    is_max = _is_max("grad_norm", norm_type)
    if not tensors:
        return torch.tensor(0.0)
    return _run("grad_norm", "mla_grad_norm", *_laid_out("grad_norm", tensors), is_max, 0.0)


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool = None) -> Tensor:
    """Scales the gradients of ``parameters`` in place by ``min(1, max_norm / (norm + 1e-6))`` and returns their norm before
    that, as ``torch.nn.utils.clip_grad_norm_`` does; parameters without a gradient are passed over.  ``norm_type``: 2 or inf.
    ``error_if_nonfinite`` waits for the norm (one more pass over the gradients) and raises before anything is scaled.
    ``foreach`` is accepted and ignored.  Gradients are fp32 or bf16 on one device, of any layout; two that share memory are
    refused, and so is torch.jit.trace, which would not record the launches."""
    op = "clip_grad_norm_"
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{op}: max_norm must be at least 0, got {max_norm}")
    is_max = _is_max(op, norm_type)
    parameters = [parameters] if isinstance(parameters, Tensor) else parameters
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.tensor(0.0)
    flat, codes = _laid_out(op, grads)
    if flat is not grads and any(g is not c for g, c in zip(grads, flat)):  # (the entry point would compare the copies)
        _refuse_shared(op, grads)
    if error_if_nonfinite:
        norm = _run(op, "mla_grad_norm", flat, codes, is_max, 0.0)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it "
                               "cannot be clipped.")
    norm = _run(op, "mla_grad_clip", flat, codes, is_max, max_norm)
    if flat is not grads:
        with torch.no_grad():
            for g, c in zip(grads, flat):
                if g is not c:
                    g.copy_(c)
    torch.autograd.graph.increment_version(grads)
    return norm
