"""The feed-forward half of a block on the MI355X: linear layers with their epilogue, and the gated block.

``linear_act(x, weight, bias, residual, activation)`` is ``act(x W^T + b) + residual`` in one HIP kernel, and
``gated_ffn(x, w_gate, w_up, w_down, residual, activation)`` the reference's ``w2(silu(w1 x) * w3 x)`` (transformer.py:117-125)
in two: both first products with the activation and the product of the two, then the second one with the block's residual sum
(transformer.py:351).  Both have backward passes of their own.  ``SwiGLU(dim, hidden)`` is the block as a module, with the
reference's state-dict keys ``w1.weight``, ``w2.weight``, ``w3.weight``.

Arithmetic is bf16 with fp32 sums: inputs are bf16, or anything that bf16 autocast casts; weights may be fp32 (read as bf16,
their gradients fp32).  The gradients of ``w_gate`` and ``w_up`` are the halves of one allocation.  Under autocast a residual
stream in fp32 stays fp32: the sum with it is then torch's.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from . import linear_ops, training


def _inputs(op: str, x: Tensor, residual):
    """(x as bf16, the residual that the kernel adds, the one that torch adds to its result)."""
    if not x.is_cuda:
        raise RuntimeError(f"transformer_amd.{op} runs on a ROCm GPU only (no CPU path)")
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16 \
            and x.dtype in training._AUTOCAST_INPUTS:
        x = x.to(torch.bfloat16)
        if residual is not None and residual.dtype != torch.bfloat16:
            return x, None, residual
    elif x.dtype != torch.bfloat16:
        raise TypeError(f"{op}: x must be bfloat16 (or be cast by bf16 autocast), got {x.dtype}")
    return x, residual, None


def _add(op: str, residual, y: Tensor) -> Tensor:
    """``residual + y`` by torch, for residuals that the kernels take: of the result's shape."""
    if residual is None:
        return y
    if residual.shape != y.shape:
        raise ValueError(f"{op}: residual must be {tuple(y.shape)}, got {tuple(residual.shape)}")
    return residual + y


def linear_act(x: Tensor, weight: Tensor, bias: Tensor = None, residual: Tensor = None, activation: str = "none") -> Tensor:
    """``act(x W^T + bias) + residual`` for ``x [..., K]``, ``weight [N, K]``, ``bias [N]`` (bf16 or fp32, added as it is) and
    ``residual [..., N]``, K and N multiples of 8; ``activation``: "none", "relu", "silu" or "gelu_tanh".  fp32 sums and
    epilogue, one rounding to bf16."""
    x, res, after = _inputs("linear_act", x, residual)
    return _add("linear_act", after, linear_ops.linear(x, weight, bias, res, activation))


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, residual: Tensor = None,
              activation: str = "silu") -> Tensor:
    """``residual + (act(x Wg^T) * (x Wu^T)) Wd^T`` for ``x [..., D]``, ``w_gate`` and ``w_up [H, D]``, ``w_down [D, H]`` and
    ``residual [..., D]``, D and H multiples of 8; ``activation``: "relu", "silu" or "gelu_tanh".  fp32 sums; the hidden layer
    and the result are rounded to bf16 once each.  With gradients the block keeps the hidden layer (bf16) and both first
    products (24 bits each): 8 bytes per hidden value."""
    x, res, after = _inputs("gated_ffn", x, residual)
    return _add("gated_ffn", after, linear_ops.gated(x, w_gate, w_up, w_down, res, activation))


class SwiGLU(nn.Module):
    """``w2(silu(w1 x) * w3 x)`` (transformer.py:117-125); ``forward(x, residual)`` adds the block's residual stream in the
    second product's epilogue.  What the kernels do not take runs through the layers as they are, in torch: layers that are not
    plain ``nn.Linear`` (hooks, adapters, a parametrization), other arithmetic than bf16 (fp32 or fp16 without bf16 autocast,
    fp16 autocast), sizes that are not multiples of 8, a layer replaced by one of another shape."""

    def __init__(self, dim: int, hidden: int):
        super().__init__()
        self.w1 = nn.Linear(dim, hidden, bias=False)
        self.w2 = nn.Linear(hidden, dim, bias=False)
        self.w3 = nn.Linear(dim, hidden, bias=False)

    def _fits(self, x: Tensor) -> bool:
        """Whether the kernels take the layers and ``x``."""
        if not all(training.plain_linear(m) for m in (self.w1, self.w2, self.w3)):
            return False
        if torch.is_autocast_enabled("cuda"):
            ok = torch.get_autocast_dtype("cuda") == torch.bfloat16 and x.dtype in training._AUTOCAST_INPUTS
        else:
            ok = x.dtype == torch.bfloat16
        w1, w2, w3 = self.w1.weight, self.w2.weight, self.w3.weight
        return ok and w1.shape == w3.shape == w2.shape[::-1] and w1.size(0) % 8 == 0 and w1.size(1) % 8 == 0 and w1.numel() > 0 \
            and all(w.dtype in (torch.bfloat16, torch.float32) for w in (w1, w2, w3))

    def forward(self, x: Tensor, residual: Tensor = None) -> Tensor:
        if not x.is_cuda:
            raise RuntimeError("transformer_amd.SwiGLU runs on a ROCm GPU only (no CPU path)")
        if self._fits(x):
            return gated_ffn(x, self.w1.weight, self.w3.weight, self.w2.weight, residual)
        return _add("SwiGLU", residual, self.w2(F.silu(self.w1(x)) * self.w3(x)))
