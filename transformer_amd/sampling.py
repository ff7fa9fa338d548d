"""Drawing the next tokens on the GPU: temperature, top-k, top-p, min-p and a draw from given random numbers.

The reference's generation loop samples one row and synchronises with the host for it (CLI.py:139-187).  ``sample_tokens`` draws a
token for each row of a batch in one kernel, each row with settings of its own where they are tensors, and leaves the tokens on the
GPU.  The random numbers are an input: the same ones give the same tokens.  There is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import kernels
from .host_calls import Entry, plain
from .kernels import _op

_entry = Entry("mla_sample", "8P3q3f2i4x", "SampleArgs")
MAX_VOCAB = 1 << 19
_SETTINGS = ("temperature", "top_k", "top_p", "min_p")


@_op("sample_tokens", mutates_args=())
def _sample(logits: Tensor, u: Tensor, temperature: float, top_k: int, top_p: float, min_p: float,
            temperature_rows: Optional[Tensor], top_k_rows: Optional[Tensor], top_p_rows: Optional[Tensor],
            min_p_rows: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    op = "mla_mi355x::sample_tokens"
    for t in (logits, u, temperature_rows, top_k_rows, top_p_rows, min_p_rows):
        if t is not None and (logits.get_device() < 0 or t.get_device() != logits.get_device()):
            kernels._require_gpu(op, t)
            raise ValueError(f"{op}: all tensors must be on one device, got {t.device} and {logits.device}")
    return _draw(logits, u, temperature, top_k, top_p, min_p, temperature_rows, top_k_rows, top_p_rows, min_p_rows)


def _draw(logits, u, temperature, top_k, top_p, min_p, temperature_rows, top_k_rows, top_p_rows, min_p_rows):
    op = "mla_mi355x::sample_tokens"
    if logits.dim() != 2 or u.dim() != 1 or not 1 <= logits.size(1) <= MAX_VOCAB or u.size(0) != logits.size(0):
        raise ValueError(f"{op}: expected logits [B, V], V up to {MAX_VOCAB}, and u [B]; got {tuple(logits.shape)}, {tuple(u.shape)}")
    bf16 = logits.dtype is torch.bfloat16
    if not (bf16 or logits.dtype is torch.float32) or u.dtype is not torch.float32:
        raise TypeError(f"{op}: logits must be bfloat16 or float32 and u float32, got {logits.dtype}, {u.dtype}")
    (B, V), dev = logits.shape, logits.get_device()
    rows, at = [temperature_rows, top_k_rows, top_p_rows, min_p_rows], [0, 0, 0, 0]
    for k, t in enumerate(rows):
        if t is None:
            continue
        if t.dtype is not (torch.int32 if k == 1 else torch.float32) or t.dim() != 1 or t.size(0) != B:
            raise ValueError(f"{op}: {_SETTINGS[k]} of rows must be {'int32' if k == 1 else 'float32'} [{B}], got {t.dtype} {tuple(t.shape)}")
        if not t.is_contiguous():
            rows[k] = t = t.contiguous()
        at[k] = t.data_ptr()
    stride, inner = logits.stride()
    if (inner != 1 and V > 1) or stride < 0:
        logits = logits.contiguous()
        stride = V
    u = u if u.is_contiguous() else u.contiguous()
    tokens = logits.new_empty(B, dtype=torch.int64)
    logprobs = u.new_empty(B)
    if B:
        _entry(op, dev, logits.data_ptr(), u.data_ptr(), *at, tokens.data_ptr(), logprobs.data_ptr(), B, V, stride, temperature, top_p,
               min_p, top_k, 0 if bf16 else 1)  # MLA_DTYPE_*
    return tokens, logprobs


@_sample.register_fake
def _(logits, u, temperature, top_k, top_p, min_p, temperature_rows, top_k_rows, top_p_rows, min_p_rows):
    B = logits.size(0)
    return logits.new_empty(B, dtype=torch.int64), logits.new_empty(B, dtype=torch.float32)


_ops = torch.ops.mla_mi355x


def sample_tokens(logits: Tensor, u: Tensor, temperature: Union[float, Tensor] = 1.0, top_k: Union[int, Tensor] = 0,
                  top_p: Union[float, Tensor] = 1.0, min_p: Union[float, Tensor] = 0.0) -> Tuple[Tensor, Tensor]:
    """``(tokens int64 [B], logprobs fp32 [B])`` drawn from ``logits [B, V]`` (bf16 or fp32; B below 2^22, V up to 2^19) with ``u [B]``
    fp32 in [0, 1).

    Weights are ``exp((x - max x) / temperature)``.  Of these are kept the ``top_k`` largest (0 or less: all), of those the shortest
    run, largest first, that holds ``top_p`` of their weight (1 or more: all), of those the ones of at least ``min_p`` of the
    largest.  The token is the first, in the order of the vocabulary, at which the kept weights add up to more than ``u`` of their
    sum; its logprob is that of the distribution drawn from.  Of equal logits the lower index counts as the larger.  Temperature 0 (or
    less) takes the largest, an infinite one weighs all finite logits alike.  A NaN counts as -inf; a row without a logit above -inf
    gives token -1 and logprob -inf.  Each setting is a number or a tensor ``[B]`` on the device (fp32; ``top_k`` int32)."""
    rows = [None, None, None, None]
    if isinstance(temperature, Tensor):
        rows[0], temperature = temperature, 1.0
    if isinstance(top_k, Tensor):
        rows[1], top_k = top_k, 0
    if isinstance(top_p, Tensor):
        rows[2], top_p = top_p, 1.0
    if isinstance(min_p, Tensor):
        rows[3], min_p = min_p, 0.0
    if type(top_k) is not int or not -(1 << 31) <= top_k < 1 << 31:
        raise ValueError(f"sample_tokens: top_k must be a whole number of 32 bits, got {top_k!r}")
    for name, v in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)):
        if type(v) is bool or v != v:
            raise ValueError(f"sample_tokens: {name} must be a number, got {v!r}")
    run = _draw if plain(logits, u, *rows) else _ops.sample_tokens
    return run(logits, u, float(temperature), top_k, float(top_p), float(min_p), *rows)
