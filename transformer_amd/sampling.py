"""Drawing the next tokens on the GPU: temperature, top-k, top-p, min-p and a draw from given random numbers.

The reference's generation loop samples one row and synchronises with the host for it (CLI.py:139-187).  ``sample_tokens`` draws a
token for each row of a batch in one kernel, each row with settings of its own where they are tensors, and leaves the tokens on the
GPU.  The random numbers are an input: the same ones give the same tokens.  There is no CPU path.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib, kernels
from .kernels import _eager_call, _op
from .linear_ops import _launch

MAX_VOCAB = 1 << 19
_SETTINGS = ("temperature", "top_k", "top_p", "min_p")


@_op("sample_tokens", mutates_args=())
def _sample(logits: Tensor, u: Tensor, temperature: float, top_k: int, top_p: float, min_p: float,
            temperature_rows: Optional[Tensor], top_k_rows: Optional[Tensor], top_p_rows: Optional[Tensor],
            min_p_rows: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    op = "mla_mi355x::sample_tokens"
    rows = (temperature_rows, top_k_rows, top_p_rows, min_p_rows)
    if logits.dim() != 2 or not 1 <= logits.size(1) <= MAX_VOCAB or u.shape != logits.shape[:1]:
        raise ValueError(f"{op}: expected logits [B, V], V up to {MAX_VOCAB}, and u [B]; got {tuple(logits.shape)}, {tuple(u.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float32) or u.dtype != torch.float32:
        raise TypeError(f"{op}: logits must be bfloat16 or float32 and u float32, got {logits.dtype}, {u.dtype}")
    B, V = logits.shape
    for name, t in zip(_SETTINGS, rows):
        want = torch.int32 if name == "top_k" else torch.float32
        if t is not None and (t.dtype != want or t.shape != (B,)):
            raise ValueError(f"{op}: {name} of rows must be {want} [{B}], got {t.dtype} {tuple(t.shape)}")
    dev = logits.get_device()
    for t in (logits, u, *rows):
        if t is not None and (not t.is_cuda or t.get_device() != dev):
            kernels._require_gpu(op, t)
            raise ValueError(f"{op}: all tensors must be on one device, got {t.device} and {logits.device}")
    if logits.stride(1) != 1 and V > 1 or logits.stride(0) < 0:
        logits = logits.contiguous()
    u, *rows = [None if t is None else t.contiguous() for t in (u, *rows)]
    tokens = torch.empty(B, dtype=torch.int64, device=logits.device)
    logprobs = torch.empty(B, dtype=torch.float32, device=logits.device)
    if B:
        args = _lib.SampleArgs(logits.data_ptr(), u.data_ptr(), *(None if t is None else t.data_ptr() for t in rows),
                               tokens.data_ptr(), logprobs.data_ptr(), B, V, logits.stride(0), temperature, top_p, min_p, top_k,
                               kernels._dt_code(logits))
        _launch("mla_sample", args, logits, op)
    return tokens, logprobs


@_sample.register_fake
def _(logits, u, temperature, top_k, top_p, min_p, temperature_rows, top_k_rows, top_p_rows, min_p_rows):
    B = logits.size(0)
    return logits.new_empty(B, dtype=torch.int64), logits.new_empty(B, dtype=torch.float32)


_call = _eager_call("sample_tokens")


def sample_tokens(logits: Tensor, u: Tensor, temperature: Union[float, Tensor] = 1.0, top_k: Union[int, Tensor] = 0,
                  top_p: Union[float, Tensor] = 1.0, min_p: Union[float, Tensor] = 0.0) -> Tuple[Tensor, Tensor]:
    """``(tokens int64 [B], logprobs fp32 [B])`` drawn from ``logits [B, V]`` (bf16 or fp32) with ``u [B]`` fp32 in [0, 1).

    Weights are ``exp((x - max x) / temperature)``.  Of these are kept the ``top_k`` largest (0 or less: all), of those the shortest
    run, largest first, that holds ``top_p`` of their weight (1 or more: all), of those the ones of at least ``min_p`` of the
    largest.  The token is the first, in the order of the vocabulary, at which the kept weights add up to more than ``u`` of their
    sum; its logprob is that of the distribution drawn from.  Of equal logits the lower index counts as the larger.  Temperature 0
    (or less) takes the largest.  A NaN counts as -inf; a row without a logit above -inf gives token -1 and logprob -inf.  Each
    setting is a number or a tensor ``[B]`` on the device (fp32; ``top_k`` int32)."""
    one = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    given, rows = dict(zip(_SETTINGS, (temperature, top_k, top_p, min_p))), {}
    for name, v in given.items():
        if isinstance(v, Tensor):
            rows[name], given[name] = v, one[name]
        elif isinstance(v, bool) or (name == "top_k" and not isinstance(v, int)) or math.isnan(v):
            raise ValueError(f"sample_tokens: {name} must be {'a whole number' if name == 'top_k' else 'a number'}, got {v!r}")
    if not -(1 << 31) <= given["top_k"] < 1 << 31:
        raise ValueError(f"sample_tokens: top_k {given['top_k']} is out of range")
    return _call(logits, u, float(given["temperature"]), given["top_k"], float(given["top_p"]), float(given["min_p"]),
                 rows.get("temperature"), rows.get("top_k"), rows.get("top_p"), rows.get("min_p"))
