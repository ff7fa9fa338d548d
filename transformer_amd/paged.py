"""A latent cache in pages, in 16 or 4 bits: serving many sequences of any length on the MI355X.

The reference keeps one tensor a batch of equally long sequences (transformer.py:215-218, :241-244).  Here the rows of all
sequences lie in pages of ``size`` tokens, and a block table says which pages a sequence has:

* ``new_paged_cache(n_pages, size, d_latent, n_k_rope_heads, bits)`` makes one layer's ``(pages, scales)``.  A token's row is
  ``[latent | rotated keys]``, W = d_latent + 64 Hr values.  16 bits: ``pages`` bf16 ``[n, size, W]``, ``scales`` None.  4 bits:
  ``pages`` uint8 ``[n, size, W / 2]`` (value 2 i in the low half of byte i), ``scales`` bf16 ``[n, W / 64, size]``; a run of 64
  values (a rotated key is one) stands for ``(code - 8) scale``, ``scale = bf16(max |x| / 7)``: off by at most half a scale.
* ``paged_append`` rotates new tokens' queries and keys and writes the keys and latents into their pages;
* ``paged_decode`` is the absorbed attention of one query token a sequence over its pages;
* ``paged_read`` takes a range of each sequence back out, as the attention of a prompt's next chunk wants it.

``block_table`` is int32 ``[B, P]`` (an entry outside the cache, such as -1, is no page), lengths and starts int32 ``[B]``, all on
the device and read there: a recorded HIP graph follows them.  Sequences may share pages that none of them appends to.  Nothing
here has a gradient.  There is no CPU path: a CPU tensor, or a missing library, raises.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib, kernels
from ._lib import Strides
from .kernels import ROPE_DIM, SUPPORTED_LATENT, _aligned4, _eager_call, _op
from .linear_ops import _fit_workspace, _launch

_BF16, _U8, _I32 = torch.bfloat16, torch.uint8, torch.int32


def new_paged_cache(n_pages: int, size: int, d_latent: int, n_k_rope_heads: int = 1, bits: int = 16, device="cuda",
                    ) -> Tuple[Tensor, Optional[Tensor]]:
    """One layer's ``(pages, scales)`` for ``n_pages`` pages of ``size`` tokens (a multiple of 16 up to 4096), of zeros."""
    if d_latent not in SUPPORTED_LATENT or n_k_rope_heads < 1 or n_pages < 0 or not 16 <= size <= 4096 or size % 16:
        raise ValueError(f"new_paged_cache: d_latent must be one of {SUPPORTED_LATENT}, size a multiple of 16 up to 4096; got "
                         f"d_latent {d_latent}, size {size}, n_k_rope_heads {n_k_rope_heads}, n_pages {n_pages}")
    W = d_latent + ROPE_DIM * n_k_rope_heads
    if bits == 16:
        return torch.zeros(n_pages, size, W, dtype=_BF16, device=device), None
    if bits != 4:
        raise ValueError(f"new_paged_cache: bits must be 16 or 4, got {bits}")
    return (torch.full((n_pages, size, W // 2), 0x88, dtype=_U8, device=device),
            torch.zeros(n_pages, W // 64, size, dtype=_BF16, device=device))


# ----------------------------------------------------------------- checks

def _cache(op: str, pages: Tensor, scales: Optional[Tensor], table: Tensor, B: int, d_latent: int) -> Tuple[_lib.PagedCache, int]:
    """(the C struct, Hr) of a cache and a block table for B sequences."""
    four = scales is not None
    if pages.dim() != 3 or pages.dtype != (_U8 if four else _BF16):
        raise TypeError(f"{op}: pages must be {'uint8 [n, size, W / 2] (with scales)' if four else 'bfloat16 [n, size, W]'}, got "
                        f"{pages.dtype} {tuple(pages.shape)}")
    n, size, W = pages.shape
    W *= 2 if four else 1
    Hr, rest = divmod(W - d_latent, ROPE_DIM)
    if d_latent not in SUPPORTED_LATENT or Hr < 1 or rest:
        raise ValueError(f"{op}: rows of {W} values are not a latent of {d_latent} ({SUPPORTED_LATENT}) and rotated keys of {ROPE_DIM}")
    if size % 16 or not 16 <= size <= 4096:
        raise ValueError(f"{op}: pages of {size} tokens; a multiple of 16 up to 4096 is needed")
    p0, p1, p2 = pages.stride()
    if pages.numel() and (p2 != 1 or p1 != pages.size(2) or pages.data_ptr() % 16 or (n > 1 and p0 * pages.element_size() % 16)):
        raise ValueError(f"{op}: the rows of a page must lie close together, pages 16-byte aligned (it is not copied)")
    s0 = 0
    if four:
        if scales.dtype != _BF16 or scales.shape != (n, W // 64, size):
            raise ValueError(f"{op}: scales must be bfloat16 {(n, W // 64, size)}, got {scales.dtype} {tuple(scales.shape)}")
        s0, s1, s2 = scales.stride()
        if scales.numel() and (s2 != 1 or s1 != size or scales.data_ptr() % 16 or (n > 1 and s0 % 8)):
            raise ValueError(f"{op}: the scales of a page must lie close together, pages 16-byte aligned (they are not copied)")
    if table.dtype != _I32 or table.dim() != 2 or table.size(0) != B:
        raise ValueError(f"{op}: block_table must be int32 [{B}, pages], got {table.dtype} {tuple(table.shape)}")
    return _lib.PagedCache(pages.data_ptr(), scales.data_ptr() if four else None, table.data_ptr(), n, size,
                           p0 * pages.element_size(), s0, table.size(1), table.stride(0), d_latent, Hr), Hr


def _on_device(op: str, like: Tensor, *tensors: Optional[Tensor]) -> None:
    dev = like.get_device()
    for t in (like, *tensors):
        if t is not None and (not t.is_cuda or t.get_device() != dev):
            kernels._require_gpu(op, t)
            raise ValueError(f"{op}: all tensors must be on one device, got {t.device} and {like.device}")


def _ints(op: str, name: str, t: Optional[Tensor], B: int) -> Optional[Tensor]:
    if t is None:
        return None
    if t.dtype != _I32 or t.shape != (B,):
        raise ValueError(f"{op}: {name} must be int32 [{B}], got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def _table(t: Tensor) -> Tensor:
    return t if t.dim() != 2 or t.size(1) <= 1 or (t.stride(1) == 1 and t.stride(0) >= 0) else t.contiguous()


def _sb(t: Tensor, i: int) -> int:
    return t.stride(i) if t.size(i) > 1 else 0


# ----------------------------------------------------------------- operators

@_op("paged_append", mutates_args=("pages", "scales"))
def _paged_append(qk: Tensor, c_new: Tensor, pages: Tensor, scales: Optional[Tensor], cos: Tensor, sin: Tensor,
                  block_table: Tensor, starts: Tensor, counts: Optional[Tensor]) -> Tensor:
    op = "mla_mi355x::paged_append"
    _on_device(op, qk, c_new, pages, scales, cos, sin, block_table, starts, counts)
    kernels._bf16(op, qk=qk, c_new=c_new, cos=cos, sin=sin)
    if qk.dim() != 4 or qk.size(-1) != ROPE_DIM or c_new.dim() != 3 or c_new.shape[:2] != qk.shape[:2]:
        raise ValueError(f"{op}: expected qk [B, T, H + Hr, 64] and c_new [B, T, d_latent], got {tuple(qk.shape)}, {tuple(c_new.shape)}")
    if cos.dim() != 2 or cos.size(1) != ROPE_DIM // 2 or cos.shape != sin.shape:
        raise ValueError(f"{op}: cos and sin must be [rows, 32] tables, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    B, T, heads, _ = qk.shape
    block_table = _table(block_table)
    cache, Hr = _cache(op, pages, scales, block_table, B, c_new.size(2))
    if heads < Hr:
        raise ValueError(f"{op}: qk has {heads} heads, the cache's rows {Hr} rotated keys")
    starts, counts = _ints(op, "starts", starts, B), _ints(op, "counts", counts, B)
    qk, c_new, cos, sin = _aligned4(qk, 8), _aligned4(c_new, 8), _aligned4(cos.contiguous(), 8), _aligned4(sin.contiguous(), 8)
    q_out = qk.new_empty(B, T, heads - Hr, ROPE_DIM)
    if B and T:
        args = _lib.PagedAppendArgs(
            cache, qk.data_ptr(), c_new.data_ptr(), q_out.data_ptr(), cos.data_ptr(), sin.data_ptr(), starts.data_ptr(),
            None if counts is None else counts.data_ptr(), B, T, heads - Hr, cos.size(0),
            Strides(_sb(qk, 0), _sb(qk, 1), _sb(qk, 2)), _sb(c_new, 0), _sb(c_new, 1))
        _launch("mla_paged_append", args, qk, op)
    return q_out


@_paged_append.register_fake
def _(qk, c_new, pages, scales, cos, sin, block_table, starts, counts):
    Hr = (pages.size(2) * (1 if scales is None else 2) - c_new.size(2)) // ROPE_DIM
    return qk.new_empty(qk.size(0), qk.size(1), qk.size(2) - Hr, ROPE_DIM)


@_op("paged_read", mutates_args=())
def _paged_read(pages: Tensor, scales: Optional[Tensor], block_table: Tensor, d_latent: int, T: int, starts: Optional[Tensor],
                counts: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    op = "mla_mi355x::paged_read"
    _on_device(op, pages, scales, block_table, starts, counts)
    B = block_table.size(0) if block_table.dim() else 0
    if T < 0:
        raise ValueError(f"{op}: T must not be negative, got {T}")
    block_table = _table(block_table)
    cache, Hr = _cache(op, pages, scales, block_table, B, d_latent)
    starts, counts = _ints(op, "starts", starts, B), _ints(op, "counts", counts, B)
    latent = torch.empty(B, T, d_latent, dtype=_BF16, device=pages.device)
    k_rope = torch.empty(B, Hr, T, ROPE_DIM, dtype=_BF16, device=pages.device)
    if B and T:
        args = _lib.PagedReadArgs(cache, latent.data_ptr(), k_rope.data_ptr(), None if starts is None else starts.data_ptr(),
                                  None if counts is None else counts.data_ptr(), B, T)
        _launch("mla_paged_read", args, pages, op)
    return latent, k_rope


@_paged_read.register_fake
def _(pages, scales, block_table, d_latent, T, starts, counts):
    B, W = block_table.size(0), pages.size(2) * (1 if scales is None else 2)
    return (pages.new_empty(B, T, d_latent, dtype=_BF16),
            pages.new_empty(B, (W - d_latent) // ROPE_DIM, T, ROPE_DIM, dtype=_BF16))


@_op("paged_decode", mutates_args=())
def _paged_decode(q_lat: Tensor, q_rope: Tensor, pages: Tensor, scales: Optional[Tensor], block_table: Tensor, seq_lens: Tensor,
                  scale: float) -> Tuple[Tensor, Tensor]:
    op = "mla_mi355x::paged_decode"
    _on_device(op, q_lat, q_rope, pages, scales, block_table, seq_lens)
    kernels._bf16(op, q_lat=q_lat, q_rope=q_rope)
    if q_lat.dim() != 3 or q_rope.shape != (*q_lat.shape[:2], ROPE_DIM):
        raise ValueError(f"{op}: expected q_lat [B, H, d_latent] and q_rope [B, H, 64], got {tuple(q_lat.shape)}, {tuple(q_rope.shape)}")
    B, H, DL = q_lat.shape
    block_table = _table(block_table)
    cache, Hr = _cache(op, pages, scales, block_table, B, DL)
    if Hr not in (1, H):
        raise ValueError(f"{op}: rows with {Hr} rotated keys do not go with {H} heads (1 or {H})")
    seq_lens = _ints(op, "seq_lens", seq_lens, B)
    q_lat, q_rope = _aligned4(q_lat, 8), _aligned4(q_rope, 8)
    ctx = q_lat.new_empty(B, H, DL)
    lse = q_lat.new_empty(B, H, dtype=torch.float32)
    if ctx.numel():
        args = _lib.PagedDecodeArgs(cache, q_lat.data_ptr(), q_rope.data_ptr(), seq_lens.data_ptr(), ctx.data_ptr(), lse.data_ptr(),
                                    None, 0, B, H, _sb(q_lat, 0), _sb(q_lat, 1), _sb(q_rope, 0), _sb(q_rope, 1), scale)
        ws = _fit_workspace("mla_paged_decode_workspace_bytes", args, q_lat)  # noqa: F841  (kept until the launch)
        _launch("mla_paged_decode", args, q_lat, op)
    return ctx, lse


@_paged_decode.register_fake
def _(q_lat, q_rope, pages, scales, block_table, seq_lens, scale):
    return q_lat.new_empty(q_lat.shape), q_lat.new_empty(q_lat.shape[:2], dtype=torch.float32)


_append_call, _read_call, _decode_call = (_eager_call(n) for n in ("paged_append", "paged_read", "paged_decode"))


# ----------------------------------------------------------------- public functions

def paged_append(qk: Tensor, c_new: Tensor, pages: Tensor, scales: Optional[Tensor], cos: Tensor, sin: Tensor, block_table: Tensor,
                 starts: Tensor, counts: Optional[Tensor] = None) -> Tensor:
    """Appends tokens t < ``counts[b]`` (None: all T) of sequence b at positions ``starts[b] + t``: the k heads of ``qk [B, T,
    H + Hr, 64]`` (q heads first) are rotated with the bf16 tables ``cos`` and ``sin [rows, 32]``, and with ``c_new [B, T,
    d_latent]`` written to their rows in ``pages`` (and ``scales``).  Returns the rotated q heads ``[B, T, H, 64]``, zeros for the
    other t.  A position without a page is not written; one outside the tables is skipped, its q heads zero.  Two tokens of a call
    must not go to the same place."""
    return _append_call(qk, c_new, pages, scales, cos, sin, block_table, starts, counts)


def paged_read(pages: Tensor, scales: Optional[Tensor], block_table: Tensor, d_latent: int, T: int, starts: Optional[Tensor] = None,
               counts: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``(latent [B, T, d_latent], k_rope [B, Hr, T, 64])``, bf16, of positions ``starts[b] + t``, t < ``counts[b]`` (None: from 0,
    all T); zeros for the other t and where there is no page."""
    return _read_call(pages, scales, block_table, d_latent, T, starts, counts)


def paged_decode(q_lat: Tensor, q_rope: Tensor, pages: Tensor, scales: Optional[Tensor], block_table: Tensor, seq_lens: Tensor,
                 scale: float) -> Tuple[Tensor, Tensor]:
    """``ctx [B, H, d_latent]`` bf16 and ``lse [B, H]`` fp32 of one query token a sequence, ``q_lat [B, H, d_latent]`` (absorbed
    through W_UK) and ``q_rope [B, H, 64]`` (rotated), over the first ``seq_lens[b]`` positions: ``softmax((q_lat . c + q_rope . k)
    scale) c``, as ``torch.ops.mla_mi355x.decode`` over a contiguous cache.  Tokens without a page take no part; a sequence
    without tokens has ctx 0 and lse -inf."""
    return _decode_call(q_lat, q_rope, pages, scales, block_table, seq_lens, scale)
