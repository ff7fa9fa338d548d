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

from . import kernels
from .host_calls import Entry, plain
from .kernels import ROPE_DIM, SUPPORTED_LATENT, _aligned4, _op

_BF16, _U8, _I32, _F32 = torch.bfloat16, torch.uint8, torch.int32, torch.float32
_CACHE = "3P8q"  # mla_paged_cache
_append_entry = Entry("mla_paged_append", _CACHE + "7P9q", "PagedAppendArgs")
_read_entry = Entry("mla_paged_read", _CACHE + "4P2q", "PagedReadArgs")
_decode_entry = Entry("mla_paged_decode", _CACHE + "6PN6qf4x", "PagedDecodeArgs")
_decode_bytes = Entry("mla_paged_decode_workspace_bytes", _CACHE + "6PN6qf4x", "PagedDecodeArgs", stream=False)
_workspaces = {}  # bytes by sizes


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

def _refuse_cache(op, pages, scales, table, B, d_latent) -> None:
    """The error of a cache or block table that :func:`_cache` did not take."""
    four = scales is not None
    if pages.dim() != 3 or pages.dtype != (_U8 if four else _BF16):
        raise TypeError(f"{op}: pages must be {'uint8 [n, size, W / 2] (with scales)' if four else 'bfloat16 [n, size, W]'}, got "
                        f"{pages.dtype} {tuple(pages.shape)}")
    n, size, W = pages.shape
    W *= 2 if four else 1
    if d_latent not in SUPPORTED_LATENT or W - d_latent < ROPE_DIM or (W - d_latent) % ROPE_DIM:
        raise ValueError(f"{op}: rows of {W} values are not a latent of {d_latent} ({SUPPORTED_LATENT}) and rotated keys of {ROPE_DIM}")
    if size % 16 or not 16 <= size <= 4096:
        raise ValueError(f"{op}: pages of {size} tokens; a multiple of 16 up to 4096 is needed")
    if four and (scales.dtype != _BF16 or scales.shape != (n, W // 64, size)):
        raise ValueError(f"{op}: scales must be bfloat16 {(n, W // 64, size)}, got {scales.dtype} {tuple(scales.shape)}")
    if table.dtype != _I32 or table.dim() != 2 or table.size(0) != B:
        raise ValueError(f"{op}: block_table must be int32 [{B}, pages], got {table.dtype} {tuple(table.shape)}")
    raise ValueError(f"{op}: the rows and scales of a page must lie close together, and pages 16-byte aligned (they are not copied); "
                     f"strides {pages.stride()}{'' if not four else f', {scales.stride()}'}")


def _cache(op: str, pages: Tensor, scales: Optional[Tensor], table: Tensor, B: int, d_latent: int):
    """(the fields of mla_paged_cache, Hr, what they point to) of a cache and a block table for B sequences."""
    if pages.dim() != 3 or table.dim() != 2:
        _refuse_cache(op, pages, scales, table, B, d_latent)
    rows, P = table.shape
    (n, size, cols), (p0, p1, p2), at = pages.shape, pages.stride(), pages.data_ptr()
    if scales is None:
        W, p0, s0, sat = cols, 2 * p0, 0, 0
        ok = pages.dtype is _BF16
    else:
        W, s0, sat = 2 * cols, 0, scales.data_ptr()
        ok = pages.dtype is _U8 and scales.dtype is _BF16 and scales.shape == (n, W >> 6, size)
        if ok and n:
            s0, s1, s2 = scales.stride()
            ok = s2 == 1 and s1 == size and not sat & 15 and (n == 1 or not s0 & 7)
    Hr, rest = divmod(W - d_latent, ROPE_DIM)
    ok = ok and d_latent in SUPPORTED_LATENT and Hr > 0 and not rest and not size & 15 and 16 <= size <= 4096 \
        and table.dtype is _I32 and rows == B \
        and (n == 0 or (p2 == 1 and p1 == cols and not at & 15 and (n == 1 or not p0 & 15)))
    if not ok:
        _refuse_cache(op, pages, scales, table, B, d_latent)
    t0, t1 = table.stride()
    if P > 1 and (t1 != 1 or t0 < 0):
        table = table.contiguous()
        t0 = P
    return (at, sat, table.data_ptr(), n, size, p0, s0, P, t0, d_latent, Hr), Hr, table


def _on_device(op: str, like: Tensor, *tensors: Optional[Tensor]) -> None:
    dev = like.get_device()
    if dev < 0:
        kernels._require_gpu(op, like)
    for t in tensors:
        if t is not None and t.get_device() != dev:
            kernels._require_gpu(op, t)
            raise ValueError(f"{op}: all tensors must be on one device, got {t.device} and {like.device}")


def _ints(op: str, name: str, t: Tensor, B: int) -> Tensor:
    if t.dtype is not _I32 or t.shape != (B,):
        raise ValueError(f"{op}: {name} must be int32 [{B}], got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _strided(t: Tensor):
    """``t`` (or a copy) with unit inner stride, 16-byte aligned, other strides multiples of 8, and those strides (0 for a dimension
    of size 1, whose own may be any number)."""
    st = t.stride()
    if st[-1] == 1 and not t.data_ptr() & 15:
        for s in st[:-1]:
            if s & 7 or s < 0:
                break
        else:
            return t, st
    t = _aligned4(t, 8)
    return t, (*(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)), 1)


def _rope_table(t: Tensor) -> Tensor:
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


# ----------------------------------------------------------------- operators

@_op("paged_append", mutates_args=("pages", "scales"))
def _paged_append(qk: Tensor, c_new: Tensor, pages: Tensor, scales: Optional[Tensor], cos: Tensor, sin: Tensor,
                  block_table: Tensor, starts: Tensor, counts: Optional[Tensor]) -> Tensor:
    _on_device("mla_mi355x::paged_append", qk, c_new, pages, scales, cos, sin, block_table, starts, counts)
    return _append(qk, c_new, pages, scales, cos, sin, block_table, starts, counts)


def _append(qk, c_new, pages, scales, cos, sin, block_table, starts, counts):
    op = "mla_mi355x::paged_append"
    if not qk.dtype is c_new.dtype is cos.dtype is sin.dtype is _BF16:
        kernels._bf16(op, qk=qk, c_new=c_new, cos=cos, sin=sin)
    if qk.dim() != 4 or c_new.dim() != 3 or qk.size(3) != ROPE_DIM or c_new.shape[:2] != qk.shape[:2]:
        raise ValueError(f"{op}: expected qk [B, T, H + Hr, 64] and c_new [B, T, d_latent], got {tuple(qk.shape)}, {tuple(c_new.shape)}")
    B, T, heads, _ = qk.shape
    if cos.dim() != 2 or cos.size(1) != ROPE_DIM // 2 or cos.shape != sin.shape:
        raise ValueError(f"{op}: cos and sin must be [rows, 32] tables, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    cache, Hr, block_table = _cache(op, pages, scales, block_table, B, c_new.size(2))
    if heads < Hr:
        raise ValueError(f"{op}: qk has {heads} heads, the cache's rows {Hr} rotated keys")
    starts = _ints(op, "starts", starts, B)
    counts = None if counts is None else _ints(op, "counts", counts, B)
    qk, (q0, q1, q2, _) = _strided(qk)
    c_new, (c0, c1, _) = _strided(c_new)
    cos, sin = _rope_table(cos), _rope_table(sin)
    q_out = qk.new_empty((B, T, heads - Hr, ROPE_DIM))
    if B and T:
        _append_entry(op, qk.get_device(), *cache, qk.data_ptr(), c_new.data_ptr(), q_out.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                      starts.data_ptr(), 0 if counts is None else counts.data_ptr(), B, T, heads - Hr, cos.size(0), q0, q1, q2, c0, c1)
    return q_out


@_paged_append.register_fake
def _(qk, c_new, pages, scales, cos, sin, block_table, starts, counts):
    Hr = (pages.size(2) * (1 if scales is None else 2) - c_new.size(2)) // ROPE_DIM
    return qk.new_empty(qk.size(0), qk.size(1), qk.size(2) - Hr, ROPE_DIM)


@_op("paged_read", mutates_args=())
def _paged_read(pages: Tensor, scales: Optional[Tensor], block_table: Tensor, d_latent: int, T: int, starts: Optional[Tensor],
                counts: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    _on_device("mla_mi355x::paged_read", pages, scales, block_table, starts, counts)
    return _read(pages, scales, block_table, d_latent, T, starts, counts)


def _read(pages, scales, block_table, d_latent, T, starts, counts):
    op = "mla_mi355x::paged_read"
    B = block_table.size(0) if block_table.dim() else 0
    if T < 0:
        raise ValueError(f"{op}: T must not be negative, got {T}")
    cache, Hr, block_table = _cache(op, pages, scales, block_table, B, d_latent)
    starts = None if starts is None else _ints(op, "starts", starts, B)
    counts = None if counts is None else _ints(op, "counts", counts, B)
    latent = pages.new_empty((B, T, d_latent), dtype=_BF16)
    k_rope = pages.new_empty((B, Hr, T, ROPE_DIM), dtype=_BF16)
    if B and T:
        _read_entry(op, pages.get_device(), *cache, latent.data_ptr(), k_rope.data_ptr(), 0 if starts is None else starts.data_ptr(),
                    0 if counts is None else counts.data_ptr(), B, T)
    return latent, k_rope


@_paged_read.register_fake
def _(pages, scales, block_table, d_latent, T, starts, counts):
    B, W = block_table.size(0), pages.size(2) * (1 if scales is None else 2)
    return (pages.new_empty(B, T, d_latent, dtype=_BF16),
            pages.new_empty(B, (W - d_latent) // ROPE_DIM, T, ROPE_DIM, dtype=_BF16))


@_op("paged_decode", mutates_args=())
def _paged_decode(q_lat: Tensor, q_rope: Tensor, pages: Tensor, scales: Optional[Tensor], block_table: Tensor, seq_lens: Tensor,
                  scale: float) -> Tuple[Tensor, Tensor]:
    _on_device("mla_mi355x::paged_decode", q_lat, q_rope, pages, scales, block_table, seq_lens)
    return _decode(q_lat, q_rope, pages, scales, block_table, seq_lens, scale)


def _decode(q_lat, q_rope, pages, scales, block_table, seq_lens, scale):
    op = "mla_mi355x::paged_decode"
    dev = q_lat.get_device()
    if not q_lat.dtype is q_rope.dtype is _BF16:
        kernels._bf16(op, q_lat=q_lat, q_rope=q_rope)
    if q_lat.dim() != 3 or q_rope.shape != (*q_lat.shape[:2], ROPE_DIM):
        raise ValueError(f"{op}: expected q_lat [B, H, d_latent] and q_rope [B, H, 64], got {tuple(q_lat.shape)}, {tuple(q_rope.shape)}")
    B, H, DL = q_lat.shape
    cache, Hr, block_table = _cache(op, pages, scales, block_table, B, DL)
    if Hr != 1 and Hr != H:
        raise ValueError(f"{op}: rows with {Hr} rotated keys do not go with {H} heads (1 or {H})")
    seq_lens = _ints(op, "seq_lens", seq_lens, B)
    q_lat, (l0, l1, _) = _strided(q_lat)
    q_rope, (r0, r1, _) = _strided(q_rope)
    ctx = q_lat.new_empty((B, H, DL))
    lse = q_lat.new_empty((B, H), dtype=_F32)
    if B and H:
        key = (B, H, DL, Hr, cache[7], cache[4], cache[1] == 0)  # (no scales: an empty cache in 4 bits too)
        nbytes = _workspaces.get(key)
        if nbytes is None:
            if len(_workspaces) > 4096:
                _workspaces.clear()
            nbytes = _decode_bytes(op, dev, *cache, 0, 0, 0, 0, 0, 0, 0, B, H, 0, 0, 0, 0, 0.0)
            if nbytes:  # (0: arguments that the call will refuse)
                _workspaces[key] = nbytes
        ws = q_lat.new_empty(nbytes, dtype=_U8)
        _decode_entry(op, dev, *cache, q_lat.data_ptr(), q_rope.data_ptr(), seq_lens.data_ptr(), ctx.data_ptr(), lse.data_ptr(),
                      ws.data_ptr(), nbytes, B, H, l0, l1, r0, r1, scale)
    return ctx, lse


@_paged_decode.register_fake
def _(q_lat, q_rope, pages, scales, block_table, seq_lens, scale):
    return q_lat.new_empty(q_lat.shape), q_lat.new_empty(q_lat.shape[:2], dtype=_F32)


_ops = torch.ops.mla_mi355x
_increment_version = torch._C._increment_version


# ----------------------------------------------------------------- public functions

def paged_append(qk: Tensor, c_new: Tensor, pages: Tensor, scales: Optional[Tensor], cos: Tensor, sin: Tensor, block_table: Tensor,
                 starts: Tensor, counts: Optional[Tensor] = None) -> Tensor:
    """Appends tokens t < ``counts[b]`` (None: all T) of sequence b at positions ``starts[b] + t``: the k heads of ``qk [B, T,
    H + Hr, 64]`` (q heads first) are rotated with the bf16 tables ``cos`` and ``sin [rows, 32]``, and with ``c_new [B, T,
    d_latent]`` written to their rows in ``pages`` (and ``scales``).  Returns the rotated q heads ``[B, T, H, 64]``, zeros for the
    other t.  A position without a page is not written; one outside the tables is skipped, its q heads zero.  Two tokens of a call
    must not go to the same place."""
    if not plain(qk, c_new, pages, scales, cos, sin, block_table, starts, counts):
        return _ops.paged_append(qk, c_new, pages, scales, cos, sin, block_table, starts, counts)
    q_rope = _append(qk, c_new, pages, scales, cos, sin, block_table, starts, counts)
    _increment_version([pages] if scales is None else [pages, scales])  # as the dispatcher does for what an operator writes
    return q_rope


def paged_read(pages: Tensor, scales: Optional[Tensor], block_table: Tensor, d_latent: int, T: int, starts: Optional[Tensor] = None,
               counts: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``(latent [B, T, d_latent], k_rope [B, Hr, T, 64])``, bf16, of positions ``starts[b] + t``, t < ``counts[b]`` (None: from 0,
    all T); zeros for the other t and where there is no page."""
    run = _read if plain(pages, scales, block_table, starts, counts) else _ops.paged_read
    return run(pages, scales, block_table, d_latent, T, starts, counts)


def paged_decode(q_lat: Tensor, q_rope: Tensor, pages: Tensor, scales: Optional[Tensor], block_table: Tensor, seq_lens: Tensor,
                 scale: float) -> Tuple[Tensor, Tensor]:
    """``ctx [B, H, d_latent]`` bf16 and ``lse [B, H]`` fp32 of one query token a sequence, ``q_lat [B, H, d_latent]`` (absorbed
    through W_UK) and ``q_rope [B, H, 64]`` (rotated), over the first ``seq_lens[b]`` positions: ``softmax((q_lat . c + q_rope . k)
    scale) c``, as ``torch.ops.mla_mi355x.decode`` over a contiguous cache.  Tokens without a page take no part; a sequence
    without tokens has ctx 0 and lse -inf."""
    run = _decode if plain(q_lat, q_rope, pages, scales, block_table, seq_lens) else _ops.paged_decode
    return run(q_lat, q_rope, pages, scales, block_table, seq_lens, scale)
