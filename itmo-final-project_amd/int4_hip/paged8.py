"""Key-value cache in pages held in 8 bits, for batches of sequences: tokens quantised as
they are written, read back, and the attention of a few new tokens of every row over
them (csrc/w4_paged8.hip).  It holds about twice the tokens of ``paged.py``'s cache; a decode
step's attention takes 0.6 to 0.75 of the time (56 us instead of 88 over 131000 slots of 8
heads of 128, 23 instead of 32 over 32 ragged rows of up to 4000 of 8 heads of 64).

One layer's cache, shared by all sequences of a batch (``rows``):

  * ``k_pages``, ``v_pages`` [pages, kv_heads, page_size, head_dim], ``torch.int8`` or
    ``torch.float8_e4m3fn``; keys are held rotated.  head_dim 64 or 128, page_size a
    power of two from 8 to 1024;
  * ``k_scale``, ``v_scale`` fp32 [pages, kv_heads, page_size / block]: a code stands for
    code * scale of its block of ``block`` slots, a power of two from 8 to 64;
  * ``table`` int32 [rows, width]: the page of slots i * page_size.. of a row (entries
    that no token of a call sees are not read).  Rows may share pages that none of them
    writes to.

The new tokens of a call are those of all rows one after the other: row b's are
``offsets[b]``..``offsets[b + 1]`` (int32 [rows + 1], not decreasing) and go to slots
``lengths[b]``.. (int32 [rows], the tokens a row has; < 0: an idle row).  ``positions``
int32 [tokens] are theirs, ``cos`` and ``sin`` the tables of all positions, fp32
[positions, head_dim / 2] (``apply_rope`` of ``llama.py``: the two halves of a head are
rotated).

A block's scale is its largest magnitude over the largest code (127, 448).  It starts with
the block's first slot; tokens that come later let it grow by a power of two if they need
it.  All other codes of the block are then divided by that power (those behind the row's
last token too), which keeps e4m3 codes exactly (but for the smallest) and costs int8 codes
one step in all.  Tokens written over (drafts that were refused) leave the scale where it is
and the other codes divided; who wants neither keeps the block and puts it back
(``BatchDecoder.verify``).  A block that an infinity or NaN comes into reads as NaN until its
first slot is written again.

The functions launch on the current stream and never synchronise, so lengths, offsets,
pages and positions, which live on the GPU, are checked there: what is out of range is
not read or written.  Nothing here takes part in autograd.
"""
from __future__ import annotations

import torch

from . import _lib
from .gemm import _with_workspace
from .llama_ops import DTYPES, _on
from .paged import HEAD_DIMS, _angles, _index, _no_grad, _rows

CODES = {torch.int8: _lib.CODE_INT8, torch.float8_e4m3fn: _lib.CODE_E4M3}
OUT = {**DTYPES, torch.float32: _lib.DTYPE_FP32}


def _cache(k_pages, v_pages, k_scale, v_scale, table):
    """The C description of a cache, its tensors checked."""
    assert k_pages.dtype in CODES and v_pages.dtype == k_pages.dtype, (k_pages.dtype, v_pages.dtype)
    assert k_pages.dim() == 4 and v_pages.shape == k_pages.shape
    P, nkv, S, d = k_pages.shape
    assert d in HEAD_DIMS and 8 <= S <= 1024 and S & (S - 1) == 0, (S, d)
    dev = k_pages.device
    tensors = (k_pages, v_pages, k_scale, v_scale, table)
    assert k_pages.is_cuda and all(t.device == dev and t.is_contiguous() and not t.is_neg() for t in tensors)
    assert k_scale.dtype == v_scale.dtype == torch.float32 and v_scale.shape == k_scale.shape
    assert k_scale.dim() == 3 and k_scale.shape[:2] == (P, nkv) and k_scale.shape[2] >= 1, k_scale.shape
    block = S // k_scale.shape[2]
    assert k_scale.shape[2] * block == S and block in (8, 16, 32, 64), (S, k_scale.shape)
    assert table.dtype == torch.int32 and table.dim() == 2 and table.shape[1] >= 1
    return _lib.Paged8Cache(k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                            table.data_ptr(), P, nkv, S, d, block, table.shape[0], table.shape[1],
                            CODES[k_pages.dtype], 0)


def _new(k, v, cos, sin, lengths, offsets, positions, c, dev):
    T, width = k.shape[0], c.kv_heads * c.head_dim
    assert k.dtype in DTYPES and k.dim() == 2, (k.dtype, k.shape)
    k, v = (_rows(t, T, width, k.dtype, dev) for t in (k, v))
    lengths, offsets, positions = _index(lengths, c.rows, dev), _index(offsets, c.rows + 1, dev), _index(positions, T, dev)
    return k, v, *_angles(cos, sin, c.head_dim, dev), lengths, offsets, positions


def paged_append8(k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions) -> None:
    """Write new tokens into the pages: keys ``k`` [tokens, kv_heads * head_dim] (bf16 or
    fp16), rotated at ``positions``, and values ``v`` are quantised (the module's docstring)
    and go to their rows' slots.

    Idle rows, rows whose slots pass the table, tokens of no row and pages outside the pool
    are left out; a position outside the tables makes a key of NaN.
    """
    if _lib.ext is not None and _lib.ext.paged_append8(k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths,
                                                       offsets, positions):
        return  # plain operands: the same call without Python's share of its cost
    _no_grad(k, v, cos, sin, k_pages, v_pages, k_scale, v_scale)
    c = _cache(k_pages, v_pages, k_scale, v_scale, table)
    dev = k_pages.device
    k, v, cos, sin, lengths, offsets, positions = _new(k, v, cos, sin, lengths, offsets, positions, c, dev)
    lib = _lib.load()
    rc = _on(dev, lambda st: lib.w4_paged8_append(
        c, DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k.shape[0], lengths.data_ptr(),
        offsets.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], st))
    if rc:
        _lib.check(rc, "w4_paged8_append")


def paged_read8(k_pages, v_pages, k_scale, v_scale, table, starts, offsets, tokens: int,
                dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys (rotated, as they are held) and values of slots ``starts[b]``.. of every row,
    [tokens, kv_heads * head_dim] each in ``dtype`` (bf16, fp16 or fp32): row b's are
    ``offsets[b]``..``offsets[b + 1]``.  Code * scale, rounded once.

    Tokens of no row and of rows with ``starts[b] < 0`` are 0; slots past the table or on a
    page outside the pool are NaN.
    """
    if _lib.ext is not None:
        kv = _lib.ext.paged_read8(k_pages, v_pages, k_scale, v_scale, table, starts, offsets, tokens, dtype)
        if kv is not None:
            return kv
    _no_grad(k_pages, v_pages, k_scale, v_scale)
    c = _cache(k_pages, v_pages, k_scale, v_scale, table)
    dev = k_pages.device
    assert dtype in OUT and tokens >= 0, (dtype, tokens)
    starts, offsets = _index(starts, c.rows, dev), _index(offsets, c.rows + 1, dev)
    k, v = (torch.empty((tokens, c.kv_heads * c.head_dim), dtype=dtype, device=dev) for _ in range(2))
    lib = _lib.load()
    rc = _on(dev, lambda st: lib.w4_paged8_read(c, OUT[dtype], starts.data_ptr(), offsets.data_ptr(), tokens,
                                                k.data_ptr(), v.data_ptr(), st))
    if rc:
        _lib.check(rc, "w4_paged8_read")
    return k, v


def paged_attention8(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets, positions,
                     longest: int | None = None, window: int | None = None, sinks: int = 0) -> torch.Tensor:
    """Attention output [tokens, heads * head_dim] of the new tokens of every row: one of a
    decode step, a few drafted ones, a prompt's or a chunk of it.

    ``q`` [tokens, heads * head_dim], ``k``, ``v`` [tokens, kv_heads * head_dim]: their
    projections before the rotary embedding, bf16 or fp16.  Keys and values are written as
    by ``paged_append8``; then the token of slot i attends in fp32 to slots 0..i or, with
    ``window``, to the last ``window`` of them and the first ``sinks``.  ``longest`` is
    the most new tokens that a row may have, where the program knows it (None or 0: any
    number): of a decode step, 1, for which one launch writes and attends where blocks have
    at most 32 slots and a key head at most 16 query heads.  ``lengths`` is left as it is (all layers of a
    model share it).

    Idle rows and tokens of no row come back 0.  NaN come back: rows with more
    than ``longest`` tokens or whose slots pass the table (nothing of them is written);
    tokens that see a page outside the pool or a block of NaN, or whose position is outside
    the tables.
    """
    if _lib.ext is not None:
        out = _lib.ext.paged_attention8(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, table, lengths, offsets,
                                        positions, longest, window, sinks)
        if out is not None:
            return out
    _no_grad(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale)
    c = _cache(k_pages, v_pages, k_scale, v_scale, table)
    dev, T = k_pages.device, q.shape[0]
    nkv, d = c.kv_heads, c.head_dim
    assert q.dim() == 2 and q.shape[1] and q.shape[1] % (nkv * d) == 0, q.shape
    assert k.shape[0] == T and k.dtype == q.dtype, (k.shape, q.shape, k.dtype, q.dtype)
    assert window is None or window >= 1, window
    assert sinks >= 0 and (longest is None or longest >= 0), (sinks, longest)
    nh = q.shape[1] // d
    k, v, cos, sin, lengths, offsets, positions = _new(k, v, cos, sin, lengths, offsets, positions, c, dev)
    q = _rows(q, T, nh * d, k.dtype, dev)
    out = torch.empty((T, nh * d), dtype=q.dtype, device=dev)
    lib = _lib.load()
    nbytes = lib.w4_paged8_attention_workspace_bytes(c.rows, T, nh, nkv, d)
    rc = _on(dev, lambda st: _with_workspace(dev, st, nbytes, lambda ws, nb: lib.w4_paged8_attention(
        c, DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0), v.stride(0), nh, T,
        longest or 0, window or 0, sinks, lengths.data_ptr(), offsets.data_ptr(), positions.data_ptr(),
        cos.data_ptr(), sin.data_ptr(), cos.shape[0], out.data_ptr(), ws, nb, st)))
    if rc:
        _lib.check(rc, "w4_paged8_attention")
    return out
