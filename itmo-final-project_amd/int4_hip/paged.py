"""Key-value cache in pages for batches of sequences: tokens written into it, the
attention of one new token of every sequence, and eviction by accumulated
attention weight (csrc/w4_paged.hip).

One layer's cache, shared by all sequences of a batch (``rows``):

  * ``k_pages``, ``v_pages`` [pages, kv_heads, page_size, head_dim], bf16 or fp16
    like the activations; keys are held rotated.  head_dim 64 or 128, page_size a
    power of two from 8 to 1024;
  * ``table`` int32 [rows, width]: the page of slots i * page_size.. of a row
    (entries past its tokens are not read);
  * ``weight`` fp32 [pages, kv_heads, page_size], where the cache is to be evicted
    from: the attention each token has received, from the queries of ``paged_attention``
    alone, since it came into the cache.

Rows may share pages (a common prefix) where there is no ``weight`` and none of them
writes there.  With ``weight`` every page is one row's alone: the attention of a row
reads, adds to and writes back its weights with no regard to another's, and
``paged_append`` sets them to 0.

A token's *slot* is its place in the cache, its *position* the one its angles are
taken from; they part once something is evicted.  ``cos`` and ``sin`` are the
tables of all positions, fp32 [positions, head_dim / 2] (``apply_rope`` of
``llama.py``: the two halves of a head are rotated).

The functions launch on the current stream and never synchronise, so lengths, slots,
pages and positions, which live on the GPU, are checked there: what is out of range
is not read or written, and an attention row that needs it comes back NaN.  Nothing
here takes part in autograd.
"""
from __future__ import annotations

import torch

from . import _lib
from .gemm import _with_workspace
from .llama_ops import DTYPES, _on, underived

HEAD_DIMS = (64, 128)


def _no_grad(*tensors):
    assert underived(*tensors), \
        "the paged cache's operators have no derivatives: call them under torch.no_grad(), on tensors without tangents"


def _cache(k_pages, v_pages, table, weight):
    """The C description of a cache, its tensors checked."""
    assert k_pages.dtype in DTYPES and v_pages.dtype == k_pages.dtype
    assert k_pages.dim() == 4 and v_pages.shape == k_pages.shape
    P, nkv, S, d = k_pages.shape
    assert d in HEAD_DIMS and 8 <= S <= 1024 and S & (S - 1) == 0, (S, d)
    dev = k_pages.device
    assert k_pages.is_cuda and v_pages.device == table.device == dev
    assert k_pages.is_contiguous() and v_pages.is_contiguous()
    assert not any(t is not None and t.is_neg() for t in (k_pages, v_pages, table, weight))
    assert table.dtype == torch.int32 and table.dim() == 2 and table.is_contiguous() and table.shape[1] >= 1
    if weight is not None:
        assert weight.dtype == torch.float32 and weight.shape == (P, nkv, S) and weight.is_contiguous()
        assert weight.device == dev
    return _lib.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), None if weight is None else weight.data_ptr(),
                           table.data_ptr(), P, nkv, S, d, table.shape[0], table.shape[1])


def _angles(cos, sin, d, dev):
    assert cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape
    assert cos.shape[1] == d // 2 and cos.shape[0] >= 1 and cos.device == sin.device == dev
    cos, sin = cos.resolve_neg(), sin.resolve_neg()
    return tuple(t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                 for t in (cos, sin))


def _rows(t, n, width, dtype, dev):
    """``t`` [n, width] with dense, 16-byte aligned rows, copied where it has none."""
    assert t.dtype == dtype and t.device == dev and t.shape == (n, width), (t.dtype, t.shape, (n, width))
    t = t.resolve_neg()
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _index(t, n, dev):
    assert t.dtype == torch.int32 and t.shape == (n,) and t.device == dev, (t.dtype, t.shape, n)
    return t.resolve_neg().contiguous()


def paged_append(k, v, cos, sin, k_pages, v_pages, table, rows, slots, positions, weight=None) -> None:
    """Write tokens into the pages: key t of ``k`` [tokens, kv_heads * head_dim], rotated
    at ``positions[t]``, and value t of ``v`` go to slot ``slots[t]`` of table row
    ``rows[t]`` (int32 [tokens] each); ``weight`` there becomes 0.

    A token whose row, slot, page or position is out of range (any negative number:
    padding) is left out.
    """
    if _lib.ext is not None and _lib.ext.paged_append(k, v, cos, sin, k_pages, v_pages, table, rows, slots, positions,
                                                      weight):
        return  # plain operands: the same call without Python's share of its cost
    _no_grad(k, v, cos, sin, k_pages, v_pages, weight)
    c = _cache(k_pages, v_pages, table, weight)
    dev, T = k_pages.device, k.shape[0]
    nkv, d = c.kv_heads, c.head_dim
    k, v = (_rows(t, T, nkv * d, k_pages.dtype, dev) for t in (k, v))
    rows, slots, positions = (_index(t, T, dev) for t in (rows, slots, positions))
    cos, sin = _angles(cos, sin, d, dev)
    lib = _lib.load()
    rc = _on(dev, lambda st: lib.w4_paged_append(
        c, DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), T, rows.data_ptr(),
        slots.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], st))
    if rc:
        _lib.check(rc, "w4_paged_append")


def paged_attention(q, k, v, cos, sin, k_pages, v_pages, table, lengths, positions, weight=None) -> torch.Tensor:
    """Attention output [rows, heads * head_dim] of one new token of every row.

    ``q`` [rows, heads * head_dim], ``k``, ``v`` [rows, kv_heads * head_dim]: the new
    tokens' projections before the rotary embedding, in the cache's dtype; ``lengths``
    int32 [rows]: the tokens a row has in the cache, ``positions`` int32 [rows]: the new
    tokens' positions.  The new key and value go to slot ``lengths[b]``, then the row's
    query attends to slots 0..lengths[b] in fp32; with ``weight`` each of them is
    credited the probabilities its head's group gave it; the call then holds rows * heads
    * width * page_size fp32 scores, so a table is best passed no wider than its longest
    row needs.  ``lengths`` is left as it is (all layers of a model share it).

    ``lengths[b] < 0``: an idle row, its output zero, nothing written.  A slot past the
    table, a page outside the pool or a position outside the tables: the row's output
    is NaN.
    """
    if _lib.ext is not None:
        out = _lib.ext.paged_attention(q, k, v, cos, sin, k_pages, v_pages, table, lengths, positions, weight)
        if out is not None:
            return out
    _no_grad(q, k, v, cos, sin, k_pages, v_pages, weight)
    c = _cache(k_pages, v_pages, table, weight)
    dev, dtype, B = k_pages.device, k_pages.dtype, table.shape[0]
    nkv, d = c.kv_heads, c.head_dim
    assert q.dim() == 2 and q.shape[1] and q.shape[1] % (nkv * d) == 0, q.shape
    nh = q.shape[1] // d
    q = _rows(q, B, nh * d, dtype, dev)
    k, v = (_rows(t, B, nkv * d, dtype, dev) for t in (k, v))
    lengths, positions = (_index(t, B, dev) for t in (lengths, positions))
    cos, sin = _angles(cos, sin, d, dev)
    out = torch.empty((B, nh * d), dtype=dtype, device=dev)
    scores = None if weight is None else torch.empty(B * nh * c.width * c.page_size, device=dev)
    lib = _lib.load()
    nbytes = lib.w4_paged_attention_workspace_bytes(B, nh, nkv, d)
    rc = _on(dev, lambda st: _with_workspace(dev, st, nbytes, lambda ws, nb: lib.w4_paged_attention(
        c, DTYPES[dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0), v.stride(0), nh,
        lengths.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], out.data_ptr(),
        None if scores is None else scores.data_ptr(), ws, nb, st)))
    if rc:
        _lib.check(rc, "w4_paged_attention")
    return out


def paged_evict(k_pages, v_pages, weight, table, lengths, new_table, keep: int, recent: int) -> torch.Tensor:
    """Copy the tokens worth keeping to the pages of ``new_table`` [rows, new_width] and
    return their number, int32 [rows].

    Of a row's n = ``lengths[b]`` tokens, and for every key-value head apart, all are kept
    where n <= ``keep``; else the last ``recent`` and, of the others, the ``keep - recent``
    of largest weight (the lower slot first among equals, NaN above every number).  They
    stay in the order of their slots and take their weights along.  The old pages are
    left whole; the pages of ``new_table`` must not be among them, nor stand in it twice.
    A row of length < 0, or longer than its table, is left alone (-1).
    """
    if _lib.ext is not None:
        n = _lib.ext.paged_evict(k_pages, v_pages, weight, table, lengths, new_table, keep, recent)
        if n is not None:
            return n
    _no_grad(k_pages, v_pages, weight)
    assert weight is not None
    c = _cache(k_pages, v_pages, table, weight)
    dev, B = k_pages.device, table.shape[0]
    lengths = _index(lengths, B, dev)
    assert new_table.dtype == torch.int32 and new_table.dim() == 2 and new_table.shape[0] == B
    assert new_table.is_contiguous() and new_table.device == dev and not new_table.is_neg()
    assert 0 <= recent <= keep and 1 <= keep <= new_table.shape[1] * c.page_size, (keep, recent, new_table.shape)
    n = torch.empty(B, dtype=torch.int32, device=dev)
    lib = _lib.load()
    scratch = torch.empty(lib.w4_paged_evict_scratch_words(c, keep), dtype=torch.int32, device=dev)
    rc = _on(dev, lambda st: lib.w4_paged_evict(
        c, DTYPES[k_pages.dtype], lengths.data_ptr(), new_table.data_ptr(), new_table.shape[1], keep, recent,
        scratch.data_ptr(), n.data_ptr(), st))
    if rc:
        _lib.check(rc, "w4_paged_evict")
    return n
