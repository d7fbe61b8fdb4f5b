"""Log probabilities of given tokens, the entropy of their distributions and the most
likely alternatives, in one pass over the logits (csrc/w4_logprobs.hip); verification of
drafted tokens against the target's probabilities (csrc/w4_verify.hip)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .gemm import _with_workspace
from .llama_ops import _on, underived

DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor | None  # fp32 [rows]: log softmax at the given tokens
    entropy: torch.Tensor         # fp32 [rows], in nats
    top_logprob: torch.Tensor     # fp32 [rows, top]
    top_token: torch.Tensor       # int64 [rows, top], the most likely first


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None, top: int = 0) -> TokenLogprobs:
    """Log probabilities (log softmax, fp32) of ``tokens`` int64 [rows] (or None) under
    ``logits`` [rows, vocab] (bf16, fp16 or fp32), the entropies, and the ``top`` (at
    most 64) most likely tokens with theirs: the lower index first among equal logits,
    so that ``top_token[:, 0]`` is the greedy choice.

    A token outside the vocabulary has log probability NaN, as has a whole row without a
    finite maximum (all -inf, a +inf or a NaN among its logits).  Launches on the current
    stream; no part in autograd.
    """
    if _lib.ext is not None:  # plain operands: the same call without Python's share of its cost
        r = _lib.ext.token_logprobs(logits, tokens, top)
        if r is not None:
            return TokenLogprobs(*r)
    assert logits.dtype in DTYPES and logits.dim() == 2 and logits.is_cuda, (logits.dtype, logits.shape)
    assert underived(logits), \
        "token_logprobs has no derivatives: call it under torch.no_grad(), on logits without tangents"
    logits = logits.resolve_neg()
    R, V = logits.shape
    dev = logits.device
    assert V >= 1 and 0 <= top <= min(MAX_TOP, V), (V, top)
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    logprob = None
    if tokens is not None:
        assert tokens.dtype == torch.int64 and tokens.shape == (R,) and tokens.device == dev, tokens.shape
        tokens = tokens.resolve_neg().contiguous()
        logprob = torch.empty(R, device=dev)
    entropy = torch.empty(R, device=dev)
    top_logprob = torch.empty((R, top), device=dev)
    top_token = torch.empty((R, top), dtype=torch.int64, device=dev)
    lib = _lib.load()
    nbytes = lib.w4_token_logprobs_workspace_bytes(R, V, top)
    rc = _on(dev, lambda st: _with_workspace(dev, st, nbytes, lambda ws, nb: lib.w4_token_logprobs(
        logits.data_ptr(), DTYPES[logits.dtype], R, V, logits.stride(0),
        None if tokens is None else tokens.data_ptr(), top, None if logprob is None else logprob.data_ptr(),
        entropy.data_ptr(), top_logprob.data_ptr(), top_token.data_ptr(), ws, nb, st)))
    if rc:
        _lib.check(rc, "w4_token_logprobs")
    return TokenLogprobs(logprob, entropy, top_logprob, top_token)


class Verified(NamedTuple):
    accepted: torch.Tensor  # int64 [rows]: how many of a row's drafts are accepted
    token: torch.Tensor     # int64 [rows]: the token after them


MAX_DRAFTS = 64


def drafts_fit(shape, dtype, dev, draft, tokens, accept, sample, counts=None) -> None:
    """Asserts what ``verify_drafts`` needs beside target probabilities of ``shape``, ``dtype`` and
    device ``dev``, so that a caller can ask before it computes them."""
    B, K, V = shape[0], shape[1] - 1, shape[2]
    assert underived(draft, accept, sample), \
        "verify_drafts has no derivatives: call it under torch.no_grad(), on probabilities without tangents"
    assert 0 <= K <= MAX_DRAFTS and V >= 1, shape
    assert tokens.dtype == torch.int64 and tokens.shape == (B, K) and tokens.device == dev, (tokens.dtype, tokens.shape)
    assert accept.dtype == sample.dtype == torch.float32 and accept.shape == (B, K) and sample.shape == (B,)
    assert accept.device == sample.device == dev
    if draft is not None:
        assert draft.dtype == dtype and draft.shape == (B, K, V) and draft.device == dev, (draft.dtype, draft.shape)
    if counts is not None:
        assert counts.dtype == torch.int32 and counts.shape == (B,) and counts.device == dev, counts.shape


def verify_drafts(target: torch.Tensor, draft: torch.Tensor | None, tokens: torch.Tensor, accept: torch.Tensor,
                  sample: torch.Tensor, counts: torch.Tensor | None = None) -> Verified:
    """Speculative sampling: which of the drafted ``tokens`` int64 [rows, drafts] (at most 64)
    stay, and the token that follows, distributed as the target's own samples are.

    ``target`` [rows, drafts + 1, vocab] has the target's probabilities before, between and
    after the drafts, ``draft`` [rows, drafts, vocab] those that they were drawn from (None:
    they were no matter of chance, as the greedy choice of a smaller model); both bf16, fp16
    or fp32.  Draft i stays where the ones before do and ``accept[b, i]`` * draft < target
    at it.  The next token is drawn with ``sample[b]`` from max(target - draft, 0) at the
    first that does not stay (from the target where that is 0 throughout, and after the last
    draft): the least token whose weights up to it pass ``sample[b]`` times their sum.
    ``accept`` fp32 [rows, drafts] and ``sample`` fp32 [rows] are uniform in [0, 1); with
    ``counts`` int32 [rows] a row has so many drafts only (outside 0..drafts: none of its
    results is a number of tokens, both are -1).

    A draft outside the vocabulary does not stay.  Negative weights count as 0; weights whose
    sum is 0, infinite or NaN have no token: -1.  Products, differences and sums are taken in
    64 bits.  Launches on the current stream; no part in autograd.
    """
    if _lib.ext is not None:
        r = _lib.ext.verify_drafts(target, draft, tokens, accept, sample, counts)
        if r is not None:
            return Verified(*r)
    assert target.dtype in DTYPES and target.dim() == 3 and target.is_cuda, (target.dtype, target.shape)
    assert underived(target), \
        "verify_drafts has no derivatives: call it under torch.no_grad(), on probabilities without tangents"
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    dev = target.device
    drafts_fit(target.shape, target.dtype, dev, draft, tokens, accept, sample, counts)
    target, tokens, accept, sample = (t.resolve_neg() for t in (target, tokens, accept, sample))
    tokens, accept, sample = tokens.contiguous(), accept.contiguous(), sample.contiguous()
    if target.stride(2) != 1 and V > 1:
        target = target.contiguous()
    if draft is not None:
        draft = draft.resolve_neg()
        if draft.stride(2) != 1 and V > 1:
            draft = draft.contiguous()
    if counts is not None:
        counts = counts.resolve_neg().contiguous()
    accepted, token = (torch.empty(B, dtype=torch.int64, device=dev) for _ in range(2))
    lib = _lib.load()
    nbytes = lib.w4_verify_drafts_workspace_bytes(B, V)
    at = None if draft is None or K == 0 else draft.data_ptr()
    rc = _on(dev, lambda st: _with_workspace(dev, st, nbytes, lambda ws, nb: lib.w4_verify_drafts(
        target.data_ptr(), at, DTYPES[target.dtype], B, K, V, target.stride(0), target.stride(1),
        0 if at is None else draft.stride(0), 0 if at is None else draft.stride(1), tokens.data_ptr(),
        None if counts is None else counts.data_ptr(), accept.data_ptr(), sample.data_ptr(), accepted.data_ptr(),
        token.data_ptr(), ws, nb, st)))
    if rc:
        _lib.check(rc, "w4_verify_drafts")
    return Verified(accepted, token)
