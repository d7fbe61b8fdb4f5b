"""Log probabilities of given tokens, the entropy of their distributions and the most
likely alternatives, in one pass over the logits (csrc/w4_logprobs.hip)."""
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
