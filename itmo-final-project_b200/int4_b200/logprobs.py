"""Log probabilities of given tokens, with each row's entropy and most probable tokens.

The reference scores text by the cross entropy of the whole vocabulary (``eval_ppl``,
``benchmarks/eval_llama.py:77-117``); a serving program returns the same numbers with each answer.
"""
from __future__ import annotations

import torch

from . import _lib

MAX_TOP = 32  # I4B_MAX_TOP


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0):
    """``(logprobs, entropy, top_logprobs, top_ids)`` of the rows ``logits[..., V]`` (bf16, fp16 or float32).

    ``logprobs[...]``: log softmax at ``targets[...]`` (int64; a negative target is padding and gives 0, one past the
    vocabulary a NaN).  ``entropy[...]``: -sum p log p.  ``top_logprobs`` / ``top_ids`` ``[..., top]``: the ``top``
    largest logits of each row in order, ties to the lower index (None when ``top`` is 0; at most 32).  float32,
    ids int64.  -inf logits have probability 0; a row of nothing else has log probabilities -inf and entropy 0; a NaN
    or +inf makes the row's numbers NaN.  The logits are read once, on the current stream; no backward pass.
    Logits that are not rows one stride apart (``x[:, :-1]`` of a batch) or whose last dimension is strided are copied
    first."""
    if logits.dtype not in _lib.DTYPE_CODE or logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be [..., vocabulary] in bfloat16, float16 or float32")
    lead, V = logits.shape[:-1], logits.shape[-1]
    if targets.dtype != torch.int64 or targets.shape != lead:
        raise ValueError(f"targets must be int64 of shape {tuple(lead)}")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top {top}: 0 to {min(MAX_TOP, V)} alternatives of {V} tokens")
    dev = logits.device
    if dev.type != "cuda" or targets.device != dev:
        raise ValueError("int4_b200 computes on the GPU only: logits and targets must be CUDA tensors of one device")
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if V > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < 0:
        x = x.contiguous()
    targets = targets.contiguous()
    lp = torch.empty_like(targets, dtype=torch.float32)
    entropy = torch.empty_like(lp)
    top_lp = lp.new_empty((*lead, top)) if top else None
    top_ids = targets.new_empty((*lead, top)) if top else None
    with _lib.on_device(dev):
        st = _lib.lib().i4b_token_logprobs(x.data_ptr(), _lib.DTYPE_CODE[x.dtype], x.shape[0], V, x.stride(0),
                                           targets.data_ptr(), top, lp.data_ptr(), entropy.data_ptr(),
                                           top_lp.data_ptr() if top else None, top_ids.data_ptr() if top else None,
                                           _lib.stream_handle(dev))
    _lib.check(st, "token_logprobs")
    return lp, entropy, top_lp, top_ids
