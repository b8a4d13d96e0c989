"""Front-end of ``csrc/kernels/token_logprobs.cu``: log probabilities of given tokens, entropies and
likeliest alternatives of logits.  The reference project has no counterpart."""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._ext import C
from .speculative import _check

MAX_TOP = 32


class TokenLogprobsFn(Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        lp, ent, tok, top_lp, stat = C().token_logprobs(logits, tokens, top, True)
        ctx.save_for_backward(logits, tokens, stat)
        ctx.mark_non_differentiable(tok, top_lp)
        ctx.set_materialize_grads(False)
        return lp, ent, tok, top_lp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlp, dent, *_):
        logits, tokens, stat = ctx.saved_tensors
        g, h = (None if t is None else t.contiguous() for t in (dlp, dent))
        if g is None and h is None:
            return None, None, None
        return C().token_logprobs_grad(logits, tokens, stat, g, h), None, None


def token_logprobs(logits, tokens, top: int):
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobsFn.apply(logits, tokens, top)
    return C().token_logprobs(logits, tokens, top, False)[:4]


def check_logprobs(logits, tokens, top: int):
    """(shape of the tokens, vocabulary), or the reason why the arguments do not fit (the CPU oracle's; the kernel's call
    makes the same checks)."""
    _check(logits.dim() >= 1 and logits.dtype in (torch.float32, torch.bfloat16), "logits: float32 or bfloat16 [..., V]")
    shape, V = logits.shape[:-1], logits.shape[-1]
    _check(1 <= V <= 1 << 30, "vocabulary of 1 .. 2^30 tokens")
    _check(V == 1 or logits.stride(-1) == 1, "logits: unit inner stride")
    _check(tokens.dtype in (torch.int64, torch.int32) and tokens.device == logits.device and tokens.shape == shape,
           "tokens: int64 or int32, one for each row of the logits, on their device")
    _check(0 <= top <= min(MAX_TOP, V), "top: 0 .. 32 alternatives, at most the vocabulary")
    return shape, V
