"""Batched decoding of prompts of different lengths for the plain GPT family, with or without shared
key/value heads (new: the reference has no generation path).

``PagedGenerator(model, max_batch, max_len).generate(prompts, n)``: the prompts lie behind one
another in one buffer and run through the model once (``ops.packed_attention``); their keys and
values go into pages that each sequence holds as many of as it needs (``ops.paged_cache_write``),
bfloat16 or quantised to ``float8_e4m3fn``; then every sequence decodes a token a step over its pages
(``ops.paged_attention``).  Each new token comes with its log probability, and on request the
likeliest alternatives (``ops.token_logprobs``).

Everything goes through the public ops, so a model on the CPU runs the fp32 oracle.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import ops
from .generate import _is_plain


class Generation(NamedTuple):
    """``tokens`` [B, n] int32 and their log probabilities [B, n]; the likeliest alternatives at each place,
    ``top_tokens`` [B, n, top] int32 with ``top_logprobs``; ``entropy`` [B, n] of the distributions in nats."""
    tokens: torch.Tensor
    logprobs: torch.Tensor
    top_tokens: torch.Tensor
    top_logprobs: torch.Tensor
    entropy: torch.Tensor


class PagedGenerator:
    """``pages`` (default: enough for ``max_batch`` sequences of ``max_len``) pages of ``page`` rows are
    shared by the sequences of a batch."""

    def __init__(self, model, max_batch: int, max_len: int, page: int = 16, pages: int | None = None,
                 kv_dtype: torch.dtype | None = None):
        if not _is_plain(model, shared_heads=True):
            raise NotImplementedError("the paged decoder serves the plain member of the family, with or without shared "
                                      "key/value heads; use generate_reference for the others")
        if max_len > model.config.sequence_len:
            raise ValueError(f"max_len {max_len} exceeds the model's sequence length {model.config.sequence_len}")
        self.m = model
        cfg = model.config
        self.dev = model.get_device()
        self.H, self.Hkv, self.D, self.V = cfg.n_head, cfg.n_kv_heads or cfg.n_head, cfg.head_dim, cfg.vocab_size
        self.scale = cfg.attn_scale if cfg.attn_scale > 0 else self.D ** -0.5
        self.B, self.max_len, self.page = max_batch, max_len, page
        self.pages = pages if pages is not None else max_batch * (-(-max_len // page))
        dt = kv_dtype or model.compute_dtype
        self.caches = [ops.kv_cache_alloc(self.pages, self.Hkv, page, self.D, dt, device=self.dev) for _ in range(cfg.n_layer)]

    # ------------------------------------------------------------------ the model over new tokens
    def _hidden(self, idx: torch.Tensor, at: torch.Tensor, table: torch.Tensor, pos: torch.Tensor, cu: torch.Tensor | None):
        """Final normed states [M, C] of tokens idx [M] at positions at [M], stored behind row pos of their
        sequences: prompts cut by cu, or (None) one token a sequence."""
        m, M = self.m, idx.shape[0]
        cos, sin = (t.reshape(-1, t.shape[-1])[at][None, :, None] for t in (m.cos, m.sin))
        x = x0 = ops.embed_norm(idx[None], m.transformer.wte.weight, m.compute_dtype)
        split = (self.H * self.D, self.Hkv * self.D, self.Hkv * self.D)
        for blk, (kp, vp, ks, vs) in zip(m.transformer.h, self.caches):
            xm, h = ops.mix_norm(x, x0, blk.resid_lambda, blk.x0_lambda)
            q, k, v = ops.linear_multi(h, [blk.attn.c_q.weight, blk.attn.c_k.weight, blk.attn.c_v.weight]).split(split, -1)
            q = ops.rope_norm(q.reshape(1, M, self.H, self.D), cos, sin)[0]
            k = ops.rope_norm(k.reshape(1, M, self.Hkv, self.D), cos, sin)[0]
            v = v[0].unflatten(-1, (self.Hkv, self.D))
            ops.paged_cache_write(k, v, kp, vp, table, pos, cu, ks, vs)
            if cu is not None:
                y = ops.packed_attention(q, k, v, cu, self.scale)
            else:
                y = ops.paged_attention(q, kp, vp, table, pos + 1, self.scale, ks, vs)
            x = ops.linear(y.reshape(1, M, -1), blk.attn.c_proj.weight, residual=xm)
            x = blk.mlp(ops.norm(x), residual=x)
        return ops.norm(x)[0]

    def _next(self, hidden: torch.Tensor, temperature: float, top: int, generator):
        """The tokens drawn after hidden [B, C] and their scores under the model's own distribution."""
        z = ops.softcap_logits(hidden, self.m.lm_head.weight, self.m.rc.logit_softcap, self.V)
        if temperature == 0.0:
            tok = z.argmax(-1)
        else:
            # Relative to the row's maximum, so that no temperature makes an infinity of a logit (the least one: a normal number
            # of float32).  A row with a NaN has none but NaN probabilities, which a draw answers with a device-side
            # assertion: its token is drawn from all alike, and its log probability says NaN.
            p = torch.softmax((z - z.amax(-1, keepdim=True)) / max(temperature, 2.0 ** -126), -1)
            tok = torch.multinomial(p.masked_fill(torch.isnan(p), 1.0), 1, generator=generator)[:, 0]
        return (tok, *ops.token_logprobs(z, tok, top))

    # ------------------------------------------------------------------ generation
    @torch.no_grad()
    def generate(self, prompts, max_new_tokens: int, temperature: float = 0.0, top: int = 0,
                 generator: torch.Generator | None = None) -> Generation:
        """``prompts``: a list of 1-D tensors of tokens.  ``temperature`` 0 is greedy; otherwise the softcapped
        logits over it are sampled with ``generator``'s numbers.  Log probabilities are those of temperature 1; where a
        model's logits hold a NaN they are NaN, and the token is any."""
        prompts = [torch.as_tensor(p) for p in prompts]
        lens = [int(p.numel()) for p in prompts]
        if not 1 <= len(prompts) <= self.B:
            raise ValueError(f"1 .. {self.B} prompts")
        if min(lens) < 1 or max_new_tokens < 1 or max(lens) + max_new_tokens > self.max_len or any(p.dim() != 1 for p in prompts):
            raise ValueError(f"prompts: 1-D, not empty, and with the new tokens at most {self.max_len} tokens")
        if any(p.is_floating_point() or p.is_complex() or p.dtype == torch.bool for p in prompts):
            raise ValueError("prompts: tokens are integers")
        if not 0 <= top <= min(32, self.V):
            raise ValueError("top: 0 .. 32 alternatives, at most the vocabulary")
        if not temperature >= 0:
            raise ValueError("temperature: 0 (greedy) or above")
        text = torch.cat([p.to(self.dev) for p in prompts])
        if int(text.min()) < 0 or int(text.max()) >= self.V:   # they index the embedding
            raise ValueError(f"prompts: tokens 0 .. {self.V - 1}")
        need = [-(-(n + max_new_tokens) // self.page) for n in lens]
        if sum(need) > self.pages:
            raise ValueError(f"the batch needs {sum(need)} pages of {self.pages}")
        B, dev = len(prompts), self.dev
        table = torch.full((B, max(need)), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n)
        table = table.to(dev)
        cut = torch.tensor([0] + lens).cumsum(0)
        at = torch.cat([torch.arange(n) for n in lens]).to(dev)
        cu, pos = cut.to(torch.int32).to(dev), torch.zeros(B, dtype=torch.int32, device=dev)
        hidden = self._hidden(text.to(torch.int32).contiguous(), at, table, pos, cu)[(cut[1:] - 1).to(dev)]
        pos = pos + torch.tensor(lens, dtype=torch.int32, device=dev)
        steps = []
        for i in range(max_new_tokens):
            if i:
                hidden = self._hidden(steps[-1][0].to(torch.int32), pos.long(), table, pos, None)
                pos = pos + 1
            steps.append(self._next(hidden, temperature, top, generator))
        tok, lp, ent, alt, alt_lp = (torch.stack(t, 1) for t in zip(*steps))
        return Generation(tok.to(torch.int32), lp, alt, alt_lp, ent)
