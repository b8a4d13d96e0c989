"""Speculative decoding for the plain GPT family (new: the reference has no generation path).

``SpeculativeGenerator(model, max_batch, max_len).generate(prompts, n)`` runs the target once a
round over a small tree of tokens -- the last token of the text and the tokens that a draft
proposes behind it -- and keeps the path that the target agrees with (``ops.verify_tree``), at
least one new token a round.  The text's law is that of one token a round over the same cache:
sampling draws from the same distribution, and greedy decoding over an unquantised cache gives
the tokens of plain greedy decoding.

Keys and values live in a cache with a length of its own for every sequence, as bfloat16 or
quantised to ``float8_e4m3fn`` with a power-of-two scale per row (half the memory): each layer
writes the tree's rows behind the context (``ops.kv_cache_write``), attends to context and
ancestors (``ops.tree_attention``) and, once a path is accepted, moves its rows up
(``ops.kv_cache_commit``).

Everything goes through the public ops, so a model on the CPU runs the fp32 oracle.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .. import ops
from .generate import _is_plain


def ngram_draft(n: int, order: int = 2):
    """A draft by rule: the n tokens that followed the latest earlier occurrence of the text's
    last ``order`` tokens, as a chain; nothing where there is none."""
    def draft(text: torch.Tensor, lens: torch.Tensor):
        B, L = text.shape
        at = torch.arange(L, device=text.device)
        ln = lens.long()[:, None]
        hit = (at + order < ln) & (at + order <= L - 1)
        for k in range(order):   # text[i + k] == text[len - order + k]
            last = text.gather(1, (ln - order + k).clamp_min(0))
            hit = hit & (torch.roll(text, -k, 1) == last)
        i = torch.where(hit & (ln >= order), at, -1).amax(1, keepdim=True)
        src = i + order + torch.arange(n, device=text.device)
        ok = (i >= 0) & (src < ln)
        tok = torch.where(ok, text.gather(1, src.clamp(0, L - 1)), -1).to(torch.int32)
        par = torch.where(ok, torch.arange(n, device=text.device), -2).to(torch.int32)
        return tok, par, None
    return draft


class SpeculativeGenerator:
    """``draft(text [B, max_len] int64, lens [B] int32) -> (tokens [B, n] int32, parents [B, n]
    int32, q)`` proposes n < 64 nodes: node i of the draft is node i + 1 of the tree, whose node
    0 is the text's last token, and ``parents`` are tree nodes (-2: unused).  A token outside the
    vocabulary is never accepted.  ``q`` [B, n + 1, V]
    holds the distributions that the children of each tree node were drawn from, or is None for
    a rule (``ops.verify_tree``)."""

    def __init__(self, model, max_batch: int, max_len: int, draft=None, kv_dtype: torch.dtype | None = None):
        if not _is_plain(model):
            raise NotImplementedError("the cached decoder serves the plain member of the family; "
                                      "use generate_reference for the others")
        if max_len > model.config.sequence_len:
            raise ValueError(f"max_len {max_len} exceeds the model's sequence length {model.config.sequence_len}")
        self.m = model
        cfg = model.config
        self.dev = model.get_device()
        self.H, self.D, self.V = cfg.n_head, cfg.head_dim, cfg.vocab_size
        self.scale = cfg.attn_scale if cfg.attn_scale > 0 else self.D ** -0.5
        self.B, self.max_len = max_batch, max_len
        self.draft = draft or ngram_draft(7)
        dt = kv_dtype or model.compute_dtype
        rows = max_len + 64   # a tree begins before max_len, and its last nodes may be the accepted ones
        self.caches = [ops.kv_cache_alloc(max_batch, self.H, rows, self.D, dt, device=self.dev)
                       for _ in range(cfg.n_layer)]
        self.rounds = 0

    # ------------------------------------------------------------------ the model over new tokens
    def _hidden(self, idx: torch.Tensor, pos: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor | None, prompt: bool):
        """Final normed states of tokens idx [B, N] at positions pos [B, N]; their keys and values
        go into the caches at row lens.  ``prompt``: causal attention among the tokens alone."""
        m, (B, N) = self.m, idx.shape
        cos, sin = (t.reshape(-1, t.shape[-1])[pos.reshape(-1)][None, :, None] for t in (m.cos, m.sin))
        x = x0 = ops.embed_norm(idx, m.transformer.wte.weight, m.compute_dtype)
        rows = (1, B * N, self.H, self.D)
        for blk, (kc, vc, ks, vs) in zip(m.transformer.h, self.caches):
            xm, h = ops.mix_norm(x, x0, blk.resid_lambda, blk.x0_lambda)
            q, k, v = ops.linear_multi(h, [blk.attn.c_q.weight, blk.attn.c_k.weight, blk.attn.c_v.weight]).chunk(3, -1)
            q = ops.rope_norm(q.reshape(rows), cos, sin).view(B, N, self.H, self.D)
            k = ops.rope_norm(k.reshape(rows), cos, sin).view(B, N, self.H, self.D)
            v = v.unflatten(-1, (self.H, self.D))
            ops.kv_cache_write(k, v, kc, vc, lens, None, ks, vs)
            if prompt:
                y = self._causal(q, k, v)
            else:
                y = ops.tree_attention(q, kc, vc, lens, parents, self.scale, ks, vs)
            x = ops.linear(y.reshape(B, N, -1), blk.attn.c_proj.weight, residual=xm)
            x = blk.mlp(ops.norm(x), residual=x)
        return ops.norm(x)

    def _causal(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Causal attention of a prompt of any length: the kernel takes whole tiles of 128 rows, and no
        row sees the ones that fill up the last tile."""
        T = q.shape[1]
        if q.is_cuda and T % 128:
            q, k, v = (F.pad(t, (0, 0, 0, 0, 0, -T % 128)) for t in (q, k, v))
        return ops.attention(q, k, v.contiguous(), True, self.scale)[:, :T]

    def _probabilities(self, hidden: torch.Tensor, temperature: float) -> torch.Tensor:
        z = ops.softcap_logits(hidden, self.m.lm_head.weight, self.m.rc.logit_softcap, self.V)
        if temperature == 0.0:   # greedy: all mass on the largest logit
            return torch.zeros_like(z).scatter_(-1, z.argmax(-1, keepdim=True), 1.0)
        return torch.softmax(z / temperature, -1)

    # ------------------------------------------------------------------ generation
    @torch.no_grad()
    def generate(self, prompts: torch.Tensor, max_new_tokens: int, temperature: float = 0.0,
                 generator: torch.Generator | None = None) -> torch.Tensor:
        """New tokens [B, max_new_tokens] (int32).  ``temperature`` 0 is greedy; otherwise the
        softcapped logits over it are sampled with ``generator``'s numbers.  ``self.rounds``
        counts the target's passes after the prompt."""
        B, T = prompts.shape
        if B != self.B:
            raise ValueError("a generator is built for a fixed batch")
        if T < 1 or max_new_tokens < 1 or T + max_new_tokens > self.max_len:
            raise ValueError(f"prompt and new tokens must fit in max_len {self.max_len}")
        if int(prompts.min()) < 0 or int(prompts.max()) >= self.V:   # they index the embedding
            raise ValueError(f"prompts: tokens 0 .. {self.V - 1}")
        dev = self.dev
        uniform = lambda *s: torch.rand(*s, device=dev, generator=generator)  # noqa: E731
        text = torch.zeros(B, self.max_len, dtype=torch.long, device=dev)
        text[:, :T] = prompts.to(dev)
        zero = torch.zeros(B, dtype=torch.int32, device=dev)
        at = torch.arange(T, device=dev).expand(B, T)
        hidden = self._hidden(text[:, :T].to(torch.int32).contiguous(), at, zero, None, True)[:, -1:]
        root = torch.full((B, 1), -1, dtype=torch.int32, device=dev)
        _, _, first = ops.verify_tree(root, root, self._probabilities(hidden.contiguous(), temperature), None, uniform(B, 1))
        text[:, T] = first[:, 0].long()
        cached = zero + T                 # rows of context in the caches; the text has one token more
        end, self.rounds = T + max_new_tokens, 0
        b = torch.arange(B, device=dev)[:, None]
        while bool((cached + 1 < end).any()):
            tok, par, q = self.draft(text, cached + 1)
            N = tok.shape[1] + 1
            tokens = torch.cat([text.gather(1, cached.long()[:, None]).to(torch.int32), tok], 1)
            parents = torch.cat([root, par], 1).contiguous()
            depth = ops.ref.tree_lines(parents, B, N, dev).sum(-1) - 1
            pos = (cached.long()[:, None] + depth).clamp(0, self.max_len - 1)
            hidden = self._hidden(tokens.clamp(0, self.V - 1), pos, cached, parents, False)
            path, count, out = ops.verify_tree(tokens, parents, self._probabilities(hidden, temperature), q, uniform(B, N))
            count = torch.minimum(count, (end - 1 - cached).clamp_min(0))   # a finished sequence stays as it is
            for kc, vc, ks, vs in self.caches:
                ops.kv_cache_commit(kc, vc, cached, path, count, ks, vs)
            i = torch.arange(N, device=dev)
            dst = torch.where(i < count[:, None], cached.long()[:, None] + 1 + i, self.max_len)
            text = torch.cat([text, text[:, :1]], 1)                         # one column for what is not taken
            text[b, dst] = out.long()
            text = text[:, :self.max_len].contiguous()
            cached = cached + count
            self.rounds += 1
        return text[:, T:end].to(torch.int32)
