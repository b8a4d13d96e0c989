"""Public op surface of the framework.

Every op has two implementations selected by the device of its inputs:
* CUDA tensors -> the hand-written sm_100a kernels (``ops.fused`` over ``_C``); the
  extension is required there and its absence raises.
* CPU tensors  -> the fp32 PyTorch oracle in ``ops.reference`` (reference op order),
  which is also what the GPU numerics tests compare against.

``oracle_mode()`` routes CUDA tensors through the oracle as well (library GEMMs, SDPA,
eager elementwise ops in the compute dtype): the bf16 library comparator of the
benchmark runs the same model and engine that way.  It is a measurement switch, never
the training path.
"""
from __future__ import annotations

import contextlib
import os

import torch

from . import reference as ref

_ORACLE = [False]


@contextlib.contextmanager
def oracle_mode(on: bool = True):
    """Within the block, every op (and the optimizer's kernel paths) uses the PyTorch
    oracle on any device."""
    prev = _ORACLE[0]
    _ORACLE[0] = bool(on)
    try:
        yield
    finally:
        _ORACLE[0] = prev


def oracle_active() -> bool:
    return _ORACLE[0]


def _cuda(t: torch.Tensor) -> bool:
    return t.is_cuda and not _ORACLE[0]


def norm(x: torch.Tensor) -> torch.Tensor:
    if _cuda(x):
        from .fused import RMSNormFn
        return RMSNormFn.apply(x)
    return ref.norm(x)


rms_norm = norm


def embed_norm(idx: torch.Tensor, wte: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if _cuda(wte) and dtype == torch.bfloat16 and wte.dtype == torch.float32:
        from .fused import EmbedNormFn
        return EmbedNormFn.apply(idx, wte)
    return ref.embed_norm(idx, wte, dtype)


def mix_norm(x, x0, resid_lambda, x0_lambda):
    """(xm, norm(xm)) with xm = resid_lambda * x + x0_lambda * x0."""
    if _cuda(x) and x.dtype == torch.bfloat16 and x0.dtype == torch.bfloat16:
        from .fused import MixNormFn
        return MixNormFn.apply(x, x0, resid_lambda, x0_lambda)
    return ref.mix_norm(x, x0, resid_lambda, x0_lambda)


def linear(x: torch.Tensor, w: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    if _cuda(x) and x.dtype == torch.bfloat16:
        from .fused import LinearFn
        return LinearFn.apply(x, w, residual)
    return ref.linear(x, w, residual)


def linear_multi(x: torch.Tensor, ws: list[torch.Tensor]) -> torch.Tensor:
    """x @ cat(ws)^T as one GEMM (outputs concatenated on the last dim)."""
    if _cuda(x) and x.dtype == torch.bfloat16:
        from .fused import LinearMultiFn
        return LinearMultiFn.apply(x, *ws)
    return torch.cat([ref.linear(x, w) for w in ws], dim=-1)


def mlp_relu2(x, w_fc, w_proj, residual=None, tau: float = 0.0):
    if _cuda(x) and x.dtype == torch.bfloat16:
        from .fused import MLPRelu2Fn
        return MLPRelu2Fn.apply(x, w_fc, w_proj, residual, float(tau))
    return ref.mlp_relu2(x, w_fc, w_proj, residual, tau)


def rope_norm(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """norm(apply_rotary_emb(x)) for x [B, T, H, D]; cos/sin [1, T, 1, D/2]."""
    if _cuda(x) and x.dtype == torch.bfloat16:
        from .fused import RopeNormFn
        T = x.shape[1]
        c2 = cos.reshape(-1, cos.shape[-1])[:T].contiguous()
        s2 = sin.reshape(-1, sin.shape[-1])[:T].contiguous()
        return RopeNormFn.apply(x, c2, s2, 0)
    return ref.rope_norm(x, cos, sin)


def attention(q, k, v, causal: bool = True, scale: float | None = None, attn_mask=None):
    """q, k, v [B, T, H, D] -> [B, T, H, D].  CUDA: tcgen05 flash attention (causal or
    full, T % 128 == 0, head_dim 64 / 128); additive masks (document / sliding-window
    variants of the family) use the reference composition."""
    if _cuda(q) and q.dtype == torch.bfloat16 and attn_mask is None:
        from .flash_attention import FlashAttnFn, supported
        B, T, H, D = q.shape
        if supported(T, D):
            return FlashAttnFn.apply(q, k, v, causal, scale if scale is not None else D ** -0.5)
    return ref.attention(q, k, v, causal, scale, attn_mask)


def attention_qkv(qkv: torch.Tensor, cos, sin, n_head: int, head_dim: int, scale: float | None):
    """Plain-block attention core from the fused projection [B, T, 3C]:
    RoPE + QK-norm on q, k, then causal attention.  Returns [B, T, C]."""
    B, T, C3 = qkv.shape
    from .flash_attention import supported
    if _cuda(qkv) and qkv.dtype == torch.bfloat16 and supported(T, head_dim):
        from .fused import AttnQKVFn
        c2 = cos.reshape(-1, cos.shape[-1])[:T].contiguous()
        s2 = sin.reshape(-1, sin.shape[-1])[:T].contiguous()
        sc = scale if scale is not None else head_dim ** -0.5
        return AttnQKVFn.apply(qkv, c2, s2, B, T, n_head, head_dim, sc)
    Cd = C3 // 3
    q, k, v = qkv.split(Cd, dim=-1)
    q = ref.rope_norm(q.view(B, T, n_head, head_dim), cos, sin)
    k = ref.rope_norm(k.view(B, T, n_head, head_dim), cos, sin)
    y = ref.attention(q, k, v.view(B, T, n_head, head_dim), True, scale)
    return y.reshape(B, T, Cd)


def qkv_attention(x: torch.Tensor, ws: list[torch.Tensor], cos, sin, n_head: int, head_dim: int,
                  scale: float | None):
    """Plain-block attention from the block input x [B, T, C] and the q / k / v weights:
    projection, RoPE + QK-norm on q and k, causal attention.  Returns [B, T, C].  On CUDA
    with heads of 128 the RoPE + QK-norm runs in the projection GEMM's epilogue
    (``TFB_QKV_ROPE=0`` makes it a separate kernel after the projection)."""
    B, T, _ = x.shape
    if _cuda(x) and x.dtype == torch.bfloat16 and os.environ.get("TFB_QKV_ROPE", "1") != "0":
        from .fused import QKVRopeAttnFn, qkv_rope_supported
        if qkv_rope_supported(T, n_head, head_dim):
            c2 = cos.reshape(-1, cos.shape[-1])[:T].contiguous()
            s2 = sin.reshape(-1, sin.shape[-1])[:T].contiguous()
            sc = scale if scale is not None else head_dim ** -0.5
            return QKVRopeAttnFn.apply(x, c2, s2, B, T, n_head, head_dim, sc, *ws)
    return attention_qkv(linear_multi(x, ws), cos, sin, n_head, head_dim, scale)


def causal_conv(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Depthwise causal conv1d over time: x [B, T, C], w [C, 1, K]."""
    if _cuda(x) and x.dtype == torch.bfloat16 and w.dtype == torch.float32 and x.shape[-1] % 8 == 0 \
            and w.shape[-1] <= 8:
        from .fused import CausalConvFn
        return CausalConvFn.apply(x, w)
    return ref.causal_conv(x, w)


def ngram_lookup(idx: torch.Tensor, table: torch.Tensor, order: int, primes, mod: int, pad: int,
                 dtype: torch.dtype) -> torch.Tensor:
    """Rows of a hashed n-gram table for every position of idx [B, T] (see
    ``reference.ngram_rows``), cast to ``dtype``: [B, T, Dn].  On CUDA the hash and the
    gather are one kernel and the backward scatters into the fp32 table gradient."""
    if _cuda(table) and table.dtype == torch.float32 and dtype == torch.bfloat16 and table.shape[1] % 4 == 0:
        from .fused import NgramLookupFn
        return NgramLookupFn.apply(idx, table, int(order), tuple(int(p) for p in primes), int(mod), int(pad))
    return table[ref.ngram_rows(idx, order, primes, mod, pad)].to(dtype)


def lm_head_softcap_ce(x, w_lm, targets, softcap: float, vocab: int, reduction: str = "mean",
                       row_weight=None):
    """Fused lm_head GEMM + softcap + cross-entropy (+ its backward)."""
    if _cuda(x) and x.dtype == torch.bfloat16:
        from .fused import LMHeadSoftcapCEFn, softcap_ce_rows
        if reduction == "none":
            return softcap_ce_rows(x, w_lm, targets, softcap, vocab)
        return LMHeadSoftcapCEFn.apply(x, w_lm, targets, softcap, vocab, row_weight, reduction)
    logits = ref.linear(x, w_lm)[..., :vocab].float()
    return ref.softcap_cross_entropy(logits, targets, softcap, reduction,
                                     None if row_weight is None else row_weight.reshape(-1))


def softcap_logits(x, w_lm, softcap: float, vocab: int):
    if _cuda(x) and x.dtype == torch.bfloat16:
        from .fused import softcap_logits as f
        return f(x, w_lm, softcap, vocab)
    return ref.softcap_logits(x, w_lm, softcap, vocab)


def kv_cache_alloc(batch: int, heads: int, rows: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                   layout: str = "head", device=None):
    """(k_cache, v_cache, k_scale, v_scale) for ``heads`` key/value heads and ``rows`` rows a
    sequence: zeroed [B, H, T, D] views of head-major (``layout="head"``, [B, H, T, D]) or
    token-major (``"token"``, [B, T, H, D]) storage.  ``dtype`` ``float8_e4m3fn`` makes a
    quantised cache, whose scales are ``float8_e8m0fnu`` [B, H, T]; else the scales are None."""
    if layout not in ("head", "token"):
        raise ValueError("layout: 'head' or 'token'")
    shape = (batch, heads, rows, head_dim) if layout == "head" else (batch, rows, heads, head_dim)
    quant = dtype == torch.float8_e4m3fn

    def make(sizes, dt):
        t = torch.zeros(sizes, dtype=torch.uint8 if dt.itemsize == 1 else dt, device=device)
        t = t.view(dt)
        return t if layout == "head" else t.transpose(1, 2)
    return (make(shape, dtype), make(shape, dtype),
            make(shape[:3], torch.float8_e8m0fnu) if quant else None,
            make(shape[:3], torch.float8_e8m0fnu) if quant else None)


def kv_cache_write(k, v, k_cache, v_cache, pos, count=None, k_scale=None, v_scale=None) -> None:
    """Rows k, v [B, N, H, D] into the caches [B, H, T, D] (any strides with a unit inner one):
    row n of sequence b goes to row ``pos[b] + n`` for ``n < count[b]`` (default: all N); rows
    that fall outside the cache are left out, and every other row stays as it is.  ``pos`` and
    ``count`` are int32 [B] in device memory.

    ``float8_e4m3fn`` caches hold each row's codes ``x * 2^-e`` rounded to nearest even and its
    scale ``2^e`` (``float8_e8m0fnu`` [B, H, T], a byte of its own for every row), ``e`` being the
    least integer (-117 at the least) with ``max|x| <= 448 * 2^e``; a row with an infinity or a NaN
    reads back as NaN.
    A value that would round to ``2^128``, which is no bfloat16, is held as ``1.875 * 2^127``.
    CUDA: k, v bfloat16 with 16-byte aligned rows, head_dim 64 / 128."""
    if _cuda(k_cache):
        from .speculative import kv_cache_write as f
        return f(k, v, k_cache, v_cache, pos, count, k_scale, v_scale)
    return ref.kv_cache_write(k, v, k_cache, v_cache, pos, count, k_scale, v_scale)


def kv_cache_read(k_cache, v_cache, lens, T: int, k_scale=None, v_scale=None):
    """The caches' first T rows as keys and values [B, T, H, D] (bfloat16; float32 for float32
    caches on the CPU), zeros from row ``lens[b]`` (int32 [B]) on.  Quantised rows read back
    exactly: every value they can hold is a bfloat16 number.  ``k.view(B * T, H * D)`` is a row
    view as ``flash_attention.flash_fwd`` takes it."""
    if _cuda(k_cache):
        from .speculative import kv_cache_read as f
        return f(k_cache, v_cache, lens, T, k_scale, v_scale)
    return ref.kv_cache_read(k_cache, v_cache, lens, T, k_scale, v_scale)


def kv_cache_commit(k_cache, v_cache, lens, path, count, k_scale=None, v_scale=None) -> None:
    """Moves the accepted rows of a drafted tree up behind the context, in place: row
    ``lens[b] + path[b, i]`` becomes row ``lens[b] + i`` for ``i < count[b]``, with its scale.
    ``path`` int32 [B, N] is ascending over those entries, as ``verify_tree`` returns it;
    ``lens`` and ``count`` int32 [B].  The caller advances ``lens`` by ``count``."""
    if _cuda(k_cache):
        from .speculative import kv_cache_commit as f
        return f(k_cache, v_cache, lens, path, count, k_scale, v_scale)
    return ref.kv_cache_commit(k_cache, v_cache, lens, path, count, k_scale, v_scale)


def tree_attention(q, k_cache, v_cache, lens, parents=None, scale: float | None = None, k_scale=None, v_scale=None):
    """Attention of N <= 64 new tokens a sequence over a cache that holds ``lens[b]`` rows of
    context and, behind them, the N tokens' own rows (``kv_cache_write`` at ``pos = lens``).
    q [B, N, Hq, D], caches [B, Hkv, T, D] with Hkv dividing Hq (query head h reads head
    ``h // (Hq // Hkv)``); returns [B, N, Hq, D].

    ``parents`` int32 [B, N]: node n sees the context, its ancestors and itself; -1 marks a
    child of the context, other parents are earlier nodes.  None: a chain (node n - 1 is node
    n's parent), so N = 1 is a plain decode step.  A node whose line of parents meets any other
    value is unused (the padding of a smaller tree: -2), as is one whose own row lies past the
    cache; its output is zero, and what its row holds reaches no other node.  ``scale`` defaults
    to D^-0.5.  An infinity or a NaN in a row (in e4m3: a NaN code, or the scale NaN) reaches every
    node that sees it; where all scores that a node sees are -inf its output is NaN.  Weights are
    rounded to bfloat16 for the product with the values, or, for few rows over a quantised cache, to
    float16 relative to the largest weight times scale, below 2^-25 of which a row may count nothing.
    No gradient."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if _cuda(k_cache):
        from .speculative import tree_attention as f
        return f(q, k_cache, v_cache, lens, parents, scale, k_scale, v_scale)
    return ref.tree_attention(q, k_cache, v_cache, lens, parents, scale, k_scale, v_scale)


def verify_tree(tokens, parents, p, q, u):
    """Speculative sampling over a tree of N <= 64 nodes: which drafted tokens are accepted, and
    the token after them.  Returns int32 ``(path [B, N], count [B], out [B, N])``: the accepted
    nodes in ascending order from node 0 (padded with -1), how many they are, and the tokens
    they add to the text -- those of ``path[1:]``, then the drawn one at ``count - 1`` (padded
    with -1).

    Node 0 is the root and always accepted; ``parents`` int32 [B, N] as in ``tree_attention``.
    p (float32 [B, N, V]) holds the target's distribution of the token after each node, q the
    distribution from which each node's children were drawn independently, or None for drafts
    that a rule proposed.  From the root on, the children n of the last accepted node c are
    tried in order with a remainder r (at first p[c], its sum counted as Z = 1): n is accepted
    iff ``u[n] * q[c, t] * Z < r[t]`` (t = tokens[n]; q None: q[c, t] = 1); otherwise ``r <-
    max(r - Z q[c], 0)`` (q None: ``r[t] <- 0``) and ``Z <- sum r``, or r and Z start again at
    p[c] and 1 if nothing is left.  When no child is left the next token is the least j with
    ``r[0] + ... + r[j] > u[0] * sum r``.  u float32 [B, N] uniform in [0, 1).  Nodes with a
    token outside the vocabulary are no node's children.  All arithmetic is in 64 bits."""
    if _cuda(p):
        from .speculative import verify_tree as f
        return f(tokens, parents, p, q, u)
    return ref.verify_tree(tokens, parents, p, q, u)
