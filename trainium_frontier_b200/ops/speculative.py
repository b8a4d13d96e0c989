"""Front-ends of the speculative-decoding kernels (``csrc/kernels/kv_cache.cu``,
``tree_attention.cu``, ``verify_tree.cu``).

One round of speculative decoding over a cache, all in device memory (no host read, so it can
be captured in a CUDA graph):

1. the tree's N tokens (node 0: the last token of the text, not yet in the cache; the others
   drafted) run through the model; each layer appends their keys and values with
   ``kv_cache_write(k, v, ..., pos=lens)`` and attends with ``tree_attention``;
2. ``verify_tree`` takes the target's probabilities after every node, accepts a path and
   draws the token after it;
3. each layer's ``kv_cache_commit`` moves the path's rows up behind the context, and
   ``lens += count``.

Arguments are checked where the kernels are launched; the CPU oracle (``ops.reference``)
makes the same checks through ``check_*`` here.  The reference has no decode path.
"""
from __future__ import annotations

import torch

from ._ext import C, err_word

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
MAX_NODES = 64


def kv_cache_write(k, v, k_cache, v_cache, pos, count, k_scale, v_scale) -> None:
    C().kv_cache_write(k, v, k_cache, v_cache, pos, count, k_scale, v_scale)


def kv_cache_read(k_cache, v_cache, lens, T, k_scale, v_scale):
    return tuple(C().kv_cache_read(k_cache, v_cache, lens, T, k_scale, v_scale))


def kv_cache_commit(k_cache, v_cache, lens, path, count, k_scale, v_scale) -> None:
    C().kv_cache_commit(k_cache, v_cache, lens, path, count, k_scale, v_scale)


def tree_attention(q, k_cache, v_cache, lens, parents, scale, k_scale, v_scale):
    if scale == 0:   # 0 * (q . k): NaN where q . k is infinite, and the masks' -inf stays what it is
        q, scale = q * 0, 1.0
    return C().tree_attention(q, k_cache, v_cache, lens, parents, scale, k_scale, v_scale, err_word(q.device))


def verify_tree(tokens, parents, p, q, u):
    return tuple(C().verify_tree(tokens, parents, p, q, u))


# ------------------------------------------------------------------------------- checks of the CPU oracle
def _check(ok: bool, what: str) -> None:
    if not ok:
        raise RuntimeError(what)


def check_cache(k_cache, v_cache, k_scale, v_scale) -> None:
    _check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride(),
           "k_cache and v_cache: [B, H, T, D] of the same sizes and strides")
    _check(k_cache.dtype == v_cache.dtype and k_cache.device == v_cache.device, "k_cache and v_cache: one type and device")
    quant = k_cache.dtype == E4M3
    _check(quant or k_cache.dtype in (torch.bfloat16, torch.float32), "caches: bfloat16 or float8_e4m3fn (float32 on the CPU)")
    _check(k_cache.shape[3] in (64, 128), "head_dim 64 or 128")
    _check(k_cache.shape[2] >= 1, "cache rows 1 .. 2^30")
    _check(all(st > 0 or n == 1 for st, n in zip(k_cache.stride(), k_cache.shape)) and k_cache.stride(3) == 1,
           "caches: unit inner stride, 16-byte aligned rows, no broadcast dimension")
    _check(quant == (k_scale is not None) == (v_scale is not None),
           "k_scale and v_scale: given with float8_e4m3fn caches, and only with them")
    if quant:
        _check(k_scale.dtype == E8M0 and v_scale.dtype == E8M0 and k_scale.device == k_cache.device
               and v_scale.device == k_cache.device, "scales: float8_e8m0fnu on the caches' device")
        _check(k_scale.shape == k_cache.shape[:3] and v_scale.shape == k_scale.shape and v_scale.stride() == k_scale.stride(),
               "scales: [B, H, T] of the same strides")


def check_scales_written(k_scale) -> None:
    _check(k_scale is None or all(st > 0 or n <= 1 for st, n in zip(k_scale.stride(), k_scale.shape)),
           "scales that are written: no broadcast dimension")


def check_ints(t, name: str, device, *sizes) -> None:
    _check(t.dtype == torch.int32 and t.device == device and tuple(t.shape) == sizes and t.is_contiguous(),
           f"{name}: contiguous int32 of {'[B]' if len(sizes) == 1 else '[B, N]'} entries on the caches' device")


def check_rows(k, v, k_cache) -> None:
    B, H, _, D = k_cache.shape
    for t in (k, v):
        _check(t.dim() == 4 and t.dtype in (torch.bfloat16, torch.float32) and t.device == k_cache.device
               and t.shape == (B, k.shape[1], H, D),
               "k and v: bfloat16 [B, N, H, D] of the caches' B, H, D on their device")
        _check(t.stride(3) == 1, "k and v: unit inner stride and 16-byte aligned rows")


def check_attention(q, k_cache, lens, parents) -> None:
    B, H, _, D = k_cache.shape
    _check(q.dim() == 4 and q.dtype in (torch.bfloat16, torch.float32) and q.device == k_cache.device,
           "q: bfloat16 [B, N, Hq, D] on the caches' device")
    _check(q.shape[0] == B and q.shape[3] == D, "q: the caches' B and D")
    _check(1 <= q.shape[1] <= MAX_NODES, "1 to 64 nodes")
    _check(q.shape[2] >= 1 and H >= 1 and q.shape[2] % H == 0, "the query heads: a multiple of the caches' heads")
    _check(q.stride(3) == 1, "q: unit inner stride and 16-byte aligned rows")
    check_ints(lens, "lens", k_cache.device, B)
    if parents is not None:
        check_ints(parents, "parents", k_cache.device, B, q.shape[1])


def check_verify(tokens, parents, p, q, u) -> None:
    _check(p.dim() == 3 and p.dtype == torch.float32, "p: float32 [B, N, V]")
    B, N, V = p.shape
    _check(1 <= N <= MAX_NODES, "1 to 64 nodes")
    _check(V >= 1, "vocabulary of 1 .. 2^30 tokens")
    for t, name in ((tokens, "tokens"), (parents, "parents")):
        _check(t.dtype == torch.int32 and t.device == p.device and tuple(t.shape) == (B, N) and t.is_contiguous(),
               f"{name}: contiguous int32 [B, N] on p's device")
    _check(u.dtype == torch.float32 and u.device == p.device and tuple(u.shape) == (B, N) and u.is_contiguous(),
           "u: contiguous float32 [B, N] on p's device")
    if q is not None:
        _check(q.dtype == torch.float32 and q.device == p.device and q.shape == p.shape,
               "q: float32 [B, N, V] with unit inner stride on p's device")
