"""Front-ends of packed attention and of the paged cache (``csrc/kernels/packed_attention.cu``,
``paged_cache.cu``, ``paged_attention.cu``).

A batch of prompts of different lengths lies behind one another in one buffer of M rows, sequence s
in rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``: ``packed_attention`` attends inside each of
them, ``paged_cache_write`` stores their keys and values in each sequence's pages, and
``paged_attention`` decodes one token a sequence from there.  Lengths, positions and tables are read
from device memory, so the calls can be captured in a CUDA graph.

Arguments are checked where the kernels are launched; the CPU oracle (``ops.reference``) makes the
same checks through ``check_*`` here.  The reference project has no counterpart.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._ext import C, err_word
from .speculative import _check, check_cache, check_ints, check_scales_written


class PackedAttnFn(Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale):
        out, lse, low = C().packed_attention_fwd(q, k, v, cu_seqlens, scale, True, err_word(q.device))
        ctx.save_for_backward(q, k, v, out, low, lse, cu_seqlens)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, low, lse, cu_seqlens = ctx.saved_tensors
        dq, dk, dv = C().packed_attention_bwd(dout, q, k, v, out, low, lse, cu_seqlens, ctx.scale, err_word(q.device))
        return dq, dk, dv, None, None


def packed_attention(q, k, v, cu_seqlens, scale: float):
    if scale < 0:   # (what is no number, or beyond float32's range, is refused at the launch)
        q, scale = -q, -scale
    elif scale == 0:   # 0 * (q . k): NaN where q . k is infinite, and the mask stays what it is
        q, scale = q * 0, 1.0
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return PackedAttnFn.apply(q, k, v, cu_seqlens, scale)
    return C().packed_attention_fwd(q, k, v, cu_seqlens, scale, False, err_word(q.device))[0]


def paged_cache_write(k, v, k_pages, v_pages, page_table, pos, cu_seqlens, k_scale, v_scale) -> None:
    C().paged_cache_write(k, v, k_pages, v_pages, page_table, pos, cu_seqlens, k_scale, v_scale)


def paged_attention(q, k_pages, v_pages, page_table, lens, scale, k_scale, v_scale):
    return C().paged_attention(q, k_pages, v_pages, page_table, lens, scale, k_scale, v_scale, err_word(q.device))


# ------------------------------------------------------------------------------- checks of the CPU oracle
def check_packed(q, k, v, cu_seqlens) -> None:
    _check(q.dim() == 3 and q.dtype in (torch.bfloat16, torch.float32), "q: bfloat16 [M, Hq, D]")
    _check(k.dim() == 3 and v.dim() == 3, "k and v: bfloat16 [M, Hkv, D]")
    M, Hq, D = q.shape
    _check(D in (64, 128), "head_dim 64 or 128")
    _check(Hq >= 1 and k.shape[1] >= 1 and Hq % k.shape[1] == 0, "the query heads: a multiple of the key/value heads")
    for t, name in ((k, "k"), (v, "v")):
        _check(t.device == q.device and t.dtype == q.dtype and t.shape == (M, k.shape[1], D),
               f"{name}: bfloat16 [M, H, D] of q's M and D on its device")
    _check(cu_seqlens.dtype == torch.int32 and cu_seqlens.device == q.device and cu_seqlens.dim() == 1
           and cu_seqlens.shape[0] >= 1 and cu_seqlens.is_contiguous(), "cu_seqlens: contiguous int32 [S + 1] on q's device")


def check_pages(k_pages, v_pages, page_table, B: int, k_scale, v_scale) -> None:
    check_cache(k_pages, v_pages, k_scale, v_scale)
    page = k_pages.shape[2]
    _check(16 <= page <= 65536 and page & (page - 1) == 0, "pages: a power of two from 16 to 65536 rows")
    _check(page_table.dtype == torch.int32 and page_table.device == k_pages.device and page_table.dim() == 2
           and page_table.shape[0] == B and (page_table.shape[1] <= 1 or page_table.stride(1) == 1),
           "page_table: int32 [B, W] with unit inner stride on the pages' device")
    _check(page_table.shape[1] * page <= 1 << 30, "page_table: at most 2^30 rows a sequence")


def check_paged_write(k, v, k_pages, v_pages, page_table, pos, cu_seqlens, k_scale, v_scale) -> None:
    B = pos.shape[0] if pos.dim() == 1 else -1
    check_pages(k_pages, v_pages, page_table, B, k_scale, v_scale)
    check_scales_written(k_scale)
    check_ints(pos, "pos", k_pages.device, B)
    _check(k.dim() == 3, "k and v: bfloat16 [M, H, D]")
    H, D = k_pages.shape[1], k_pages.shape[3]
    for t in (k, v):
        _check(t.dim() == 3 and t.dtype in (torch.bfloat16, torch.float32) and t.device == k_pages.device
               and t.shape == (k.shape[0], H, D), "k and v: bfloat16 [M, H, D] of the pages' H, D on their device")
        _check(t.stride(2) == 1, "k and v: unit inner stride and 16-byte aligned rows")
    if cu_seqlens is not None:
        check_ints(cu_seqlens, "cu_seqlens", k_pages.device, B + 1)
    else:
        _check(k.shape[0] == B, "without cu_seqlens: one row for each sequence")


def check_paged_attention(q, k_pages, v_pages, page_table, lens, scale, k_scale, v_scale) -> None:
    _check(q.dim() == 3, "q: bfloat16 [B, Hq, D] of the pages' D on their device")
    check_pages(k_pages, v_pages, page_table, q.shape[0], k_scale, v_scale)
    _check(q.dtype in (torch.bfloat16, torch.float32) and q.device == k_pages.device and q.shape[2] == k_pages.shape[3],
           "q: bfloat16 [B, Hq, D] of the pages' D on their device")
    H = k_pages.shape[1]
    _check(q.shape[1] >= 1 and H >= 1 and q.shape[1] % H == 0, "the query heads: a multiple of the pages' heads")
    _check(q.stride(2) == 1, "q: unit inner stride and 16-byte aligned rows")
    _check(math.isfinite(scale), "scale: a finite number")
    check_ints(lens, "lens", k_pages.device, q.shape[0])
