"""fp32 PyTorch oracle of every fused op (the CPU path, and the numerics reference the
GPU tests compare the sm_100a kernels against).

Each function follows the reference's eager op order so a CPU run reproduces the
reference's CPU numerics: ``norm`` = parameter-free ``F.rms_norm`` (train.py:1432-1433),
``apply_rotary_emb`` half-split rotation (train.py:2415-2420), softcap
``S*tanh(z/S)`` then cross-entropy (train.py:2203-2215), relu^2 MLP (train.py:2218-2234).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F


def norm(x: torch.Tensor) -> torch.Tensor:
    return F.rms_norm(x, (x.size(-1),))


def apply_rotary_emb(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    d = x.shape[-1] // 2
    x1, x2 = x[..., :d], x[..., d:]
    y1 = x1 * cos + x2 * sin
    y2 = x1 * (-sin) + x2 * cos
    return torch.cat((y1, y2), dim=-1)


def rope_norm(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    return norm(apply_rotary_emb(x, cos, sin))


def embed_norm(idx: torch.Tensor, wte: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return norm(F.embedding(idx.long(), wte).to(dtype))


def mix_norm(x, x0, resid_lambda, x0_lambda):
    """xm = resid_lambda x + x0_lambda x0 in x's dtype (the shape-[1] fp32 lambdas are cast
    first, so a bf16 residual stream stays bf16 as in the fused kernel; for fp32 inputs this
    is the reference's expression unchanged)."""
    if resid_lambda.dtype != x.dtype:
        resid_lambda, x0_lambda = resid_lambda.to(x.dtype), x0_lambda.to(x.dtype)
    xm = resid_lambda * x + x0_lambda * x0
    return xm, norm(xm)


def linear(x: torch.Tensor, w: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    y = F.linear(x, w.to(x.dtype))
    return y if residual is None else residual + y


def relu_squared(h: torch.Tensor, tau: float = 0.0) -> torch.Tensor:
    if tau != 0.0:
        return F.relu(h - tau).square()
    return F.relu(h).square()


def mlp_relu2(x, w_fc, w_proj, residual=None, tau: float = 0.0):
    y = linear(relu_squared(linear(x, w_fc), tau), w_proj)
    return y if residual is None else residual + y


def attention(q, k, v, causal: bool = True, scale: float | None = None, attn_mask=None):
    """q/k/v as [B, T, H, D]; returns [B, T, H, D]."""
    qt, kt, vt = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
    if attn_mask is None:
        y = F.scaled_dot_product_attention(qt, kt, vt, is_causal=causal, scale=scale)
    else:
        y = F.scaled_dot_product_attention(qt, kt, vt, attn_mask=attn_mask, scale=scale)
    return y.transpose(1, 2)


def causal_conv(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Depthwise causal conv1d over time of x [B, T, C] with w [C, 1, K] (K-1 zeros of left
    padding, the weight cast to x's dtype), train.py:1316-1329."""
    k = w.shape[-1]
    xt = F.pad(x.transpose(1, 2), (k - 1, 0))
    return F.conv1d(xt, w.to(x.dtype), groups=x.shape[-1]).transpose(1, 2)


def ngram_rows(idx: torch.Tensor, order: int, primes, mod: int, pad: int) -> torch.Tensor:
    """Hashed n-gram table rows of every position (train.py:3087-3140): the token and its
    one (bigram) or two (trigram) predecessors, each times a layer prime, XORed, modulo
    the table's prime row count; a missing predecessor is the pad id."""
    cur = idx.long()
    prev = F.pad(cur[:, :-1], (1, 0), value=pad)
    if order == 2:
        h = (prev * primes[0]) ^ (cur * primes[1])
    else:
        prev2 = F.pad(cur[:, :-2], (2, 0), value=pad)
        h = (prev2 * primes[0]) ^ (prev * primes[1]) ^ (cur * primes[2])
    return h % mod


def softcap_logits(x, w_lm, softcap: float, vocab_size: int):
    logits = F.linear(x, w_lm.to(x.dtype))[..., :vocab_size].float()
    return softcap * torch.tanh(logits / softcap)


def softcap_cross_entropy(logits, targets, softcap: float, reduction: str = "mean", weight=None,
                          ignore_index: int = -1):
    capped = softcap * torch.tanh(logits / softcap)
    loss = F.cross_entropy(capped.reshape(-1, capped.size(-1)), targets.reshape(-1).long(),
                           reduction="none" if (weight is not None or reduction == "none") else reduction,
                           ignore_index=ignore_index)
    if weight is not None and reduction == "mean":
        return (loss * weight).sum() / weight.sum()
    if reduction == "none":
        return loss.view(targets.shape)
    return loss


# ------------------------------------------------------------------------- speculative decoding
def quantise_rows(x: torch.Tensor):
    """(e4m3 codes, e8m0 scales [...]) of rows x [..., D]: see ``ops.kv_cache_write``."""
    x = x.float()
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)      # 448 = 0.875 * 2^9
    e = torch.where(amax == 0, -117, e).clamp_min(-117)
    bad = ~torch.isfinite(amax)
    y = torch.ldexp(torch.ldexp(x, -(e // 2)[..., None]), -(e - e // 2)[..., None])
    y = torch.where(e[..., None] == 120, y.clamp(-240, 240), y)           # 256 would be 2^128, which no bf16 is
    codes = torch.where(bad[..., None], 0.0, y).to(torch.float8_e4m3fn)   # the scale says that such a row is NaN
    return codes, torch.where(bad, 255, e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def cache_values(cache: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    """What cached rows stand for, in fp32."""
    return cache.float() if scale is None else cache.float() * scale.float()[..., None]


def _raw(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.uint8) if t.element_size() == 1 else t


def kv_cache_write(k, v, k_cache, v_cache, pos, count=None, k_scale=None, v_scale=None) -> None:
    from . import speculative as sp
    sp.check_cache(k_cache, v_cache, k_scale, v_scale)
    sp.check_scales_written(k_scale)
    sp.check_rows(k, v, k_cache)
    B, N = k.shape[:2]
    sp.check_ints(pos, "pos", k_cache.device, B)
    if count is not None:
        sp.check_ints(count, "count", k_cache.device, B)
    n = torch.arange(N, device=k.device)
    t = pos.long()[:, None] + n
    live = (t >= 0) & (t < k_cache.shape[2])
    if count is not None:
        live &= n < count[:, None]
    b, n = live.nonzero(as_tuple=True)
    t = t[b, n]
    for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        rows = x[b, n]
        if scale is not None:
            rows, codes = quantise_rows(rows)
            _raw(scale)[b, :, t] = _raw(codes)
        _raw(cache)[b, :, t] = _raw(rows.to(cache.dtype))


def kv_cache_read(k_cache, v_cache, lens, T: int, k_scale=None, v_scale=None):
    from . import speculative as sp
    sp.check_cache(k_cache, v_cache, k_scale, v_scale)
    sp.check_ints(lens, "lens", k_cache.device, k_cache.shape[0])
    if not 0 <= T <= k_cache.shape[2]:
        raise RuntimeError("T: 0 .. the cache's rows")
    live = (torch.arange(T, device=k_cache.device) < lens[:, None])[:, :, None, None]
    dt = torch.float32 if k_cache.dtype == torch.float32 else torch.bfloat16
    return tuple(torch.where(live, cache_values(c[:, :, :T], None if s is None else s[:, :, :T]).transpose(1, 2), 0.0)
                 .to(dt).contiguous() for c, s in ((k_cache, k_scale), (v_cache, v_scale)))


def kv_cache_commit(k_cache, v_cache, lens, path, count, k_scale=None, v_scale=None) -> None:
    from . import speculative as sp
    sp.check_cache(k_cache, v_cache, k_scale, v_scale)
    sp.check_scales_written(k_scale)
    B, T = k_cache.shape[0], k_cache.shape[2]
    if path.dim() != 2:
        raise RuntimeError("path: int32 [B, N]")
    N = path.shape[1]
    sp.check_ints(lens, "lens", k_cache.device, B)
    sp.check_ints(path, "path", k_cache.device, B, N)
    sp.check_ints(count, "count", k_cache.device, B)
    i = torch.arange(N, device=path.device)
    src = lens.long()[:, None] + path
    live = (i < count[:, None]) & (path > i) & (path < N) & (lens >= 0)[:, None] & (src < T)
    b, i = live.nonzero(as_tuple=True)
    src, dst = src[b, i], lens.long()[b] + i
    for t in (k_cache, v_cache, k_scale, v_scale):
        if t is not None:
            _raw(t)[b, :, dst] = _raw(t)[b, :, src]


def tree_lines(parents: torch.Tensor | None, B: int, N: int, device) -> torch.Tensor:
    """bool [B, N, N]: node j is node n or one of its ancestors; unused nodes have none."""
    if parents is None:
        return torch.ones(N, N, dtype=torch.bool, device=device).tril().expand(B, N, N)
    line = torch.zeros(B, N, N, dtype=torch.bool, device=device)
    for n in range(N):
        p = parents[:, n].long()
        up = torch.zeros(B, N, dtype=torch.bool, device=device)
        if n:
            up = torch.where(((p >= 0) & (p < n))[:, None], line[torch.arange(B, device=device), p.clamp(0, n - 1)], up)
        line[:, n] = up
        line[:, n, n] = (p == -1) | up.any(-1)
    return line


def tree_attention(q, k_cache, v_cache, lens, parents, scale: float, k_scale=None, v_scale=None):
    from . import speculative as sp
    sp.check_cache(k_cache, v_cache, k_scale, v_scale)
    sp.check_attention(q, k_cache, lens, parents)
    B, N, Hq, D = q.shape
    H, T = k_cache.shape[1:3]
    lens = lens.long().clamp(0, T)
    line = tree_lines(parents, B, N, q.device)
    off = torch.arange(T, device=q.device) - lens[:, None]                      # node of each row, < 0: context
    used = line.any(-1) & (torch.arange(N, device=q.device) < (T - lens)[:, None])
    at = off.clamp(0, N - 1)
    drafted = (off >= 0) & (off < N) & used.gather(1, at)
    sees = (off < 0)[:, None] | (drafted[:, None] & line.gather(2, at[:, None].expand(B, N, T)))
    sees = (sees & used[:, :, None])[:, None, :, None]                          # [B, 1, N, 1, T]
    k = cache_values(k_cache, k_scale)
    # a row that is neither context nor a used node holds anything
    v = torch.where(((off < 0) | drafted)[:, None, :, None], cache_values(v_cache, v_scale), 0.0)
    qg = q.float().unflatten(2, (H, Hq // H)).permute(0, 2, 1, 3, 4)            # [B, H, N, G, D]
    x = torch.einsum("bhngd,bhtd->bhngt", qg, k) * scale
    x = x.masked_fill(~sees, float("-inf"))
    m = x.amax(-1, keepdim=True)
    w = torch.where(sees, torch.exp(x - torch.where(m == float("-inf"), 0.0, m)), 0.0)
    bad = ~torch.isfinite(v)
    o = torch.einsum("bhngt,bhtd->bhngd", w, torch.where(bad, 0.0, v))
    if bool(bad.any()):   # an infinity or a NaN reaches the nodes that see its row, and no other
        s = sees.expand(x.shape).float()
        hit = [torch.einsum("bhngt,bhtd->bhngd", s, f.float()) > 0
               for f in (v == float("inf"), v == float("-inf"), torch.isnan(v))]
        o = o + torch.where(hit[0], float("inf"), 0.0) - torch.where(hit[1], float("inf"), 0.0)
        o = torch.where(hit[2], float("nan"), o)
    o = torch.where(used[:, None, :, None, None], o / w.sum(-1, keepdim=True), 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(B, N, Hq, D).to(q.dtype)


def verify_tree(tokens, parents, p, q, u):
    from . import speculative as sp
    sp.check_verify(tokens, parents, p, q, u)
    B, N, V = p.shape
    dev, f64 = p.device, torch.float64
    at = torch.arange(B, device=dev)
    tokens, parents, u = tokens.long(), parents.long(), u.to(f64)
    path = torch.full((B, N), -1, dtype=torch.long, device=dev)
    path[:, 0] = 0
    cur = torch.zeros(B, dtype=torch.long, device=dev)
    count = torch.ones(B, dtype=torch.long, device=dev)
    one = torch.ones(B, dtype=f64, device=dev)
    r, z = p[:, 0].to(f64), one
    for n in range(1, N):
        t = tokens[:, n].clamp(0, V - 1)
        child = (parents[:, n] == cur) & (tokens[:, n] >= 0) & (tokens[:, n] < V)
        qt = one if q is None else q[at, cur, t].to(f64)
        yes = child & (u[:, n] * qt * z < r[at, t])
        no = child & ~yes
        rest = r.index_put((at, t), torch.zeros_like(z)) if q is None else (r - z[:, None] * q[at, cur].to(f64)).clamp_min(0)
        total = rest.sum(-1)
        empty = ~(total > 0)
        rest = torch.where(empty[:, None], p[at, cur].to(f64), rest)
        total = torch.where(empty, one, total)
        cur = torch.where(yes, n, cur)
        r = torch.where(yes[:, None], p[at, cur].to(f64), torch.where(no[:, None], rest, r))
        z = torch.where(yes, one, torch.where(no, total, z))
        path[at[yes], count[yes]] = n
        count = count + yes
    up = r.cumsum(-1)
    last = (up <= u[:, :1] * up[:, -1:]).sum(-1).clamp_max(V - 1)
    out = torch.full((B, N), -1, dtype=torch.long, device=dev)
    out[:, :-1] = torch.where(path[:, 1:] >= 0, tokens.gather(1, path[:, 1:].clamp_min(0)), -1)
    out[at, count - 1] = last
    return path.to(torch.int32), count.to(torch.int32), out.to(torch.int32)
