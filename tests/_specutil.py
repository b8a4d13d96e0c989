"""Plain 64-bit forms of the speculative-decoding operators, written row by row from their
definitions, and the inputs that the tests share."""
import math

import torch

E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def quant_row(x):
    """(codes' values, scale) of one row in 64 bits; (NaN, NaN) for a row that is not finite."""
    x = [float(v) for v in x]
    if not all(math.isfinite(v) for v in x):
        return [math.nan] * len(x), math.nan
    a = max(abs(v) for v in x)
    e = -117
    while a > 448 * 2.0 ** e:
        e += 1
    out = []
    for v in x:
        y = abs(v) / 2.0 ** e
        ulp = 2.0 ** (max(math.frexp(y)[1] - 1, -6) - 3) if y else 1.0
        out.append(math.copysign(round(y / ulp) * ulp, v))   # round(): half to even
    return out, 2.0 ** e


def values(cache, scale):
    v = cache.double()
    return v if scale is None else v * scale.double()[..., None]


def lines(parents, N):
    """Per node the list of its ancestors and itself, empty for an unused one."""
    out = []
    for n in range(N):
        p = n - 1 if parents is None else int(parents[n])
        out.append([n] if p == -1 else out[p] + [n] if 0 <= p < n and out[p] else [])
    return out


def attention64(q, kc, vc, lens, parents, scale, ks, vs):
    """(o, bound): the formula in 64 bits, and how far a bf16 result may be off.

    Scores and sums are held in 32 bits; p is rounded to bf16 before the product with v, and o
    once at the end.  A rounding to bf16 is off by 2^-8 of the value at most, so o by 2^-8
    sum p|v| / l from the first and 2^-8 |o| from the second.  The 32-bit scores are off by at
    most 2^-20 sum |q k| scale (128 products and additions of 2^-24 each, truncation in the
    tensor core included), which enters p as a relative error twice (p and l); exponentials
    and sums add 2^-18 of sum p|v| / l.  Over a quantised cache the weights p * scale may be held
    in f16 instead of bf16: 2^-11 of their value, or half a subnormal step, 2^-25 of the largest
    one, against each code."""
    B, N, Hq, D = q.shape
    H, T = kc.shape[1:3]
    G = Hq // H
    q, k, v = q.double().cpu(), values(kc.cpu(), None if ks is None else ks.cpu()), values(vc.cpu(), None if vs is None else vs.cpu())
    o = torch.zeros(B, N, Hq, D, dtype=torch.float64)
    bound = torch.zeros_like(o)
    for b in range(B):
        m = max(0, min(int(lens[b]), T))
        for n, line in enumerate(lines(None if parents is None else parents[b].tolist(), N)):
            if not line or m + n >= T:
                continue
            rows = list(range(m)) + [m + j for j in line]
            for h in range(Hq):
                kk, vv = k[b, h // G][rows], v[b, h // G][rows]
                x = kk @ q[b, n, h] * scale
                p = torch.softmax(x, 0)
                o[b, n, h] = (p[:, None] * vv).sum(0)
                a = (p[:, None] * vv.abs()).sum(0)
                ds = 2.0 ** -20 * float((kk.abs() @ q[b, n, h].abs()).max()) * abs(scale)
                sub = 0.0
                if vs is not None:
                    sv = vs.cpu()[b, h // G][rows].double()
                    sub = 2.0 ** -25 * float((p * sv).max()) * vc.cpu()[b, h // G][rows].double().abs().sum(0)
                bound[b, n, h] = sub + 2.0 ** -8 * o[b, n, h].abs() + (2.0 ** -8 * 1.01 + 2 * ds + 2.0 ** -18) * a + 2.0 ** -126
    return o, bound


def verify64(tokens, parents, p, q, u):
    """The walk over the tree in 64 bits, one sequence and one node at a time."""
    B, N, V = p.shape
    paths, counts, outs = [], [], []
    for b in range(B):
        pp = p[b].double().cpu()
        qq = None if q is None else q[b].double().cpu()
        cur, path, r, z = 0, [0], pp[0].clone(), 1.0
        while True:
            for n in range(cur + 1, N):
                t = int(tokens[b, n])
                if int(parents[b, n]) != cur or not 0 <= t < V:
                    continue
                had = 1.0 if qq is None else float(qq[cur, t])
                if float(u[b, n]) * had * z < float(r[t]):
                    path.append(n)
                    cur, r, z = n, pp[n].clone(), 1.0
                    break
                if qq is None:
                    r[t] = 0.0
                else:
                    r = (r - z * qq[cur]).clamp_min(0)
                z = float(r.sum())
                if not z > 0:
                    r, z = pp[cur].clone(), 1.0
            else:
                break
        c = r.cumsum(0)
        last = min(int((c <= float(u[b, 0]) * float(c[-1])).sum()), V - 1)
        out = [int(tokens[b, n]) for n in path[1:]] + [last]
        paths.append(path + [-1] * (N - len(path)))
        counts.append(len(path))
        outs.append(out + [-1] * (N - len(out)))
    i32 = dict(dtype=torch.int32)
    return torch.tensor(paths, **i32), torch.tensor(counts, **i32), torch.tensor(outs, **i32)


def make_cache(B, H, T, D, dtype, layout, device, gen):
    """A cache with rows in it (unequal sizes in the quantised form)."""
    from trainium_frontier_b200 import ops
    kc, vc, ks, vs = ops.kv_cache_alloc(B, H, T, D, dtype, layout, device)
    for c, s in ((kc, ks), (vc, vs)):
        x = torch.randn(B, H, T, D, generator=gen)
        if dtype == E4M3:
            raw(c).copy_(raw((x * 40).to(E4M3)))
            raw(s).copy_(torch.randint(120, 124, (B, H, T), generator=gen).to(torch.uint8))
        else:
            c.copy_(x)
    return kc, vc, ks, vs


def make_tree(B, N, gen, unused=False):
    """Random parents a few places back; with `unused`, some nodes (and so their descendants) unused."""
    back = torch.randint(1, 6, (B, N), generator=gen)
    par = (torch.arange(N) - back).clamp_min(0)
    par[:, 0] = -1
    if unused:
        drop = torch.rand(B, N, generator=gen) < 0.2
        par = torch.where(drop, torch.where(torch.rand(B, N, generator=gen) < 0.5, -2, N + 5), par)
    return par.to(torch.int32)


@torch.no_grad()
def quantised_logits(m, text, T):
    """Logits [B, L, V] of a plain model on the CPU for text [B, L], by recomputation: the T tokens of the
    prompt see each other's keys and values as they are, every later token sees all rows, its own
    among them, as an e4m3 cache holds them."""
    from trainium_frontier_b200 import ops
    B, L = text.shape
    cfg = m.config
    H, D = cfg.n_head, cfg.head_dim
    scale = cfg.attn_scale if cfg.attn_scale > 0 else D ** -0.5
    cos, sin = (t.reshape(-1, t.shape[-1])[:L][None, :, None].float() for t in (m.cos, m.sin))
    causal = torch.ones(L, L, dtype=torch.bool).tril()
    x = x0 = ops.embed_norm(text, m.transformer.wte.weight, m.compute_dtype)
    for blk in m.transformer.h:
        xm, h = ops.mix_norm(x, x0, blk.resid_lambda, blk.x0_lambda)
        q, k, v = (t.view(B, L, H, D) for t in ops.linear_multi(h, [blk.attn.c_q.weight, blk.attn.c_k.weight, blk.attn.c_v.weight]).chunk(3, -1))
        q, k = ops.rope_norm(q, cos, sin), ops.rope_norm(k, cos, sin)
        rows = []
        for kk, vv in ((k, v), tuple(ops.ref.cache_values(*ops.ref.quantise_rows(t)) for t in (k, v))):
            w = torch.einsum("bqhd,bkhd->bhqk", q, kk) * scale
            rows.append(torch.einsum("bhqk,bkhd->bqhd", torch.softmax(w.masked_fill(~causal, -math.inf), -1), vv))
        y = torch.cat([rows[0][:, :T], rows[1][:, T:]], 1).reshape(B, L, H * D)
        x = ops.linear(y, blk.attn.c_proj.weight, residual=xm)
        x = blk.mlp(ops.norm(x), residual=x)
    return ops.softcap_logits(ops.norm(x), m.lm_head.weight, m.rc.logit_softcap, cfg.vocab_size)
