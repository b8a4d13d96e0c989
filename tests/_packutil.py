"""Plain 64-bit forms of packed attention, the paged cache and token log probabilities, with bounds on
how far a result may be off, and the inputs that the tests share.

Roundings: to bf16 2^-8 of the value at most, to f16 2^-11, to fp32 2^-24."""
import math

import torch

E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def values(cache, scale):
    v = cache.double()
    return v if scale is None else v * scale.double()[..., None]


def pack(lens, hq, hkv, d, device, seed=0, pad=0, dtype=BF16, fill=0.0):
    """(q, k, v, cu, dout) of sequences behind one another, q / k / v slices of one projection's rows; the
    pad rows hold `fill`."""
    g = torch.Generator().manual_seed(seed)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    M = cu[-1] + pad
    qkv = torch.randn(M, (hq + 2 * hkv) * d, generator=g).to(dtype)
    do = torch.randn(M, hq, d, generator=g).to(dtype)
    qkv[cu[-1]:] = fill
    do[cu[-1]:] = fill
    qkv, do = qkv.to(device), do.to(device)
    q, k, v = qkv[:, :hq * d].unflatten(-1, (hq, d)), qkv[:, hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d)), qkv[:, (hq + hkv) * d:].unflatten(-1, (hkv, d))
    return q, k, v, torch.tensor(cu, dtype=torch.int32, device=device), do


def packed64(q, k, v, cu, scale, do=None):
    """{name: (value, bound)} of the output and, with `do`, the gradients.

    The output: scores in 32 bits are off by at most 2^-20 sum |q k| scale (128 products and sums of 2^-24
    each, truncation in the tensor core included); an exponential by 2^-13.6 of its value (7.5e-5, the
    polynomial's; the unit's own are better), and both enter twice (p and the sum).  p is rounded to bf16
    before the product with v, the output once at the end.
    Gradients: p as above, rounded to bf16 for dV; D = dO . o is of the rounded output, so off by
    |dO| . (the output's bound); ds = p (dP - D) from p rounded to bf16, rounded to bf16 itself; each gradient
    is rounded once at the end."""
    M, Hq, d = q.shape
    H = k.shape[1]
    g = Hq // H
    f = dict(dtype=torch.float64, device=q.device)
    res = {n: (torch.zeros(t.shape, **f), torch.zeros(t.shape, **f)) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    r8, e, tiny = 2.0 ** -8, 2.0 ** -13.6, 2.0 ** -120
    cu = cu.tolist()
    for a, b in zip(cu[:-1], cu[1:]):
        if b <= a:
            continue
        see = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).tril()
        for h in range(Hq):
            qq, kk, vv = q[a:b, h].double(), k[a:b, h // g].double(), v[a:b, h // g].double()
            x = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            ds_rel = 2 * (2.0 ** -20 * (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~see, 0).amax(-1, keepdim=True) + e)
            p = torch.softmax(x, -1)
            o = p @ vv
            ob = r8 * o.abs() + (p * (r8 * 1.01 + ds_rel)) @ vv.abs() + tiny
            res["o"][0][a:b, h], res["o"][1][a:b, h] = o, ob
            if do is None:
                continue
            dd = do[a:b, h].double()
            res["dv"][0][a:b, h // g] += p.T @ dd
            res["dv"][1][a:b, h // g] += (p * (r8 * 1.01 + ds_rel)).T @ dd.abs()
            dp = dd @ vv.T
            D = (dd * o).sum(-1, keepdim=True)
            t = (dp - D) * see
            s = p * t
            sb = p * ((2.02 * r8 + ds_rel) * t.abs() + 2.0 ** -20 * (dd.abs() @ vv.abs().T) + (dd.abs() * (ob * 1.02 + 2.0 ** -18 * o.abs())).sum(-1, keepdim=True)) * see
            res["dq"][0][a:b, h] = s @ kk * scale
            res["dq"][1][a:b, h] = sb @ kk.abs() * abs(scale)
            res["dk"][0][a:b, h // g] += s.T @ qq * scale
            res["dk"][1][a:b, h // g] += sb.T @ qq.abs() * abs(scale)
    for n in ("dq", "dk", "dv"):
        res[n][1].add_(r8 * 1.01 * res[n][0].abs() + tiny)
    return res


def make_pages(P, H, page, D, dtype, layout, device, seed=0):
    """Pages with rows in them (unequal scales in the quantised form)."""
    from trainium_frontier_b200 import ops
    gen = torch.Generator().manual_seed(seed)
    kp, vp, ks, vs = ops.kv_cache_alloc(P, H, page, D, dtype, layout, device)
    for c, s in ((kp, ks), (vp, vs)):
        x = torch.randn(P, H, page, D, generator=gen)
        if dtype == E4M3:
            raw(c).copy_(raw((x * 40).to(E4M3)))
            raw(s).copy_(torch.randint(120, 124, (P, H, page), generator=gen).to(torch.uint8))
        else:
            c.copy_(x)
    return kp, vp, ks, vs


def make_table(B, W, P, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    assert B * W <= P
    return torch.randperm(P, generator=g)[:B * W].view(B, W).to(torch.int32).to(device)


def rows_of(pages, scale, table_row, n):
    """Rows [H, n', D] that a sequence of n rows sees, in 64 bits."""
    P, _, page, _ = pages.shape
    got = []
    for t in range(n):
        p = int(table_row[t // page])
        if 0 <= p < P:
            got.append(values(pages[p, :, t % page], None if scale is None else scale[p, :, t % page]))
    return torch.stack(got, 1) if got else None


def paged64(q, kp, vp, table, lens, scale, ks, vs):
    """(o, bound); as `packed64`'s output, and over quantised pages the weights p * scale are held in f16:
    2^-11 of their value, or half a subnormal step, 2^-25 of the largest one, against each code."""
    B, Hq, D = q.shape
    H, page = kp.shape[1:3]
    cpu = [None if t is None else t.cpu() for t in (kp, vp, ks, vs)]
    o = torch.zeros(B, Hq, D, dtype=torch.float64)
    bound = torch.zeros_like(o)
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * page))
        kk, vv = (rows_of(c, s, table[b].tolist(), n) for c, s in ((cpu[0], cpu[2]), (cpu[1], cpu[3])))
        if kk is None:
            continue
        for h in range(Hq):
            k, v, qq = kk[h // (Hq // H)], vv[h // (Hq // H)], q[b, h].double().cpu()
            p = torch.softmax(k @ qq * scale, 0)
            o[b, h] = p @ v
            ds = 2.0 ** -20 * float((k.abs() @ qq.abs()).max()) * abs(scale)
            sub = 0.0
            if vs is not None:
                sc = rows_of(cpu[3][..., None], None, table[b].tolist(), n)[h // (Hq // H)][:, 0].nan_to_num(0.0)   # the rows' scales
                sub = 2.0 ** -25 * float((p * sc).nan_to_num(0.0).max()) * (v / sc.clamp_min(2.0 ** -140)[:, None]).nan_to_num(0.0).abs().sum(0)
            bound[b, h] = sub + 2.0 ** -8 * o[b, h].abs() + (p * (2.0 ** -8 * 1.01 + 2 * ds + 2.0 ** -18)) @ v.abs() + 2.0 ** -120
    return o, bound


def scores64(z, tokens, top, g=None, h=None):
    """{name: (value, bound)}.  Exponentials are off by 2^-21 + 2^-23 |z - m| of their value (the unit's 2^-22 and
    the rounded argument), the sums of up to 2^17 of them by 2^-18 (64 in a row, then by halves);
    a logarithm and a difference by 2^-23 of their values."""
    z = z.double()
    V = z.shape[-1]
    m = z.amax(-1, keepdim=True)
    log_sum = torch.log((z - m).exp().sum(-1, keepdim=True))
    l = z - m - log_sum
    p = l.exp()
    far = (p * (z - m).clamp_min(-1e4).abs()).sum(-1)
    es = 2.0 ** -18 + 2.0 ** -21 + 2.0 ** -23 * far
    t = tokens.long()
    there = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1)[..., None]
    lp = torch.where(there, l.gather(-1, at)[..., 0], 0.0)
    zm = torch.where(there, (z - m).gather(-1, at)[..., 0].abs(), 0.0)
    ent = -torch.where(p == 0, 0.0, p * l).sum(-1)
    far2 = (p * (z - m).clamp_min(-1e4) ** 2).sum(-1)
    eb = es * (1 + far) + 2.0 ** -17 * far + 2.0 ** -22 * far2 + 2.0 ** -22
    key = torch.sort(z, dim=-1, descending=True, stable=True)
    tops = key.values[..., :top] - m - log_sum
    out = {"logprob": (lp, es + 2.0 ** -22 * (zm + lp.abs()) + 2.0 ** -22), "entropy": (ent, eb),
           "top_tokens": (key.indices[..., :top].to(torch.int32), None),
           "top_logprobs": (tops, es[..., None] + 2.0 ** -22 * 2 * tops.abs() + 2.0 ** -22)}
    if g is not None:
        one = torch.zeros_like(z).scatter_(-1, at, 1.0) * there[..., None]
        gg, hh = torch.where(there, g.double(), 0.0)[..., None], h.double()[..., None]
        lc = torch.where(p == 0, 0.0, l)
        dz = one * gg - p * (gg + hh * (lc + ent[..., None]))
        rel = 2.0 ** -20 + es[..., None] + 2.0 ** -22 * lc.abs()
        b = p * (rel * (gg.abs() + hh.abs() * (lc.abs() + ent[..., None] + 1)) + hh.abs() * (eb + es)[..., None])
        out["dlogits"] = (dz, b + 2.0 ** -23 * (one * gg).abs() + 2.0 ** -120)
    return out


def close(got, want, bound, what=""):
    """|got - want| <= bound, entry by entry; entries of `want` that are no number have to be the same in `got`."""
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.cpu()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN at other places"
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what + ": infinities"
    off = torch.where(odd, 0.0, (got - want).abs() - bound)
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: off by {float((got - want)[~odd].abs().max()):.3e}, {float(off.max()):.3e} above the bound"
