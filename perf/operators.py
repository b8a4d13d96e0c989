"""Speculative decoding over a key/value cache: what is measured of the serving operators.

* ``kv_cache_write``  - rows of new keys and values into a cache at each sequence's own
  position, as they are (bf16) or quantised (e4m3 with a power-of-two scale per row);
* ``kv_cache_read``   - the cached rows back as bf16 keys and values;
* ``kv_cache_commit`` - the accepted rows of a drafted tree moved up behind the context;
* ``tree_attention``  - queries of a tree of drafted tokens (or of a single token) against
  the cache: every node sees the context, its ancestors and itself;
* ``verify_tree``     - drafted tokens accepted or rejected against the target's
  probabilities from given uniform numbers, and the token after the accepted path drawn.

``own = False`` computes them in elementary torch operations, ``own = True`` through
``trainium_frontier_b200.ops``.
"""
import math

import torch

own = False

E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of the d20 model at the inference benchmark's batch: 32 sequences, 10 heads
        dict(name="write-step", op="write", b=32, n=1, hq=10, hkv=10, d=128, tmax=2048, kv="e4m3", layout="head"),
        # the prompts of 16 sequences stored after prefill
        dict(name="write-prompts", op="write", b=16, n=4096, hq=32, hkv=8, d=128, tmax=4096, kv="e4m3", layout="head"),
        # a few short, ragged sequences read back for a second prefill over their prefix (d26's 13 heads)
        dict(name="read-short", op="read", b=4, t=577, hkv=13, d=128, tmax=1024, kv="e4m3", layout="token"),
        # long contexts read back
        dict(name="read-long", op="read", b=8, t=16384, hkv=8, d=128, tmax=16384, kv="e4m3", layout="head"),
        # accepted nodes of small trees moved behind their contexts, one layer of d20
        dict(name="commit-step", op="commit", b=32, n=8, hkv=10, d=128, tmax=2048, kv="e4m3", layout="head"),
        # the largest trees at a large batch
        dict(name="commit-large", op="commit", b=256, n=64, hkv=8, d=128, tmax=1024, kv="bf16", layout="head"),
        # single-token decoding at the inference benchmark's batch and length
        dict(name="attn-step", op="attn", b=32, n=1, hq=10, hkv=10, d=128, ctx=575, tmax=2048, kv="bf16",
             layout="head", tree="chain"),
        # one user, a short draft: latency
        dict(name="attn-one", op="attn", b=1, n=6, hq=10, hkv=10, d=64, ctx=1023, tmax=2048, kv="e4m3",
             layout="token", tree="tree"),
        # full trees with shared key/value heads over ragged contexts: 256 rows a key/value head
        dict(name="attn-wide", op="attn", b=16, n=64, hq=32, hkv=8, d=128, ctx=8191, tmax=8320, kv="bf16",
             layout="head", tree="tree"),
        # long ragged contexts in a quantised cache
        dict(name="attn-long", op="attn", b=8, n=24, hq=32, hkv=8, d=128, ctx=65535, tmax=65664, kv="e4m3",
             layout="head", tree="tree"),
        # short drafts over the 8192-token vocabulary
        dict(name="verify-step", op="verify", b=8, n=6, v=8192, q=True, tree="chain"),
        # trees over a large vocabulary at a serving batch
        dict(name="verify-large", op="verify", b=64, n=24, v=131072, q=True, tree="tree"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "commit", "attn", "attn", "attn", "verify", "verify"])
    hkv, g, d = rng.choice([1, 2, 4, 8, 10, 13]), rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([64, 128, 128])
    kv, layout = rng.choice(["e4m3", "e4m3", "bf16"]), rng.choice(["head", "token"])
    tree = rng.choice(["tree", "tree", "chain"])
    if op == "verify":
        v = _log(rng, 257, 131072)
        n = _log(rng, 1, 64)
        b = _log(rng, 1, max(1, min(256, 64 * 24 * 131072 // (n * v))))
        return dict(op=op, b=b, n=n, v=v, q=rng.random() < 0.75, tree=tree)
    if op == "commit":
        b, n = _log(rng, 1, 256), _log(rng, 1, 64)
        tmax = n + _log(rng, 1, max(1, min(4096, 256 * 8 * 1024 * 128 // (b * hkv * d))))
        return dict(op=op, b=b, n=n, hkv=hkv, d=d, tmax=tmax, kv=kv, layout=layout)
    if op in ("write", "read"):
        b = _log(rng, 1, 64)
        t = _log(rng, 1, max(1, min(65536, 16 * 4096 * 8 * 128 // (b * hkv * d))))
        tmax = t + rng.choice([0, 1, 77])
        if op == "read":
            return dict(op=op, b=b, t=t, hkv=hkv, d=d, tmax=tmax, kv=kv, layout=layout)
        return dict(op=op, b=b, n=t, hq=hkv * min(g, 4), hkv=hkv, d=d, tmax=tmax, kv=kv, layout=layout)
    b, n = _log(rng, 1, 64), _log(rng, 1, 64)
    most = min(65535, 8 * 65535 * 8 * 128 // (b * hkv * d), 16 * 8191 * 64 * 32 * 128 // (b * n * hkv * g * d))
    if kv == "bf16":
        most = min(most, 16 * 8191 * 8 * 128 // (b * hkv * d))
    ctx = _log(rng, 1, max(1, most))
    return dict(op=op, b=b, n=n, hq=hkv * g, hkv=hkv, d=d, ctx=ctx, tmax=ctx + n + rng.choice([0, 3, 128]), kv=kv,
                layout=layout, tree=tree)


def _lens(case):
    """Context lengths from ctx down to half of it."""
    b, ctx = case["b"], case["ctx"]
    return [ctx - (ctx // 2) * i // max(1, b - 1) for i in range(b)]


def _read_lens(case):
    b, t = case["b"], case["t"]
    return [t - (t // 4) * i // max(1, b - 1) for i in range(b)]


def _counts(case):
    return [1 + (i * 7919 + case["n"] // 2) % case["n"] for i in range(case["b"])]


def work(case):
    op = case["op"]
    if op == "verify":
        # the rows that the last draw has to read whole: the target's, and the draft's where a child was rejected
        rows = case["b"] * case["v"] * (2 if case["q"] else 1)
        return {"bytes": 4.0 * rows + 16.0 * case["b"] * case["n"], "flops": 2.0 * rows}
    es = 1 if case["kv"] == "e4m3" else 2
    sc = 1 if case["kv"] == "e4m3" else 0
    hkv, d = case["hkv"], case["d"]
    if op == "write":
        rows = 2 * case["b"] * case["n"] * hkv
        return {"bytes": float(rows * (d * (2 + es) + sc)), "flops": 2.0 * rows * d}
    if op == "read":
        got, out = 2 * sum(_read_lens(case)) * hkv, 2 * case["b"] * case["t"] * hkv
        return {"bytes": float(got * (d * es + sc) + out * d * 2), "flops": float(got * d)}
    if op == "commit":
        rows = 2 * sum(c - 1 for c in _counts(case)) * hkv
        return {"bytes": 2.0 * rows * (d * es + sc) + 4.0 * case["b"] * (case["n"] + 2), "flops": 0.0}
    keys = sum(_lens(case)) + case["b"] * case["n"]
    qo = 2 * case["b"] * case["n"] * case["hq"] * d
    return {"bytes": float(2 * keys * hkv * (d * es + sc) + 2 * qo), "flops": 4.0 * keys * case["n"] * case["hq"] * d}


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _parents(case, g):
    b, n = case["b"], case["n"]
    at = torch.arange(n, device="cuda").expand(b, n)
    if case["tree"] == "chain":
        back = torch.ones(b, n, dtype=torch.long, device="cuda")
    else:  # parents a few places back: a few children a node, branches of a few nodes
        back = torch.randint(1, 6, (b, n), device="cuda", generator=g)
    return torch.where(at == 0, -1, (at - back).clamp_min(0)).to(torch.int32).contiguous()


def _cache(case, g):
    """A cache with rows in it: [B, H, T, D] views of head-major or token-major storage."""
    b, h, t, d = case["b"], case["hkv"], case["tmax"], case["d"]
    shape = (b, h, t, d) if case["layout"] == "head" else (b, t, h, d)
    got = []
    for _ in range(2):
        x = torch.randn(shape, device="cuda", dtype=BF16, generator=g)
        if case["kv"] == "e4m3":
            x = (x * 64).to(E4M3)
        got.append(x if case["layout"] == "head" else x.transpose(1, 2))
    if case["kv"] != "e4m3":
        return got + [None, None]
    for _ in range(2):  # rows of unequal sizes, near 2^-6 of their codes
        s = torch.randint(120, 123, shape[:3], device="cuda", dtype=torch.uint8, generator=g).view(E8M0)
        got.append(s if case["layout"] == "head" else s.transpose(1, 2))
    return got


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = {"case": case}
    b = case["b"]
    if op == "verify":
        n, v = case["n"], case["v"]
        z = torch.randn(b, n, v, device="cuda", generator=g) * 2.0
        st["p"] = torch.softmax(z, -1)
        st["parents"] = _parents(case, g)
        up = st["parents"].long().clamp_min(0)
        if case["q"]:
            z += torch.randn(b, n, v, device="cuda", generator=g) * 0.7
            q = torch.softmax(z, -1)
            del z
            rows = q[torch.arange(b, device="cuda")[:, None], up].reshape(b * n, v)
            st["q"] = q
        else:  # drafts that a rule proposes: often one of the target's likely tokens
            del z
            rows = st["p"][torch.arange(b, device="cuda")[:, None], up].reshape(b * n, v) ** 1.5
            st["q"] = None
        st["tokens"] = torch.multinomial(rows, 1, generator=g).view(b, n).to(torch.int32)
        st["u"] = torch.rand(b, n, device="cuda", generator=g)
        return st
    st["kc"], st["vc"], st["ks"], st["vs"] = _cache(case, g)
    mix = torch.randperm(b, device="cuda", generator=g)
    if op == "write":
        # keys and values as slices of a fused projection's rows
        n, hq, h, d = case["n"], case["hq"], case["hkv"], case["d"]
        qkv = torch.randn(b, n, (hq + 2 * h) * d, device="cuda", dtype=BF16, generator=g)
        size = torch.exp(torch.randn(b, n, 1, device="cuda", generator=g)).to(BF16)
        qkv *= size
        st["k"] = qkv[..., hq * d:(hq + h) * d].unflatten(-1, (h, d))
        st["v"] = qkv[..., (hq + h) * d:].unflatten(-1, (h, d))
        st["pos"] = torch.randint(0, case["tmax"] - n + 1, (b,), device="cuda", dtype=torch.int32, generator=g)
        return st
    if op == "read":
        st["lens"] = torch.tensor(_read_lens(case), dtype=torch.int32, device="cuda")[mix].contiguous()
        return st
    n = case["n"]
    if op == "commit":
        st["lens"] = torch.randint(0, case["tmax"] - n + 1, (b,), device="cuda", dtype=torch.int32, generator=g)
        st["count"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")[mix].contiguous()
        order = torch.rand(b, n, device="cuda", generator=g).argsort(-1)
        order = torch.cat([torch.zeros_like(order[:, :1]), order[order != 0].view(b, n - 1)], 1)
        keep = torch.arange(n, device="cuda") < st["count"][:, None]
        path = torch.where(keep, order, n).sort(-1).values
        st["path"] = torch.where(keep, path, -1).to(torch.int32).contiguous()
        return st
    st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[mix].contiguous()
    st["parents"] = _parents(case, g)
    # unit-size rows as a QK norm leaves them, in a projection's layout
    st["q"] = torch.randn(b, n, case["hq"], case["d"], device="cuda", dtype=BF16, generator=g)
    return st


# ------------------------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from trainium_frontier_b200 import ops
        if op == "write":
            ops.kv_cache_write(s["k"], s["v"], s["kc"], s["vc"], s["pos"], None, s["ks"], s["vs"])
            return {k: s[k] for k in ("kc", "vc", "ks", "vs")}
        if op == "read":
            return ops.kv_cache_read(s["kc"], s["vc"], s["lens"], s["case"]["t"], s["ks"], s["vs"])
        if op == "commit":
            ops.kv_cache_commit(s["kc"], s["vc"], s["lens"], s["path"], s["count"], s["ks"], s["vs"])
            return {k: s[k] for k in ("kc", "vc", "ks", "vs")}
        if op == "attn":
            return ops.tree_attention(s["q"], s["kc"], s["vc"], s["lens"], s["parents"], None, s["ks"], s["vs"])
        return ops.verify_tree(s["tokens"], s["parents"], s["p"], s["q"], s["u"])
    return {"write": _write, "read": _read, "commit": _commit, "attn": _attn, "verify": _verify}[op](s)


def _quantise(x):
    """e4m3 codes and e8m0 scales of bf16 rows: the scale is the least power of two (2^-117 at the least) by
    which the row's largest value fits 448; a row with an infinity or a NaN has the scale NaN."""
    x = x.float()
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax == 0, -117, e).clamp_min(-117)
    code = torch.where(torch.isfinite(amax), e + 127, 255).to(torch.uint8).view(E8M0)
    y = torch.ldexp(torch.ldexp(x, -(e // 2)[..., None]), -(e - e // 2)[..., None])
    return y.to(E4M3), code


def _values(codes, scale):
    """What cached rows stand for, in fp32."""
    return codes.float() if scale is None else codes.float() * scale.float()[..., None]


def _u8(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _write(s):
    n = s["k"].shape[1]
    b = torch.arange(s["k"].shape[0], device="cuda")[:, None]
    at = s["pos"].long()[:, None] + torch.arange(n, device="cuda")
    for x, cache, scale in (("k", "kc", "ks"), ("v", "vc", "vs")):
        x = s[x]
        if s[scale] is not None:
            x, code = _quantise(x)
            _u8(s[scale]).transpose(1, 2)[b, at] = _u8(code)
        _u8(s[cache]).transpose(1, 2)[b, at] = _u8(x)
    return {k: s[k] for k in ("kc", "vc", "ks", "vs")}


def _read(s):
    t = s["case"]["t"]
    there = torch.arange(t, device="cuda") < s["lens"][:, None]
    got = []
    for cache, scale in (("kc", "ks"), ("vc", "vs")):
        x = _values(s[cache][:, :, :t], None if s[scale] is None else s[scale][:, :, :t]).transpose(1, 2)
        got.append(torch.where(there[:, :, None, None], x, 0.0).to(BF16).contiguous())
    return tuple(got)


def _commit(s):
    n = s["path"].shape[1]
    i = torch.arange(n, device="cuda")
    b = torch.arange(s["path"].shape[0], device="cuda")[:, None]
    live = i < s["count"][:, None]
    src = s["lens"].long()[:, None] + torch.where(live, s["path"].long(), i)
    dst = s["lens"].long()[:, None] + i
    for name in ("kc", "vc", "ks", "vs"):
        if s[name] is not None:
            rows = _u8(s[name]).transpose(1, 2)
            rows[b, dst] = rows[b, src]
    return {k: s[k] for k in ("kc", "vc", "ks", "vs")}


def _attn(s):
    q, lens, parents = s["q"], s["lens"].long(), s["parents"].long()
    b, n, hq, d = q.shape
    h, t = s["kc"].shape[1], s["kc"].shape[2]
    node = torch.arange(n, device="cuda")
    # reach[i, j]: j is i or one of its ancestors (powers of the identity plus the parent matrix)
    step = (parents[:, :, None] == node).float() + torch.eye(n, device="cuda")
    reach = torch.linalg.matrix_power(step, n) > 0
    off = torch.arange(t, device="cuda") - lens[:, None]
    drafted = (off >= 0) & (off < n)
    sees = torch.gather(reach, 2, off.clamp(0, n - 1)[:, None].expand(b, n, t)) & drafted[:, None]
    sees = (sees | (off < 0)[:, None])[:, None]                                       # [B, 1, N, T]
    k = _values(s["kc"], s["ks"])
    v = torch.where((off < n)[:, None, :, None], _values(s["vc"], s["vs"]), 0.0)     # unused rows hold anything
    qr = q.float().unflatten(2, (h, hq // h)).permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    x = torch.matmul(qr, k.transpose(-1, -2)) * d ** -0.5
    x = x.view(b, h, n, hq // h, t).masked_fill(~sees[:, :, :, None], -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(w.view(b, h, -1, t), v).view(b, h, n, hq // h, d) / w.sum(-1, keepdim=True)
    return o.permute(0, 2, 1, 3, 4).reshape(b, n, hq, d).to(BF16)


def _verify(s):
    tokens, parents, p, q, u = s["tokens"].long(), s["parents"], s["p"], s["q"], s["u"].double()
    b, n, v = p.shape
    at = torch.arange(b, device="cuda")
    cur = torch.zeros(b, dtype=torch.long, device="cuda")
    count = torch.ones(b, dtype=torch.long, device="cuda")
    path = torch.full((b, n), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    left, z = p[:, 0].double(), torch.ones(b, dtype=torch.float64, device="cuda")
    for i in range(1, n):  # a node is tried when its parent is the last accepted one
        child, tok = parents[:, i] == cur, tokens[:, i]
        had = 1.0 if q is None else q[at, cur, tok].double()
        yes = child & (u[:, i] * had * z < left[at, tok])
        no = child & ~yes
        if q is None:
            rest = left.index_put((at, tok), torch.zeros_like(z))
        else:
            rest = (left - z[:, None] * q[at, cur].double()).clamp_min(0)
        total = rest.sum(-1)
        empty = total <= 0
        rest = torch.where(empty[:, None], p[at, cur].double(), rest)
        total = torch.where(empty, torch.ones_like(z), total)
        cur = torch.where(yes, i, cur)
        left = torch.where(yes[:, None], p[at, cur].double(), torch.where(no[:, None], rest, left))
        z = torch.where(yes, torch.ones_like(z), torch.where(no, total, z))
        path[at, count.clamp_max(n - 1)] = torch.where(yes, i, path[at, count.clamp_max(n - 1)])
        count = count + yes
    up = left.cumsum(-1)
    last = (up <= u[:, :1] * up[:, -1:]).sum(-1).clamp_max(v - 1)
    out = torch.cat([torch.where(path >= 0, tokens.gather(1, path.clamp_min(0)), -1)[:, 1:],
                     torch.full((b, 1), -1, dtype=torch.long, device="cuda")], 1)
    out[at, count - 1] = last
    return path.to(torch.int32), count.to(torch.int32), out.to(torch.int32)


# ------------------------------------------------------------------------------- 64 bits
def _e4m3_values(x):
    """(values of the codes, scale) of rows, from the definitions of the two formats, in 64 bits."""
    x = x.double()
    m, e = torch.frexp((x.abs().amax(-1, keepdim=True) / 448).clamp_min(2.0 ** -117))
    e = torch.where(m == 0.5, e - 1, e)                       # the least e with amax <= 448 * 2^e
    y = torch.ldexp(x, -e)
    ulp = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp_min(2.0 ** -6)).exponent - 4)
    return torch.round(y / ulp) * ulp, torch.ldexp(torch.ones_like(m), e)[..., 0]


def exact(case, seed):
    op = case["op"]
    if op == "verify":
        return None  # choices, not computed numbers
    s = prepare(case, seed)
    if op in ("write", "commit"):
        got = {}
        for name, x, scale in (("kc", "k", "ks"), ("vc", "v", "vs"), ("ks", "k", None), ("vs", "v", None)):
            if s[name] is None:
                got[name] = None
                continue
            rows = s[name].transpose(1, 2)
            full = torch.empty(s[name].shape, dtype=torch.float64, device="cuda").transpose(1, 2)
            full.copy_(rows)
            if op == "write":
                new = s[x].double() if s["ks"] is None else _e4m3_values(s[x])[0 if scale else 1]
                for b, at in enumerate(s["pos"].tolist()):
                    full[b, at:at + case["n"]] = new[b]
            else:
                lens, path = s["lens"].tolist(), s["path"].tolist()
                for b, c in enumerate(s["count"].tolist()):
                    old = full[b, lens[b]:lens[b] + case["n"]].clone()
                    full[b, lens[b]:lens[b] + c] = old[path[b][:c]]
            got[name] = full.transpose(1, 2)
        return got
    if op == "read":
        got = []
        for cache, scale in (("kc", "ks"), ("vc", "vs")):
            out = torch.zeros(case["b"], case["t"], case["hkv"], case["d"], dtype=torch.float64, device="cuda")
            for b, m in enumerate(s["lens"].tolist()):
                x = s[cache][b, :, :m].double()
                if s[scale] is not None:
                    x = x * s[scale][b, :, :m].double()[..., None]
                out[b, :m] = x.transpose(0, 1)
            got.append(out)
        return tuple(got)
    n, h, d = case["n"], case["hkv"], case["d"]
    out = torch.empty(case["b"], n, case["hq"], d, dtype=torch.float64, device="cuda")
    for b, (m, up) in enumerate(zip(s["lens"].tolist(), s["parents"].tolist())):
        line = []
        for i in range(n):
            line.append((line[up[i]] if up[i] >= 0 else []) + [i])
        sees = torch.zeros(n, m + n, dtype=torch.bool)
        sees[:, :m] = True
        for i in range(n):
            sees[i, [m + j for j in line[i]]] = True
        k, v = (s[c][b, :, :m + n].double() * (1.0 if s[e] is None else s[e][b, :, :m + n].double()[..., None])
                for c, e in (("kc", "ks"), ("vc", "vs")))
        q = s["q"][b].double().unflatten(1, (h, -1)).transpose(0, 1)            # [h, N, G, D]
        x = torch.einsum("hngd,htd->hngt", q, k) / math.sqrt(d)
        x = x.masked_fill(~sees.cuda()[None, :, None], -math.inf)
        o = torch.einsum("hngt,htd->hngd", torch.softmax(x, -1), v)
        out[b] = o.transpose(0, 1).reshape(n, -1, d)
    return out
