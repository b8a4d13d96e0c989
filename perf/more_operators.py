"""Prompts packed behind one another, decoded over a paged key/value cache and scored: what is
measured of these operators.

* ``packed_attention``   - causal attention over sequences of different lengths that lie behind one
  another in one buffer, with shared key/value heads; forward (prompts) and with its gradients
  (documents of a training batch);
* ``paged_cache_write``  - rows of new keys and values into the pages of each sequence, as they are
  (bf16) or quantised (e4m3 with a power-of-two scale per row);
* ``paged_attention``    - one new token of every sequence against its pages;
* ``token_logprobs``     - the log probability of a given token, the entropy and the likeliest
  alternatives of every row of logits, and the gradient of the first two.

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
        # a few short user prompts, d20's heads: latency
        dict(name="prompts-short", op="packed", s=8, t=100, mix="prompts", pad=0, hq=10, hkv=10, d=128),
        # the prompts of a serving batch with shared key/value heads
        dict(name="prompts-long", op="packed", s=16, t=8191, mix="prompts", pad=0, hq=32, hkv=8, d=128),
        # one layer of a d20 training batch, attention inside documents: 192 documents in some 65,000 tokens
        dict(name="train-documents", op="train", s=192, t=1024, mix="documents", pad=64, hq=10, hkv=10, d=128),
        # long documents with shared key/value heads
        dict(name="train-long", op="train", s=4, t=8192, mix="prompts", pad=0, hq=32, hkv=8, d=128),
        # one decode step at the inference benchmark's batch and length (d20)
        dict(name="paged-step", op="paged", b=32, hq=10, hkv=10, d=128, ctx=576, page=16, kv="bf16", layout="head"),
        # one user with a long context
        dict(name="paged-one", op="paged", b=1, hq=32, hkv=8, d=128, ctx=131071, page=64, kv="bf16", layout="head"),
        # a serving batch of long ragged contexts in a quantised cache
        dict(name="paged-batch", op="paged", b=64, hq=32, hkv=8, d=128, ctx=16384, page=16, kv="e4m3", layout="head"),
        # the new token of 32 sequences stored, one layer of d20
        dict(name="write-step", op="write", s=32, t=1, hq=10, hkv=10, d=128, page=16, kv="e4m3", layout="head"),
        # the prompts of 16 sequences stored after prefill
        dict(name="write-prompts", op="write", s=16, t=4096, hq=32, hkv=8, d=128, page=16, kv="bf16", layout="head"),
        # a decode step's logits over a large vocabulary: the chosen token's log probability and eight alternatives
        dict(name="score-step", op="score", n=8, v=131072, top=8, kind="fp32", grad=False),
        # held-out text scored over the 8192-token vocabulary, five alternatives a token
        dict(name="score-text", op="score", n=16384, v=8192, top=5, kind="fp32", grad=False),
        # log probabilities with an entropy term and their gradient, over a large vocabulary
        dict(name="score-train", op="score", n=4096, v=131072, top=0, kind="bf16", grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "train", "train", "paged", "paged", "paged", "write", "score", "score"])
    hkv, g, d = rng.choice([1, 2, 4, 8, 10, 13]), rng.choice([1, 1, 2, 3, 4, 8]), rng.choice([64, 128, 128])
    kv, layout, page = rng.choice(["bf16", "e4m3"]), rng.choice(["head", "head", "token"]), rng.choice([16, 16, 32, 64, 128, 256])
    if op == "score":
        v, grad = _log(rng, 257, 131072), rng.random() < 0.4
        n = _log(rng, 1, max(1, min(16384, 2 ** 27 // v)))
        return dict(op=op, n=n, v=v, top=rng.choice([0, 1, 5, 20, 32]), kind=rng.choice(["fp32", "bf16"]), grad=grad)
    if op == "paged":
        b = _log(rng, 1, 256)
        ctx = _log(rng, 1, max(1, min(131072, 64 * 12288 * 8 * 128 // (b * hkv * d) // (1 if kv == "e4m3" else 2))))
        return dict(op=op, b=b, hq=hkv * g, hkv=hkv, d=d, ctx=ctx, page=page, kv=kv, layout=layout)
    if op == "write":
        s = _log(rng, 1, 64)
        t = _log(rng, 1, max(1, min(16384, 16 * 4096 * 8 * 128 // (s * hkv * d))))
        return dict(op=op, s=s, t=t, hq=hkv * min(g, 4), hkv=hkv, d=d, page=page, kv=kv, layout=layout)
    s, mix = _log(rng, 1, 128), rng.choice(["prompts", "documents"])
    # rows and products below the largest listed cases'
    most = min(16384, 131072 * 16 * 128 // (s * hkv * g * d), math.isqrt(16 * 6144 ** 2 * 32 * 128 // (s * hkv * g * d) // (4 if op == "train" else 1)))
    return dict(op=op, s=s, t=_log(rng, 1, max(1, most)), mix=mix, pad=rng.choice([0, 0, 5, 100]), hq=hkv * g, hkv=hkv, d=d)


def _lens(case):
    """Tokens of every sequence, the longest of t (ctx in a cache)."""
    if case["op"] == "paged":
        b, t = case["b"], case["ctx"]
        return [t - (t // 2) * i // max(1, b - 1) for i in range(b)]
    s, t = case["s"], case["t"]
    if case["op"] == "write" or case["mix"] == "prompts":
        return [t - (t // 2) * i // max(1, s - 1) for i in range(s)]
    return [max(1, round(t * ((i + 1) * 0.6180339887 % 1.0) ** 2)) for i in range(s)]   # many short, few long


def work(case):
    op = case["op"]
    if op == "score":
        es = 4 if case["kind"] == "fp32" else 2
        cells = case["n"] * case["v"]
        out = case["n"] * (8.0 + 8.0 + 8.0 * case["top"])
        if not case["grad"]:
            return {"bytes": es * cells + out, "flops": 5.0 * cells}
        return {"bytes": 2.0 * es * cells + out + 8.0 * case["n"], "flops": 12.0 * cells}
    lens, hq, hkv, d = _lens(case), case["hq"], case["hkv"], case["d"]
    if op in ("packed", "train"):
        rows, pairs = sum(lens) + case["pad"], sum(n * (n + 1) / 2 for n in lens)
        if op == "packed":
            return {"bytes": 2.0 * rows * d * (2 * hq + 2 * hkv), "flops": 4.0 * pairs * hq * d}
        return {"bytes": 2.0 * rows * d * (4 * hq + 4 * hkv), "flops": 14.0 * pairs * hq * d}
    es, sc = (1, 1) if case["kv"] == "e4m3" else (2, 0)
    if op == "write":
        rows = 2 * sum(lens) * hkv
        return {"bytes": float(rows * (d * (2 + es) + sc)), "flops": 2.0 * rows * d}
    keys = sum(lens)
    return {"bytes": float(2 * keys * hkv * (d * es + sc) + 4 * case["b"] * hq * d + 4 * sum(-(-n // case["page"]) for n in lens)),
            "flops": 4.0 * keys * hq * d}


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pages(case, g, need):
    """A cache of pages with rows in it ([P, H, page, D] views of head-major or token-major storage) and the
    sequences' tables: ``need`` pages each, in any order."""
    h, t, d = case["hkv"], case["page"], case["d"]
    width, spare = max(need), 3
    total = sum(need) + spare
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table, at = torch.zeros(len(need), width, dtype=torch.int32), 0
    order = order.cpu()
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (total, h, t, d) if case["layout"] == "head" else (total, t, h, d)
    got = []
    for _ in range(2):
        x = torch.randn(shape, device="cuda", dtype=BF16, generator=g)
        if case["kv"] == "e4m3":
            x = (x * 64).to(E4M3)
        got.append(x if case["layout"] == "head" else x.transpose(1, 2))
    for _ in range(2):
        s = None
        if case["kv"] == "e4m3":   # rows of unequal sizes, near 2^-6 of their codes
            s = torch.randint(120, 123, shape[:3], device="cuda", dtype=torch.uint8, generator=g).view(E8M0)
            s = s if case["layout"] == "head" else s.transpose(1, 2)
        got.append(s)
    return got, table.cuda()


def _cut(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = {"case": case}
    if op == "score":
        n, v = case["n"], case["v"]
        z = torch.randn(n, v, device="cuda", generator=g)
        # a few likely tokens a row, as a trained model's logits have; softcapped at 15
        z[torch.arange(n, device="cuda")[:, None], torch.randint(0, v, (n, 4), device="cuda", generator=g)] += 8.0
        z = 15.0 * torch.tanh(z.mul_(2.0 / 15.0))
        if case["kind"] == "bf16":   # the head's product over a padded vocabulary
            full = torch.zeros(n, (v + 63) // 64 * 64, device="cuda", dtype=BF16)
            full[:, :v] = z
            z = full[:, :v]
        st["logits"] = z.detach().requires_grad_(case["grad"])
        tokens = torch.randint(0, v, (n,), device="cuda", generator=g)
        st["tokens"] = torch.where(torch.rand(n, device="cuda", generator=g) < 0.02, -1, tokens)   # padding
        if case["grad"]:
            st["dlp"] = torch.randn(n, device="cuda", generator=g) / n
            st["dh"] = torch.full((n,), 0.01 / n, device="cuda")
        return st
    hq, h, d = case["hq"], case["hkv"], case["d"]
    lens = _lens(case)
    order = torch.randperm(len(lens), device="cuda", generator=g).tolist()
    lens = [lens[i] for i in order]
    if op == "paged":
        (st["kp"], st["vp"], st["ks"], st["vs"]), st["table"] = _pages(case, g, [-(-n // case["page"]) for n in lens])
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = torch.randn(len(lens), hq, d, device="cuda", dtype=BF16, generator=g)
        return st
    cut = _cut(lens)
    st["cut"] = cut                                   # a user's program knows its batch's lengths
    st["cu"] = torch.tensor(cut, dtype=torch.int32, device="cuda")
    rows = cut[-1] + case.get("pad", 0)
    qkv = torch.randn(rows, (hq + 2 * h) * d, device="cuda", dtype=BF16, generator=g)   # a fused projection's rows
    st["q"] = qkv[:, :hq * d].unflatten(-1, (hq, d))
    st["k"] = qkv[:, hq * d:(hq + h) * d].unflatten(-1, (h, d))
    st["v"] = qkv[:, (hq + h) * d:].unflatten(-1, (h, d))
    if op == "write":
        qkv *= torch.exp(torch.randn(rows, 1, device="cuda", generator=g)).to(BF16)
        # every sequence writes behind what it holds, the first page partly filled
        first = torch.randint(0, 2 * case["page"], (len(lens),), device="cuda", generator=g).tolist()
        (st["kp"], st["vp"], st["ks"], st["vs"]), st["table"] = _pages(case, g, [2 + -(-n // case["page"]) for n in lens])
        st["pos"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        st["first"] = first
        return st
    if op == "train":
        for x in ("q", "k", "v"):
            st[x] = st[x].detach().requires_grad_(True)
        st["do"] = torch.randn(rows, hq, d, device="cuda", dtype=BF16, generator=g)
    return st


# ------------------------------------------------------------------------------- one pass
def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"packed": _packed, "train": _train, "paged": _paged, "write": _write, "score": _score}[op](s)
    from trainium_frontier_b200 import ops
    if op == "packed":
        return ops.packed_attention(s["q"], s["k"], s["v"], s["cu"])
    if op == "train":
        o = ops.packed_attention(s["q"], s["k"], s["v"], s["cu"])
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    if op == "paged":
        return ops.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], None, s["ks"], s["vs"])
    if op == "write":
        ops.paged_cache_write(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["pos"], s["cu"], s["ks"], s["vs"])
        return {k: s[k] for k in ("kp", "vp", "ks", "vs")}
    lp, ent, tok, top = ops.token_logprobs(s["logits"], s["tokens"], s["case"]["top"])
    if not s["case"]["grad"]:
        return {"logprob": lp, "entropy": ent, "top": tok, "top_logprob": top}
    dz, = torch.autograd.grad((lp, ent), (s["logits"],), (s["dlp"], s["dh"]))
    return {"logprob": lp.detach(), "entropy": ent.detach(), "top": tok, "top_logprob": top, "dlogits": dz}


CHUNK = 2 ** 27   # scores held at a time


def _heads(x, g):
    """[T, H, D] as [H * g, T, D] in 32 bits, every head g times."""
    return x.float().transpose(0, 1).repeat_interleave(g, 0)


def _scores(q, k, i0):
    """Scaled scores [H, N, T] of queries i0 .. i0 + N - 1 against keys 0 .. T - 1, and which are seen."""
    x = torch.matmul(q, k.transpose(1, 2)) * q.shape[-1] ** -0.5
    i = torch.arange(i0, i0 + x.shape[1], device="cuda")[:, None]
    return x.masked_fill_(torch.arange(x.shape[2], device="cuda") > i, -math.inf)


def _packed(s, lse=None):
    q, hkv = s["q"].detach(), s["case"]["hkv"]
    out = torch.zeros(q.shape, dtype=BF16, device="cuda")
    g = q.shape[1] // hkv
    for a, b in zip(s["cut"][:-1], s["cut"][1:]):
        n = b - a
        if n == 0:
            continue
        k, v = _heads(s["k"].detach()[a:b], g), _heads(s["v"].detach()[a:b], g)
        step = max(1, CHUNK // (q.shape[1] * n))
        for i in range(0, n, step):
            e = min(n, i + step)
            x = _scores(_heads(q[a + i:a + e], 1), k[:, :e], i)
            m = x.amax(-1, keepdim=True)
            w = torch.exp(x.sub_(m))
            z = w.sum(-1, keepdim=True)
            out[a + i:a + e] = (torch.matmul(w, v[:, :e]) / z).transpose(0, 1).to(BF16)
            if lse is not None:
                lse[:, a + i:a + e] = (m + torch.log(z))[..., 0]
    return out


def _train(s):
    q, hkv = s["q"].detach(), s["case"]["hkv"]
    hq, d = q.shape[1:]
    g, c = hq // hkv, d ** -0.5
    lse = torch.zeros(hq, q.shape[0], device="cuda")
    o = _packed(s, lse)
    dq, dk, dv = (torch.zeros(s[x].shape, dtype=BF16, device="cuda") for x in ("q", "k", "v"))
    for a, b in zip(s["cut"][:-1], s["cut"][1:]):
        n = b - a
        if n == 0:
            continue
        k, v = _heads(s["k"].detach()[a:b], g), _heads(s["v"].detach()[a:b], g)
        sk, sv = torch.zeros_like(k), torch.zeros_like(v)
        step = max(1, CHUNK // (hq * n))
        for i in range(0, n, step):
            e = min(n, i + step)
            qi, do = _heads(q[a + i:a + e], 1), _heads(s["do"][a + i:a + e], 1)
            p = torch.exp(_scores(qi, k[:, :e], i).sub_(lse[:, a + i:a + e, None]))
            sv[:, :e] += torch.matmul(p.transpose(1, 2), do)
            dp = torch.matmul(do, v[:, :e].transpose(1, 2))
            ds = p.mul_(dp - (p * dp).sum(-1, keepdim=True))
            dq[a + i:a + e] = (torch.matmul(ds, k[:, :e]) * c).transpose(0, 1).to(BF16)
            sk[:, :e] += torch.matmul(ds.transpose(1, 2), qi) * c
        dk[a:b] = sk.view(hkv, g, n, d).sum(1).transpose(0, 1).to(BF16)
        dv[a:b] = sv.view(hkv, g, n, d).sum(1).transpose(0, 1).to(BF16)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _values(codes, scale):
    """What cached rows stand for, in 32 bits."""
    return codes.float() if scale is None else codes.float() * scale.float()[..., None]


def _paged(s):
    q, lens, table = s["q"], s["lens"].long(), s["table"].long()
    b, hq, d = q.shape
    h, page = s["kp"].shape[1:3]
    out = torch.empty(b, hq, d, dtype=BF16, device="cuda")
    width = table.shape[1]
    step = max(1, CHUNK // (h * width * page * d))
    seen = torch.arange(width * page, device="cuda") < lens[:, None]
    for i in range(0, b, step):
        e = min(b, i + step)
        k, v = (_values(_u8(c)[table[i:e]].view(c.dtype), None if z is None else _u8(z)[table[i:e]].view(E8M0))
                .transpose(1, 2).reshape(e - i, h, -1, d) for c, z in ((s["kp"], s["ks"]), (s["vp"], s["vs"])))
        see = seen[i:e, None]
        x = torch.matmul(q[i:e].float().view(e - i, h, hq // h, d), k.transpose(2, 3)) * d ** -0.5
        x = x.masked_fill(~see[:, :, None], -math.inf)
        w = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(w, torch.where(see[..., None], v, 0.0)) / w.sum(-1, keepdim=True)   # rows behind the end hold anything
        out[i:e] = o.view(e - i, hq, d).to(BF16)
    return out


def _u8(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _quantise(x):
    """e4m3 codes and e8m0 scales of bf16 rows: the scale is the least power of two (2^-117 at the least) by
    which the row's largest value fits 448."""
    x = x.float()
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax == 0, -117, e).clamp_min(-117)
    y = torch.ldexp(torch.ldexp(x, -(e // 2)[..., None]), -(e - e // 2)[..., None])
    return y.to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def _write(s):
    page = s["case"]["page"]
    n = torch.tensor([b - a for a, b in zip(s["cut"][:-1], s["cut"][1:])])
    seq = torch.repeat_interleave(torch.arange(len(n)), n).cuda()
    at = torch.arange(s["cut"][-1], device="cuda") - s["cu"].long()[seq] + s["pos"].long()[seq]
    to, off = s["table"].long()[seq, at // page], at % page
    for x, cache, scale in (("k", "kp", "ks"), ("v", "vp", "vs")):
        x = s[x]
        if s[scale] is not None:
            x, code = _quantise(x)
            _u8(s[scale])[to, :, off] = _u8(code)
        _u8(s[cache])[to, :, off] = _u8(x)
    return {k: s[k] for k in ("kp", "vp", "ks", "vs")}


def _score(s):
    z, tokens, top = s["logits"].detach(), s["tokens"], s["case"]["top"]
    n = z.shape[0]
    lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    tok, tlp = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
    dz = torch.empty(z.shape, dtype=z.dtype, device="cuda") if s["case"]["grad"] else None
    step = max(1, CHUNK // z.shape[1])
    for i in range(0, n, step):
        x, t = z[i:i + step].float(), tokens[i:i + step]
        m = x.amax(-1, keepdim=True)
        w = torch.exp(x - m)
        total = w.sum(-1, keepdim=True)
        lse = m + torch.log(total)
        p = w / total
        l = x - lse
        h = -(p * l).sum(-1)
        there = (t >= 0) & (t < z.shape[1])
        lp[i:i + step] = torch.where(there, l.gather(1, t.clamp(0, z.shape[1] - 1)[:, None])[:, 0], 0.0)
        ent[i:i + step] = h
        if top:   # equal logits: the lowest token first
            best, at = torch.sort(x, dim=-1, descending=True, stable=True)
            tok[i:i + step] = at[:, :top].to(torch.int32)
            tlp[i:i + step] = best[:, :top] - lse
        if dz is not None:
            d = torch.where(there, s["dlp"][i:i + step], 0.0)[:, None]
            grad = -p * (d + s["dh"][i:i + step, None] * (l + h[:, None]))
            grad.scatter_add_(1, t.clamp(0, z.shape[1] - 1)[:, None], d)
            dz[i:i + step] = grad.to(z.dtype)
    out = {"logprob": lp, "entropy": ent, "top": tok, "top_logprob": tlp}
    if dz is not None:
        out["dlogits"] = dz
    return out


# ------------------------------------------------------------------------------- 64 bits
def _exact_packed(s, grads):
    q, k, v = (s[x].detach() for x in ("q", "k", "v"))
    hkv, d = k.shape[1:]
    g = q.shape[1] // hkv
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v))
    for a, b in zip(s["cut"][:-1], s["cut"][1:]):
        if a == b:
            continue
        for j in range(hkv):
            kk, vv = k[a:b, j].double(), v[a:b, j].double()
            for h in range(j * g, j * g + g):
                for i in range(a, b, 4096):
                    e = min(b, i + 4096)
                    qq = q[i:e, h].double()
                    x = qq @ kk[:e - a].T / math.sqrt(d)
                    hide = torch.ones(x.shape, dtype=torch.bool, device="cuda").triu(i - a + 1)
                    p = torch.softmax(x.masked_fill_(hide, -math.inf), -1)
                    o[i:e, h] = p @ vv[:e - a]
                    if grads:
                        do = s["do"][i:e, h].double()
                        dv[a:e, j] += p.T @ do
                        dp = do @ vv[:e - a].T
                        ds = p * (dp - (do * o[i:e, h]).sum(-1, keepdim=True)) / math.sqrt(d)
                        dq[i:e, h] = ds @ kk[:e - a]
                        dk[a:e, j] += ds.T @ qq
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if grads else o


def _e4m3_rows(x):
    """(values of the codes, scales) of rows, from the definitions of the two formats, in 64 bits."""
    x = x.double()
    m, e = torch.frexp((x.abs().amax(-1, keepdim=True) / 448).clamp_min(2.0 ** -117))
    e = torch.where(m == 0.5, e - 1, e)                       # the least e with amax <= 448 * 2^e
    y = torch.ldexp(x, -e)
    ulp = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp_min(2.0 ** -6)).exponent - 4)
    return torch.round(y / ulp) * ulp, torch.ldexp(torch.ones_like(m), e)[..., 0]


def exact(case, seed):
    op = case["op"]
    if op in ("packed", "train") and work(case)["flops"] > 4e13:
        return None
    s = prepare(case, seed)
    if op in ("packed", "train"):
        return _exact_packed(s, op == "train")
    if op == "score":
        n, v = case["n"], case["v"]
        names = ("logprob", "entropy") + (("dlogits",) if case["grad"] else ())
        got = {k: torch.empty((n, v) if k == "dlogits" else (n,), dtype=torch.float64, device="cuda") for k in names}
        got["top"], got["top_logprob"] = None, torch.empty(n, case["top"], dtype=torch.float64, device="cuda")
        step = max(1, 2 ** 25 // v)
        for i in range(0, n, step):
            at = slice(i, min(n, i + step))
            l = torch.log_softmax(s["logits"].detach()[at].double(), -1)
            t = s["tokens"][at]
            h = -(l.exp() * l).sum(-1)
            one = torch.zeros_like(l).scatter_(1, t.clamp_min(0)[:, None], 1.0) * (t >= 0)[:, None]
            got["logprob"][at], got["entropy"][at] = (one * l).sum(-1), h
            if case["top"]:
                got["top_logprob"][at] = l.topk(case["top"], -1).values
            if case["grad"]:
                dl = s["dlp"][at].double()[:, None] * (t >= 0)[:, None]
                got["dlogits"][at] = dl * (one - l.exp()) - s["dh"][at].double()[:, None] * l.exp() * (l + h[:, None])
        return got
    page = case["page"]
    if op == "paged":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        h = case["hkv"]
        for b, (n, row) in enumerate(zip(s["lens"].tolist(), s["table"].tolist())):
            at = torch.tensor(row[:-(-n // page)], device="cuda")
            kv = []
            for c, z in (("kp", "ks"), ("vp", "vs")):
                x = torch.stack([s[c][p] for p in row[:-(-n // page)]]).double() if s[c].dtype == BF16 else s[c].view(torch.uint8)[at].view(E4M3).double()
                if s[z] is not None:
                    x = x * s[z].view(torch.uint8)[at].view(E8M0).double()[..., None]
                kv.append(x.transpose(0, 1).reshape(h, -1, case["d"])[:, :n])
            x = torch.einsum("hgd,htd->hgt", s["q"][b].double().view(h, -1, case["d"]), kv[0]) / math.sqrt(case["d"])
            out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(x, -1), kv[1]).reshape(-1, case["d"])
        return out
    got = {}
    for name, x, scale in (("kp", "k", "ks"), ("vp", "v", "vs"), ("ks", "k", None), ("vs", "v", None)):
        if s[name] is None:
            got[name] = None
            continue
        full = torch.empty(s[name].shape, dtype=torch.float64, device="cuda")
        full.copy_(s[name])
        new = s[x].double() if s["ks"] is None else _e4m3_rows(s[x])[0 if scale else 1]
        for a, b, p0, row in zip(s["cut"][:-1], s["cut"][1:], s["first"], s["table"].tolist()):
            while a < b:   # a page at a time
                k = min(b - a, page - p0 % page)
                full[row[p0 // page], :, p0 % page:p0 % page + k] = new[a:a + k].transpose(0, 1)
                a, p0 = a + k, p0 + k
        got[name] = full
    return got
