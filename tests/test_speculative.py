"""Speculative decoding over a key/value cache: the operators against plain 64-bit forms, on the
CPU (the oracle) and on the GPU (the kernels), the calls that they refuse, and rounds of them
together."""
import math

import pytest
import torch

from tests._specutil import (BF16, E4M3, E8M0, attention64, lines, make_cache, make_tree, quant_row, raw, values, verify64)
from trainium_frontier_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
KINDS = [(BF16, "head"), (BF16, "token"), (E4M3, "head"), (E4M3, "token")]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def special_rows(D):
    """Rows at the edges of the quantiser."""
    rows = torch.randn(12, D, generator=gen(3)) * torch.logspace(-3, 3, 12)[:, None]
    rows[0] = 0.0
    rows[1] = 448.0 * torch.linspace(-1, 1, D)           # exactly the largest code
    rows[2] = 450.0 * torch.linspace(-1, 1, D)           # one binade up
    rows[3] *= 2.0 ** 100
    rows[4] *= 2.0 ** -125                               # below the least scale
    rows[5] *= 2.0 ** -90
    rows[6, 3] = math.inf
    rows[7, D - 1] = math.nan
    rows[8] = 2.0 ** -133                                # the least bf16
    rows[9, 0] = -math.inf
    rows[10] = 0.0
    rows[10, 5] = -7.0 * 2.0 ** 40
    return rows.to(BF16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,layout", KINDS)
@pytest.mark.parametrize("B,N,H,D,T", [(1, 1, 1, 64, 1), (3, 7, 2, 128, 20), (2, 33, 5, 64, 64), (4, 12, 3, 128, 40)])
def test_cache_write_and_read(device, dtype, layout, B, N, H, D, T):
    g = gen(B * N)
    kc, vc, ks, vs = make_cache(B, H, T, D, dtype, layout, device, g)
    before = [None if t is None else raw(t).clone().cpu() for t in (kc, vc, ks, vs)]
    # keys and values as slices of a wider projection's rows, 16-byte aligned
    buf = torch.randn(B, N, (2 * H + 3) * D + 8, generator=g).to(BF16)
    if N == 12:
        buf[..., 3 * D + 8:3 * D + 8 + D] = special_rows(D)[None]
        buf[..., (3 + H) * D + 8:(4 + H) * D + 8] = special_rows(D).flip(0)[None]
    buf = buf.to(device)
    k = buf[..., 3 * D + 8:(3 + H) * D + 8].unflatten(-1, (H, D))
    v = buf[..., (3 + H) * D + 8:].unflatten(-1, (H, D))
    pos = [(5 * b) % max(1, T - N + 1) for b in range(B)]
    if B > 1:
        pos[0], pos[-1] = T - N // 2, -2                  # rows past both ends are left out
    count = None if B == 1 else [N, max(0, N - 3), N, 0][:B]
    ops.kv_cache_write(k, v, kc, vc, i32(pos, device), None if count is None else i32(count, device), ks, vs)
    want = [None if t is None else t.clone() for t in before]
    kn, vn = k.cpu(), v.cpu()
    for b in range(B):
        for n in range(N if count is None else count[b]):
            t = pos[b] + n
            if not 0 <= t < T:
                continue
            for i, x in ((0, kn), (1, vn)):
                for h in range(H):
                    if dtype == E4M3:
                        codes, scale = quant_row(x[b, n, h])
                        codes = torch.tensor(codes, dtype=torch.float64)
                        # a row that is not finite has the scale NaN and codes 0
                        want[i][b, h, t] = raw(torch.where(codes.isnan(), 0.0, codes).to(E4M3))
                        want[2 + i][b, h, t] = 255 if math.isnan(scale) else 127 + int(math.log2(scale))
                    else:
                        want[i][b, h, t] = x[b, n, h]
    for w, t in zip(want, (kc, vc, ks, vs)):
        if w is not None:
            a, b = raw(t).cpu(), w
            if dtype == E4M3 and t.dim() == 4:            # the sign of a NaN or a zero says nothing
                a, b = a.clone().view(E4M3).float(), b.view(E4M3).float()
            torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
    lens = i32([(7 * b + 3) % (T + 1) if b else T for b in range(B)], device)
    for R in {T, max(1, T - 1)}:
        got = ops.kv_cache_read(kc, vc, lens, R, ks, vs)
        for y, c, s in zip(got, (kc, vc), (ks, vs)):
            w = values(c.cpu(), None if s is None else s.cpu())[:, :, :R].transpose(1, 2).clone()
            for b in range(B):
                w[b, int(lens[b]):] = 0
            assert y.shape == (B, R, H, D) and y.dtype == BF16 and y.is_contiguous()
            # quantised values are bf16 numbers: nothing is rounded
            torch.testing.assert_close(y.double().cpu(), w, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("device", DEVICES)
def test_quantising_is_off_by_half_a_step(device):
    """A value within the normal range of its row's scale is off by 2^-4 of it at most (e4m3),
    the others by half a subnormal step, 2^-10 of the scale."""
    x = (torch.randn(4, 50, 2, 128, generator=gen(1)) * torch.logspace(-4, 4, 50)[:, None, None]).to(BF16).to(device)
    kc, vc, ks, vs = ops.kv_cache_alloc(4, 2, 50, 128, E4M3, device=device)
    ops.kv_cache_write(x, x, kc, vc, i32([0] * 4, device), None, ks, vs)
    y, _ = ops.kv_cache_read(kc, vc, i32([50] * 4, device), 50, ks, vs)
    scale = ks.double().transpose(1, 2)[..., None]
    err = (y.double() - x.double()).abs()
    assert bool((err <= torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)).all())
    assert bool((x.double().abs().amax(-1, keepdim=True) > 224 * scale).all())   # the least scale that fits


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,layout", KINDS)
@pytest.mark.parametrize("B,N,H,D,T", [(1, 1, 1, 64, 1), (5, 8, 3, 128, 40), (6, 64, 2, 64, 100)])
def test_cache_commit(device, dtype, layout, B, N, H, D, T):
    g = gen(N)
    kc, vc, ks, vs = make_cache(B, H, T, D, dtype, layout, device, g)
    lens, path, count = [], [], []
    for b in range(B):
        c = [N, 1, 0, (N + 1) // 2, N // 3 + 1, N - 1][b % 6]
        p = sorted(torch.randperm(N, generator=g)[:c].tolist())
        if b % 2 == 0 and c and c < N:
            p = [0] + p[1:]
        lens.append([3, T - N, 0, T - N // 2, 1, 7][b % 6] if T > 1 else 0)   # some nodes past the cache
        path.append(p + [-1] * (N - c))
        count.append(c)
    want = [None if t is None else raw(t).clone().cpu() for t in (kc, vc, ks, vs)]
    old = [None if t is None else t.clone() for t in want]
    for b in range(B):
        for i in range(count[b]):
            if lens[b] + path[b][i] < T:
                for w, o in zip(want, old):
                    if w is not None:
                        w[b, :, lens[b] + i] = o[b, :, lens[b] + path[b][i]]
    ops.kv_cache_commit(kc, vc, i32(lens, device), i32(path, device), i32(count, device), ks, vs)
    for w, t in zip(want, (kc, vc, ks, vs)):
        if w is not None:
            assert torch.equal(raw(t).cpu(), w)


def run_attention(device, B, N, Hq, H, D, T, lens, dtype, layout, parents, seed=0, scale=None, spoil=True, qscale=1.0):
    g = gen(seed)
    kc, vc, ks, vs = make_cache(B, H, T, D, dtype, layout, device, g)
    if spoil:   # rows that no node sees hold NaN
        for b in range(B):
            ln = max(0, min(lens[b], T))
            line = lines(None if parents is None else parents[b].tolist(), N)
            bad = [ln + n for n in range(N) if not line[n] and ln + n < T] + list(range(min(T, ln + N), T))
            for c, s in ((kc, ks), (vc, vs)):
                if s is None:
                    c[b, :, bad] = math.nan
                else:
                    raw(s)[b, :, bad] = 255
    q = (torch.randn(B, N, Hq * D + 8, generator=g) * qscale).to(BF16).to(device)[..., 8:].unflatten(-1, (Hq, D))
    o = ops.tree_attention(q, kc, vc, i32(lens, device), None if parents is None else parents.to(device), scale, ks, vs)
    want, bound = attention64(q, kc, vc, lens, parents, D ** -0.5 if scale is None else scale, ks, vs)
    assert o.shape == q.shape and o.dtype == BF16
    err = (o.double().cpu() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound.clamp_min(1e-30)).max()), err.max())
    return o


ATTN = [
    # B, N, Hq, H, D, T, lens
    (1, 1, 1, 1, 128, 1, [0]),
    (1, 1, 1, 1, 64, 300, [299]),
    (3, 1, 4, 2, 128, 300, [0, 127, 128]),
    (2, 5, 10, 10, 64, 200, [64, 123]),
    (2, 6, 13, 13, 128, 260, [122, 255]),       # nodes over a tile's end; nodes past the cache
    (2, 64, 3, 1, 128, 400, [250, 100]),        # 192 rows a key/value head
    (1, 64, 8, 1, 64, 600, [500]),              # 512 rows
    (4, 17, 12, 4, 128, 1000, [900, 3, 511, 640]),
    (1, 9, 40, 2, 64, 150, [100]),              # 20 query heads a key/value head
    (2, 33, 7, 1, 128, 700, [600, 640]),        # 18 nodes a 128-row tile
    (2, 3, 130, 1, 64, 140, [130, 1]),          # more than 128 query heads a key/value head
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,layout", [KINDS[0], KINDS[3]])
@pytest.mark.parametrize("case", ATTN)
def test_tree_attention(device, dtype, layout, case):
    B, N, Hq, H, D, T, lens = case
    for kind in ("chain", "tree", "unused"):
        par = None if kind == "chain" else make_tree(B, N, gen(N), unused=kind == "unused")
        run_attention(device, B, N, Hq, H, D, T, lens, dtype, layout, par, seed=len(kind))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,layout", KINDS)
@pytest.mark.parametrize("B,N,Hq,H,D,T", [(9, 3, 6, 3, 128, 4200), (7, 40, 8, 2, 64, 4100), (12, 64, 2, 1, 128, 3900), (5, 50, 18, 6, 128, 2500),
                                          (200, 33, 12, 12, 64, 70), (150, 64, 20, 10, 128, 66), (100, 9, 16, 16, 128, 40)])
def test_tree_attention_many_tiles(cuda_device, dtype, layout, B, N, Hq, H, D, T):
    """Several key tiles and several (sequence, head) pairs a CTA, one and two row tiles, and many
    pairs of a tile or two each; many calls in a row give the same bits and no wait runs out."""
    from trainium_frontier_b200.ops._ext import check_errors
    g = gen(T)
    lens = [max(0, T - N - 1) * (b + 1) // B if b % 3 else b * 130 % T for b in range(B)]
    par = make_tree(B, N, g)
    some = B if T > 1000 else 6       # the 64-bit form takes its time
    o = run_attention("cuda", some, N, Hq, H, D, T, lens[:some], dtype, layout, par[:some], seed=1)
    kc, vc, ks, vs = make_cache(B, H, T, D, dtype, layout, "cuda", gen(2))
    q = torch.randn(B, N, Hq, D, generator=g).to(BF16).cuda()
    args = (q, kc, vc, i32(lens, "cuda"), par.cuda(), None, ks, vs)
    first = ops.tree_attention(*args)
    one = [ops.tree_attention(q[b:b + 1], kc[b:b + 1], vc[b:b + 1], args[3][b:b + 1], args[4][b:b + 1], None,
                              None if ks is None else ks[b:b + 1], None if vs is None else vs[b:b + 1]) for b in range(B)]
    # a sequence by itself is cut elsewhere: the same within two roundings of p and one of o, 3 * 2^-8
    assert bool(((torch.cat(one).float() - first.float()).norm() <= 3 * 2.0 ** -8 * first.float().norm()))
    wrong = torch.zeros((), dtype=torch.long, device="cuda")
    for _ in range(1500):
        wrong += (ops.tree_attention(*args) != first).any()
    check_errors()
    assert o.shape[1:] == first.shape[1:] and int(wrong) == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_tree_attention_no_row_left(device, dtype):
    """Every node unused, and sequences without context: zeros, whatever the cache holds."""
    B, N, H, D, T = 3, 4, 2, 64, 10
    par = torch.full((B, N), -2, dtype=torch.int32)
    par[1] = torch.tensor([-1, -1, 7, 2])      # two roots, a parent that is no earlier node, its child
    par[2] = torch.tensor([-1, 0, 1, 2])
    o = run_attention(device, B, N, 4, H, D, T, [5, 0, 10], dtype, "head", par)
    assert float(o[0].float().abs().max()) == 0 and float(o[2].float().abs().max()) == 0
    assert float(o[1, 2:].float().abs().max()) == 0 and float(o[1, :2].float().abs().min()) > 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("scale,qscale", [(1.0, 1.0), (0.02, 1.0), (None, 20.0), (0.0, 1.0), (-0.3, 1.0)])
def test_tree_attention_scales(device, dtype, scale, qscale):
    """Scores that are nearly one-hot, nearly flat, all equal, and of the other sign."""
    run_attention(device, 2, 7, 4, 2, 128, 700, [600, 77], dtype, "head", make_tree(2, 7, gen(5)), scale=scale, qscale=qscale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_bad_drafted_rows(device, dtype, D):
    """An infinity or a NaN in a drafted node's key or value reaches the nodes that see it and
    no other."""
    B, N, H, T, ln = 1, 6, 1, 300, 125
    par = torch.tensor([[-1, 0, 0, 1, 1, 2]], dtype=torch.int32)
    kc, vc, ks, vs = make_cache(B, H, T, D, dtype, "head", device, gen(2))
    if dtype == E4M3:
        raw(vs)[0, 0, ln + 2] = 255
        raw(ks)[0, 0, ln + 4] = 255
    else:
        vc[0, 0, ln + 2, 5] = math.inf
        vc[0, 0, ln + 2, 7] = math.nan
        vc[0, 0, ln + 2, 9] = -math.inf
        kc[0, 0, ln + 4, 3] = math.nan
    q = torch.randn(B, N, 2, D, generator=gen(4)).to(BF16).to(device)
    o = ops.tree_attention(q, kc, vc, i32([ln], device), par.to(device), None, ks, vs).double().cpu()
    want, bound = attention64(q, kc, vc, [ln], par, D ** -0.5, ks, vs)
    torch.testing.assert_close(torch.isnan(o), torch.isnan(want))
    torch.testing.assert_close(torch.isinf(o) * o.sign(), torch.isinf(want) * want.sign(), equal_nan=True)
    fine = torch.isfinite(want)
    assert bool(((o - want).abs() <= bound)[fine].all()) and bool(fine[0, [0, 1, 3]].all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,Hq,H", [(3, 2, 1), (6, 8, 2), (40, 4, 1)])
def test_scales_of_any_size(device, N, Hq, H):
    """Value rows from 2^-100 to 2^100, zero rows among them (the least scale), key rows from 2^-20 on."""
    B, T, D, ln = 2, 420, 128, [370, 5]
    g = gen(N)
    x = torch.randn(2, B, T, H, D, generator=g)
    x[0] *= torch.exp2(torch.randint(-20, 2, (B, T, H, 1), generator=g).float())
    x[1] *= torch.exp2(torch.randint(-100, 100, (B, T, H, 1), generator=g).float())
    x[1, :, ::3] = 0
    x[1, 0] *= 2.0 ** -24
    cache = ops.kv_cache_alloc(B, H, T, D, E4M3, device=device)
    kc, vc, ks, vs = cache
    x = x.to(BF16).to(device)
    ops.kv_cache_write(x[0], x[1], kc, vc, i32([0, 0], device), None, ks, vs)
    par = make_tree(B, N, g)
    q = torch.randn(B, N, Hq, D, generator=g).to(BF16).to(device)
    o = ops.tree_attention(q, kc, vc, i32(ln, device), par.to(device), None, ks, vs)
    want, bound = attention64(q, kc, vc, ln, par, D ** -0.5, ks, vs)
    assert bool(((o.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128])
def test_every_code_and_scale_is_read_exactly(device, D):
    """A token without context attends to itself alone: its output is its value row, each of the
    254 finite codes times scales from the least to the greatest that stays in range."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 0x7f) != 0x7f]
    exps = [10, 11, 60, 126, 127, 128, 133, 134, 135, 136, 200, 246]
    B = -(-len(codes) // D) * len(exps)
    kc, vc, ks, vs = ops.kv_cache_alloc(B, 1, 3, D, E4M3, device=device)
    for i in range(B):
        part = codes[(i // len(exps)) * D:][:D]
        raw(vc)[i, 0, 0, :len(part)] = part.to(device)
        raw(vs)[i, 0, 0] = exps[i % len(exps)]
    q = torch.randn(B, 1, 1, D, generator=gen(1)).to(BF16).to(device)
    o = ops.tree_attention(q, kc, vc, i32([0] * B, device), None, None, ks, vs)
    assert torch.equal(o[:, 0, 0].double(), values(vc, vs)[:, 0, 0])


@pytest.mark.parametrize("device", DEVICES)
def test_tree_attention_is_the_same_every_time(device):
    par = make_tree(2, 20, gen(1))
    a, b = (run_attention(device, 2, 20, 8, 2, 128, 1500, [1400, 900], E4M3, "head", par) for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_offsets_past_32_bits(cuda_device, dtype):
    """A cache whose second sequence lies more than 2^32 bytes into it."""
    T, D, N = (1 << 25) + 40 if dtype == E4M3 else (1 << 24) + 40, 128, 3
    kc, vc, ks, vs = ops.kv_cache_alloc(2, 1, T, D, dtype, "head", cuda_device)
    for ln, b in ((300, 1), (T - 2, 0)):
        lens = i32([T if b == 1 else ln, ln], cuda_device)
        lo = max(0, ln - 300)
        x = torch.randn(2, 300 + N, 1, D, generator=gen(1)).to(BF16).to(cuda_device)
        ops.kv_cache_write(x, x, kc, vc, i32([lo, lo], cuda_device), None, ks, vs)
        got = [t[b, 0, lo:lo + 300 + N] for t in (kc, vc)]
        w = [None if s is None else s[b, 0, lo:lo + 300 + N] for s in (ks, vs)]
        want = torch.tensor([quant_row(r)[0] for r in x[b, :, 0].cpu().float()]) if dtype == E4M3 else x[b, :, 0].cpu().double()
        assert torch.equal(got[0].double().cpu()[:T - lo], want[:T - lo])
        if b == 0:
            break     # attention over all of it in 64 bits would take too long
        q = torch.randn(2, N, 2, D, generator=gen(2)).to(BF16).to(cuda_device)
        lens[0] = 5
        o = ops.tree_attention(q, kc, vc, lens, None, None, ks, vs)
        ref, bound = attention64(q[1:], got[0][None, None], got[1][None, None], [ln], None, D ** -0.5,
                                 *(None if s is None else s[None, None] for s in w))
        assert bool(((o[1:].double().cpu() - ref).abs() <= bound).all())
        ops.kv_cache_commit(kc, vc, i32([ln, ln], cuda_device), i32([[0, 2, -1]] * 2, cuda_device), i32([2, 2], cuda_device), ks, vs)
        assert torch.equal(raw(kc)[1, 0, ln + 1], raw(kc)[1, 0, ln + 2])
        y, _ = ops.kv_cache_read(kc, vc, i32([0, ln], cuda_device), ln, ks, vs)
        torch.testing.assert_close(y[1, :, 0].double(), values(kc[1, 0, :ln], None if ks is None else ks[1, 0, :ln]), rtol=0, atol=0)


def probabilities(B, N, V, g, spread=2.0):
    return torch.softmax(torch.randn(B, N, V, generator=g) * spread, -1)


VERIFY = [(1, 1, 1), (2, 1, 7), (3, 2, 5), (8, 6, 8192), (5, 64, 130), (4, 24, 2047), (3, 17, 50000), (2, 9, 131072), (40, 5, 300)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,N,V", VERIFY)
def test_verify_tree(device, B, N, V):
    for kind in ("draft", "near", "rule", "same"):
        g = gen(B + N + V)
        p = probabilities(B, N, V, g)
        par = make_tree(B, N, g, unused=kind == "near")
        q = {"draft": probabilities(B, N, V, g), "same": p.clone(), "rule": None,
             "near": torch.softmax(p.log() + 0.5 * torch.randn(B, N, V, generator=g), -1)}[kind]
        rows = (p if q is None else q).gather(1, par.long().clamp(0, N - 1)[..., None].expand(B, N, V))
        tok = torch.multinomial(rows.reshape(B * N, V), 1, generator=g).view(B, N).to(torch.int32)
        if kind == "near":
            tok[torch.rand(B, N, generator=g) < 0.1] = -1     # padding
            tok[torch.rand(B, N, generator=g) < 0.05] = V
        u = torch.rand(B, N, generator=g)
        if kind == "same":
            u[::2] = 0.99999994                               # the last draw at the end of the row
        want = verify64(tok, par, p, q, u)
        got = ops.verify_tree(*(None if t is None else t.to(device) for t in (tok, par, p, q, u)))
        for a, b in zip(got, want):
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), kind


@pytest.mark.parametrize("device", DEVICES)
def test_verify_tree_edges(device):
    """Siblings that repeat a token, a draft without the target's mass, nothing left after a
    rejection, u = 0, and zeros at both ends of a row."""
    V, N = 6, 5
    par = torch.tensor([[-1, 0, 0, 0, 3]] * 5, dtype=torch.int32)
    tok = torch.tensor([[0, 2, 2, 2, 4], [0, 1, 1, 3, 4], [0, 2, 3, 4, 4], [0, 5, 0, 5, 1], [0, 2, 2, 2, 2]], dtype=torch.int32)
    p = torch.zeros(5, N, V)
    p[..., 1:5] = 0.25
    p[2] = torch.tensor([0, 0, 1.0, 0, 0, 0])
    q = torch.full((5, N, V), 1 / 6)
    q[1] = torch.tensor([0, 0.5, 0, 0.5, 0, 0])
    q[2] = p[2]
    q[4] = torch.tensor([0, 0, 1.0, 0, 0, 0])
    for useq in (q, None):
        for lo in (0.0, 0.5, 0.999):
            u = torch.full((5, N), lo)
            u[2, 1:] = 0.9999999
            want = verify64(tok, par, p, useq, u)
            got = ops.verify_tree(*(None if t is None else t.to(device) for t in (tok, par, p, useq, u)))
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b), (lo, useq is None)


@pytest.mark.parametrize("device", DEVICES)
def test_verify_tree_strided_rows(device):
    """Probabilities as views of a padded vocabulary, aligned and not."""
    B, N = 3, 6
    for V, pad in ((1000, 24), (1001, 0), (999, 2)):
        g = gen(V)
        buf = torch.softmax(torch.randn(B, N + 1, V + pad, generator=g), -1).to(device)
        p, q = buf[:, :N, :V], buf.flip(2)[:, 1:, pad:]
        par = make_tree(B, N, g)
        tok = torch.randint(0, V, (B, N), generator=g).to(torch.int32)
        u = torch.rand(B, N, generator=g) * 0.5
        want = verify64(tok, par, p.cpu(), q.cpu(), u)
        for a, b in zip(ops.verify_tree(tok.to(device), par.to(device), p, q, u.to(device)), want):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rule", [False, True])
def test_verify_tree_keeps_the_targets_law(device, rule):
    """The first new token is distributed as p[root], whatever the draft: over M sequences the
    share of each token is within 5 standard deviations, sqrt(p (1 - p) / M), of p."""
    M, N, V = 40000, 4, 6
    g = gen(11)
    p = probabilities(1, N, V, g, 1.0).expand(M, N, V).contiguous()
    q = probabilities(1, N, V, g, 1.0).expand(M, N, V).contiguous()
    par = torch.tensor([[-1, 0, 0, 1]], dtype=torch.int32).expand(M, N).contiguous()
    if rule:
        tok, q = torch.tensor([[0, 3, 1, 2]], dtype=torch.int32).expand(M, N).contiguous(), None
    else:
        tok = torch.multinomial(q[:, [0, 0, 0, 1]].reshape(-1, V), 1, generator=g).view(M, N).to(torch.int32)
    u = torch.rand(M, N, generator=g)
    _, _, out = ops.verify_tree(*(None if t is None else t.to(device) for t in (tok, par, p, q, u)))
    share = torch.bincount(out[:, 0].cpu().long(), minlength=V).double() / M
    want = p[0, 0].double()
    assert bool(((share - want).abs() <= 5 * (want * (1 - want) / M).sqrt()).all())


def one_round(kc, vc, ks, vs, lens, g, device, B, N, Hq, H, D, V):
    """Tree rows written, attended, verified and committed; returns what an oracle needs."""
    par = make_tree(B, N, g).to(device)
    k, v, q = (torch.randn(B, N, h, D, generator=g).to(BF16).to(device) for h in (H, H, Hq))
    ops.kv_cache_write(k, v, kc, vc, lens, None, ks, vs)
    o = ops.tree_attention(q, kc, vc, lens, par, None, ks, vs)
    p = probabilities(B, N, V, g).to(device)
    up = par.long().clamp_min(0)[..., None].expand(B, N, V)
    tok = torch.multinomial(p.gather(1, up).cpu().reshape(B * N, V), 1, generator=g).view(B, N).to(torch.int32).to(device)
    u = torch.rand(B, N, generator=g).to(device)
    path, count, out = ops.verify_tree(tok, par, p, p, u)
    ops.kv_cache_commit(kc, vc, lens, path, count, ks, vs)
    return k, v, q, o, par, path, count


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,layout", KINDS)
def test_rounds_of_speculative_decoding(device, dtype, layout):
    """Three rounds of write, attention, verification and commit leave the same cache as the
    accepted rows written one after another, and each round's attention reads it."""
    B, N, Hq, H, D, T, V = 3, 8, 4, 2, 64, 160, 50
    g = gen(9)
    kc, vc, ks, vs = ops.kv_cache_alloc(B, H, T, D, dtype, layout, device)
    rk, rv, rks, rvs = ops.kv_cache_alloc(B, H, T, D, dtype, layout, "cpu")
    start = torch.randn(B, 110, H, D, generator=g).to(BF16)
    lens = i32([110, 3, 60], device)
    ops.kv_cache_write(start.to(device), start.to(device), kc, vc, i32([0] * B, device), lens, ks, vs)
    ops.kv_cache_write(start, start, rk, rv, i32([0] * B, "cpu"), lens.cpu(), rks, rvs)
    for _ in range(3):
        k, v, q, o, par, path, count = one_round(kc, vc, ks, vs, lens, g, device, B, N, Hq, H, D, V)
        # the oracle's cache: context, then the whole tree behind it for this round's attention
        ops.kv_cache_write(k.cpu(), v.cpu(), rk, rv, lens.cpu(), None, rks, rvs)
        want, bound = attention64(q, rk, rv, lens.tolist(), par.cpu(), D ** -0.5, rks, rvs)
        assert bool(((o.double().cpu() - want).abs() <= bound).all())
        at = path.long().clamp_min(0).cpu()[:, :, None, None].expand(B, N, H, D)
        ops.kv_cache_write(k.cpu().gather(1, at), v.cpu().gather(1, at), rk, rv, lens.cpu(), count.cpu(), rks, rvs)
        lens = lens + count
        m = int(lens.max())
        for a, b in zip(ops.kv_cache_read(kc, vc, lens, m, ks, vs), ops.kv_cache_read(rk, rv, lens.cpu(), m, rks, rvs)):
            assert torch.equal(a.cpu(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_rounds_captured_in_two_graphs(cuda_device, dtype):
    """Two captured rounds over caches of their own, replayed by turns and on two streams at
    once, give what the same calls give eagerly."""
    B, N, Hq, H, D, T, V = 4, 12, 8, 2, 128, 700, 513
    dev = cuda_device
    graphs, held = [], []
    for i in range(2):
        g = gen(20 + i)
        cache = make_cache(B, H, T, D, dtype, "head", dev, g)
        lens = i32([600, 5, 128, 333 + i], dev)
        par = make_tree(B, N, g).to(dev)
        k, v, q = (torch.randn(B, N, h, D, generator=g).to(BF16).to(dev) for h in (H, H, Hq))
        p = probabilities(B, N, V, g).to(dev)
        tok = torch.randint(0, V, (B, N), generator=g).to(torch.int32).to(dev)
        u = (torch.rand(B, N, generator=g) * 1e-3).to(dev)
        kc, vc, ks, vs = cache

        def call():
            ops.kv_cache_write(k, v, kc, vc, lens, None, ks, vs)
            o = ops.tree_attention(q, kc, vc, lens, par, None, ks, vs)
            path, count, out = ops.verify_tree(tok, par, p, p, u)
            ops.kv_cache_commit(kc, vc, lens, path, count, ks, vs)
            return o, path, count, out
        start = [None if t is None else raw(t).clone() for t in cache]
        eager = [t.clone() for t in call()]
        after = [None if t is None else raw(t).clone() for t in cache]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = call()
        graphs.append((graph, res, eager, cache, start, after))
        held.append((lens, par, k, v, q, p, tok, u))      # a graph reads its inputs where they were

    def reset():
        for _, res, _, cache, start, _ in graphs:
            for t, s in zip(cache, start):
                if t is not None:
                    raw(t).copy_(s)
            for t in res:
                t.zero_()
        torch.cuda.synchronize()

    def check():
        torch.cuda.synchronize()
        for _, res, eager, cache, _, after in graphs:
            for a, b in zip(res, eager):
                assert torch.equal(a, b)
            for t, s in zip(cache, after):
                assert t is None or torch.equal(raw(t), s)
    for _ in range(3):
        reset()
        for gr in graphs:
            gr[0].replay()
        check()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    reset()
    for _ in range(4):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for t, st in zip(gr[3], gr[4]):
                    if t is not None:
                        raw(t).copy_(st)
                gr[0].replay()
    check()


@pytest.mark.gpu
def test_on_another_stream(cuda_device):
    """Calls on a side stream wait for nothing but that stream's own work."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        par = make_tree(2, 9, gen(1))
        run_attention("cuda", 2, 9, 4, 2, 64, 500, [400, 77], BF16, "head", par)
        test_verify_tree("cuda", 4, 24, 2047)
    s.synchronize()


@pytest.mark.parametrize("device", DEVICES)
def test_empty_batches(device):
    kc, vc, ks, vs = ops.kv_cache_alloc(0, 2, 16, 64, E4M3, device=device)
    none = torch.empty(0, dtype=torch.int32, device=device)
    rows = torch.empty(0, 3, 2, 64, dtype=BF16, device=device)
    ops.kv_cache_write(rows, rows, kc, vc, none, None, ks, vs)
    assert ops.kv_cache_read(kc, vc, none, 4, ks, vs)[0].shape == (0, 4, 2, 64)
    ops.kv_cache_commit(kc, vc, none, none.view(0, 0), none, ks, vs)
    assert ops.tree_attention(rows, kc, vc, none, None, None, ks, vs).shape == rows.shape
    e = torch.empty(0, 3, 5, device=device)
    nodes = none.view(0, 3)
    assert ops.verify_tree(nodes, nodes, e, None, torch.empty(0, 3, device=device))[1].shape == (0,)
    kc, vc, _, _ = ops.kv_cache_alloc(2, 2, 16, 64, device=device)
    ops.kv_cache_write(torch.empty(2, 0, 2, 64, dtype=BF16, device=device), torch.empty(2, 0, 2, 64, dtype=BF16, device=device),
                       kc, vc, i32([0, 0], device))
    assert ops.kv_cache_read(kc, vc, i32([1, 1], device), 0)[0].shape == (2, 0, 2, 64)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    B, N, H, D, T, V = 2, 3, 2, 64, 16, 11
    kc, vc, ks, vs = ops.kv_cache_alloc(B, H, T, D, E4M3, device=device)
    bk, bv, _, _ = ops.kv_cache_alloc(B, H, T, D, device=device)
    k = torch.zeros(B, N, H, D, dtype=BF16, device=device)
    q = torch.zeros(B, N, 4, D, dtype=BF16, device=device)
    lens, par = i32([1, 2], device), i32([[-1, 0, 1]] * 2, device)
    p = torch.full((B, N, V), 1 / V, device=device)
    u = torch.zeros(B, N, device=device)
    a = ops.kv_cache_alloc(B, H, T, 32, device=device)
    n65 = torch.zeros(B, 65, 4, D, dtype=BF16, device=device)
    calls = [
        (lambda: ops.kv_cache_write(k, k, kc, vc, lens), "k_scale"),
        (lambda: ops.kv_cache_write(k, k, bk, bv, lens, None, ks, vs), "k_scale"),
        (lambda: ops.kv_cache_write(k, k, bk, vc, lens), "one type"),
        (lambda: ops.kv_cache_write(k, k, bk, bv[:, :, :8], lens), "same sizes"),
        (lambda: ops.kv_cache_write(k, k, kc, vc, lens, None, ks, vs[:, :, :8]), "scales"),
        (lambda: ops.kv_cache_write(k, k, kc, vc, lens, None, ks, raw(vs)), "e8m0"),
        (lambda: ops.kv_cache_write(k.half(), k.half(), bk, bv, lens), "bfloat16"),
        (lambda: ops.kv_cache_write(k[:, :, :1], k[:, :, :1], bk, bv, lens), "k and v"),
        (lambda: ops.kv_cache_write(k, k[:, :2], bk, bv, lens), "k and v"),
        (lambda: ops.kv_cache_write(k.transpose(1, 3).contiguous().transpose(1, 3), k, bk, bv, lens), "unit inner"),
        (lambda: ops.kv_cache_write(k, k, bk, bv, lens.long()), "int32"),
        (lambda: ops.kv_cache_write(k, k, bk, bv, lens[:1]), "int32"),
        (lambda: ops.kv_cache_write(k, k, bk, bv, lens, lens.float()), "int32"),
        (lambda: ops.kv_cache_write(k, k, bk[:1].expand(B, H, T, D), bv[:1].expand(B, H, T, D), lens), "broadcast"),
        (lambda: ops.kv_cache_write(k, k, bk.half(), bv.half(), lens), "bfloat16"),
        (lambda: ops.kv_cache_read(a[0], a[1], lens, 4), "head_dim"),
        (lambda: ops.kv_cache_read(bk, bv, lens, T + 1), "T:"),
        (lambda: ops.kv_cache_read(bk, bv, lens, -1), "T:"),
        (lambda: ops.kv_cache_read(bk, bv, i32([1, 2, 3], device), 4), "int32"),
        (lambda: ops.kv_cache_commit(bk, bv, lens, lens, lens), "path"),
        (lambda: ops.kv_cache_commit(bk, bv, lens, par.float(), lens), "path"),
        (lambda: ops.kv_cache_commit(bk, bv, lens, par, i32([1], device)), "count"),
        (lambda: ops.tree_attention(q[:, :, :3], bk, bv, lens), "multiple"),
        (lambda: ops.tree_attention(n65, bk, bv, lens), "64 nodes"),
        (lambda: ops.tree_attention(q[:, :0], bk, bv, lens), "64 nodes"),
        (lambda: ops.tree_attention(q.half(), bk, bv, lens), "bfloat16"),
        (lambda: ops.tree_attention(q[:1], bk, bv, lens), "the caches' B"),
        (lambda: ops.tree_attention(q[0], bk, bv, lens), "q:"),
        (lambda: ops.tree_attention(q, bk, bv, lens, par[:, :2]), "parents"),
        (lambda: ops.tree_attention(q, bk, bv, lens, par.long()), "parents"),
        (lambda: ops.tree_attention(q, kc, vc, lens, par), "k_scale"),
        (lambda: ops.verify_tree(par, par, p.double(), None, u), "float32"),
        (lambda: ops.verify_tree(par, par, p, p[:, :, :5], u), "q:"),
        (lambda: ops.verify_tree(par.long(), par, p, None, u), "tokens"),
        (lambda: ops.verify_tree(par, par[:1], p, None, u), "parents"),
        (lambda: ops.verify_tree(par, par, p, None, u[:, :2]), "u:"),
        (lambda: ops.verify_tree(par, par, p[:, :0], None, u), "64 nodes"),
        (lambda: ops.verify_tree(torch.zeros(B, 65, dtype=torch.int32, device=device), torch.zeros(B, 65, dtype=torch.int32, device=device),
                                 torch.zeros(B, 65, V, device=device), None, torch.zeros(B, 65, device=device)), "64 nodes"),
    ]
    if device == "cuda":
        wide = torch.zeros(B, N, H * D + 4, dtype=BF16, device=device)[..., 4:].unflatten(-1, (H, D))
        calls += [
            (lambda: ops.kv_cache_write(wide, k, bk, bv, lens), "aligned"),
            (lambda: ops.tree_attention(torch.zeros(B, N, 4 * D + 4, dtype=BF16, device=device)[..., 4:].unflatten(-1, (4, D)),
                                        bk, bv, lens), "aligned"),
            (lambda: ops.kv_cache_write(k.cpu(), k.cpu(), bk, bv, lens), "device"),
            (lambda: ops.kv_cache_write(k, k, bk, bv, lens.cpu()), "device"),
            (lambda: ops.kv_cache_write(k.float(), k.float(), bk, bv, lens), "bfloat16"),
            (lambda: ops.tree_attention(q.cpu(), bk, bv, lens), "device"),
            (lambda: ops.verify_tree(par, par, p, p.cpu(), u), "device"),
        ]
    for call, word in calls:
        with pytest.raises(RuntimeError, match=word):
            call()
    with pytest.raises(ValueError):
        ops.kv_cache_alloc(1, 1, 1, 64, layout="row")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [64, 20000, 131072])
@pytest.mark.parametrize("sharp", [0.5, 0.99, 0.9999])
def test_verify_remainder_far_below_one(device, V, sharp):
    """Many rejections of tokens that the target wants less than the draft, where one token keeps a
    remainder: it falls by 1 - q[t] at each (down to 1e-4 ** 23 here), and stays the only one left,
    so that the next token is t whatever the numbers are."""
    B, N, t = 4, 24, V // 3
    q = torch.full((B, N, V), (1 - sharp) / (V - 1))
    p = torch.full((B, N, V), (1 - sharp) / (V - 1) / 2)
    q[..., t], p[..., t] = sharp, (1 + sharp) / 2
    g = torch.Generator().manual_seed(V)
    tokens = torch.randint(0, V - 1, (B, N), generator=g, dtype=torch.int32)
    tokens += (tokens >= t).to(torch.int32)
    parents = torch.zeros(B, N, dtype=torch.int32)
    parents[:, 0] = -1
    u = torch.rand(B, N, generator=g)
    u[:, 1] = 0.75                        # 2 u q > 2 p; later ones have no remainder, whatever u
    u[1:, 2:] = u[1:, 2:] / 4
    args = [x.to(device) for x in (tokens, parents, p, q, u)]
    path, count, out = ops.verify_tree(*args)
    assert count.tolist() == [1] * B
    assert path[:, 0].tolist() == [0] * B and out[:, 0].tolist() == [t] * B
