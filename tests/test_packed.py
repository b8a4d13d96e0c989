"""Packed attention, the paged cache and token log probabilities against plain 64-bit forms: the CPU
oracle and the sm_100a kernels."""
import math

import pytest
import torch

from _packutil import BF16, E4M3, E8M0, close, make_pages, make_table, pack, packed64, paged64, raw, scores64, values
from trainium_frontier_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LENS = [[1], [0, 1, 0], [127, 128, 129], [5, 300, 1, 0, 256], [383, 2], [64, 64, 64], [640], [1] * 40]
HEADS = [(1, 1, 128), (4, 2, 128), (3, 1, 64), (6, 6, 64), (8, 1, 128), (5, 5, 128), (4, 2, 64)]


def check_errors(device):
    if device == "cuda":
        from trainium_frontier_b200.ops import _ext
        torch.cuda.synchronize()
        _ext.check_errors()


# ------------------------------------------------------------------------------- packed attention
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:5])))
def test_packed_attention(lens, heads, device):
    hq, hkv, d = heads
    q, k, v, cu, do = pack(lens, hq, hkv, d, device, seed=len(lens), pad=3, fill=math.nan)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, cu)
    grads = torch.autograd.grad(o, leaves, do)
    check_errors(device)
    want = packed64(q[:-3], k[:-3], v[:-3], cu, d ** -0.5, do[:-3])
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        close(got[:-3].detach(), *want[name], name)
        assert got.dtype == BF16 and (got[-3:] == 0).all(), name + " of rows behind the last sequence"
    with torch.no_grad():
        assert torch.equal(ops.packed_attention(q, k, v, cu), o)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads", [([3000, 1, 1500], (8, 2, 128)), ([2049, 700], (3, 3, 64)), ([4097], (2, 1, 128))], ids=str)
def test_packed_attention_long(lens, heads):
    hq, hkv, d = heads
    q, k, v, cu, do = pack(lens, hq, hkv, d, "cuda", seed=1)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, cu)
    grads = torch.autograd.grad(o, leaves, do)
    want = packed64(q, k, v, cu, d ** -0.5, do)
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        close(got.detach(), *want[name], name)
    again = torch.autograd.grad(ops.packed_attention(*leaves, cu), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "gradients are sums in order"


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_packed_attention_scale(scale, device):
    q, k, v, cu, do = pack([130, 40], 2, 1, 64, device, seed=5)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, cu, scale)
    grads = torch.autograd.grad(o, leaves, do)
    want = packed64(q, k, v, cu, scale, do)
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        close(got.detach(), *want[name], name)


@pytest.mark.parametrize("device", DEVICES)
def test_packed_attention_rows_outside(device):
    """Rows in front of the first sequence and behind the last one, any values in them, and no sequence at all."""
    q, k, v, _, do = pack([400], 2, 2, 64, device, seed=6)
    cu = torch.tensor([150, 150, 333], dtype=torch.int32, device=device)
    out = torch.ones(400, dtype=torch.bool)
    out[150:333] = False
    for t in (q, k, v, do):
        t[out.to(device)] = math.inf
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, cu)
    grads = torch.autograd.grad(o, leaves, do)
    want = packed64(*(t[150:333] for t in (q, k, v)), torch.tensor([0, 183]), 0.125, do[150:333])
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        close(got[150:333].detach(), *want[name], name)
        assert (got[out.to(device)] == 0).all(), name
    assert (ops.packed_attention(q, k, v, cu[:1]) == 0).all()
    assert ops.packed_attention(q[:0], k[:0], v[:0], cu[:1] * 0).shape == (0, 2, 64)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hkv", [1, 2])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_packed_attention_not_finite(bad, hkv, device):
    """What a token holds reaches those that see it, and neither earlier tokens nor other sequences."""
    lens, at = [200, 300, 150], 200 + 140
    q, k, v, cu, do = pack(lens, 2, hkv, 64, device, seed=7)
    clean = packed64(q, k, v, cu, 0.125, do)
    after = torch.zeros(650, dtype=torch.bool)
    after[at:500] = True
    seq = torch.zeros(650, dtype=torch.bool)
    seq[200:500] = True
    for i in range(3):
        x = [q.clone(), k.clone(), v.clone()]
        x[i][at, -1, 3] = bad
        leaves = [t.detach().requires_grad_() for t in x]
        o = ops.packed_attention(*leaves, cu)
        grads = torch.autograd.grad(o, leaves, do)
        keep = ~after.to(device)
        if i == 0:   # a query is seen by itself alone
            keep = torch.ones_like(keep)
            keep[at] = False
        close(o.detach()[keep], clean["o"][0][keep], clean["o"][1][keep], "o")
        if i == 2:
            col = o.detach()[at:500, -1, 3].float().cpu()
            assert (torch.isnan(col) if math.isnan(bad) else col == bad).all()
            assert torch.isfinite(o.detach()[at:500, -1, 4]).all()
        elif math.isnan(bad):
            assert torch.isnan(o.detach()[at, -1]).all()
        for name, got in zip(("dq", "dk", "dv"), grads):
            m = ~seq.to(device)
            close(got[m], clean[name][0][m], clean[name][1][m], name)


@pytest.mark.parametrize("device", DEVICES)
def test_packed_attention_all_scores_minus_infinity(device):
    q, k, v, cu, _ = pack([300], 2, 1, 64, device, seed=8)
    q.abs_()
    k[:130, :, 0] = -math.inf
    o = ops.packed_attention(q, k, v, cu)
    want, bound = packed64(q, k.clamp_min(-1e9), v, cu, 0.125)["o"]
    want[:130] = math.nan
    close(o, want, bound, "o")


@pytest.mark.parametrize("device", DEVICES)
def test_packed_attention_broadcast_inputs(device):
    """Keys and values that are one head broadcast, and an output gradient that is a broadcast number."""
    q, k, v, cu, _ = pack([140, 20], 2, 1, 64, device, seed=9)
    q, k1, v1 = (t.detach().clone().requires_grad_() for t in (q, k, v))
    o = ops.packed_attention(q, k1.expand(-1, 2, -1), v1.expand(-1, 2, -1), cu)
    o.sum().backward()
    want = packed64(q.detach(), k, v, cu, 0.125, torch.ones_like(q))
    for t, name in ((q, "dq"), (k1, "dk"), (v1, "dv")):
        value, bound = want[name]
        if name != "dq":   # each head's gradient is rounded before they are added
            bound = bound * 2 + 2.0 ** -7 * value.abs()
            bound = bound + 2.0 ** -7 * sum(packed64(q.detach()[:, h:h + 1], k, v, cu, 0.125, torch.ones_like(q[:, :1]))[name][0].abs() for h in (0, 1))
        close(t.grad, value, bound, name)


def test_packed_attention_differences():
    """The oracle's gradients against differences of its output, in 32 bits."""
    q, k, v, cu, do = pack([9, 1, 5], 2, 1, 64, "cpu", seed=10, dtype=torch.float32)
    x = [t.contiguous().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.packed_attention(*x, cu), x, do)
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        step = torch.randn(x[i].shape, generator=g)
        # 2^-8: differences are off by its square and by 2^-24 / 2^-8 of the sums
        y = [ops.packed_attention(*[t.detach() + (s * 2.0 ** -8 * step if j == i else 0) for j, t in enumerate(x)], cu) for s in (1, -1)]
        slope = float(((y[0] - y[1]).double() * do).sum() * 2.0 ** 7)
        want = float((grads[i].double() * step).sum())
        size = float((grads[i].double().abs() * step.abs()).sum())
        assert abs(slope - want) <= 2.0 ** -9 * size


@pytest.mark.parametrize("device", DEVICES)
def test_packed_attention_refuses(device):
    q, k, v, cu, _ = pack([20], 4, 2, 64, device)
    bad = [(q[..., :48], k[..., :48], v[..., :48], cu), (q, k[:, :1].expand(-1, 3, -1), v, cu), (q, k[:-1], v, cu), (q.double(), k, v, cu),
           (q, k, v, cu.long()), (q, k, v, cu[None]), (q, k, v, torch.stack([cu, cu], 1)[:, 0]), (q, k, v.float(), cu), (q[0], k, v, cu)]
    for args in bad:
        with pytest.raises(RuntimeError):
            ops.packed_attention(*args)
    for scale in (math.nan, math.inf, -math.inf, 1e39, -1e39, 1e-60):
        with pytest.raises(RuntimeError):
            ops.packed_attention(q, k, v, cu, scale)


@pytest.mark.parametrize("device", DEVICES)
def test_packed_attention_any_strides(device):
    """Inputs whose rows are not 16-byte aligned or lie in another order."""
    M, H, D = 150, 2, 64
    g = torch.Generator().manual_seed(13)
    cu = torch.tensor([0, 100, 150], dtype=torch.int32, device=device)
    odd = torch.randn(M, H * D + 3, generator=g).to(BF16).to(device)[:, 3:].unflatten(-1, (H, D))
    turned = torch.randn(D, H, M, generator=g).to(BF16).to(device).permute(2, 1, 0)
    heads = torch.randn(H, M, D, generator=g).to(BF16).to(device).transpose(0, 1)
    do = torch.randn(H, M, D, generator=g).to(BF16).to(device).transpose(0, 1)
    leaves = [t.detach().requires_grad_() for t in (odd, turned, heads)]
    o = ops.packed_attention(*leaves, cu)
    grads = torch.autograd.grad(o, leaves, do)
    want = packed64(odd, turned, heads, cu, 0.125, do)
    for name, got in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)):
        close(got, *want[name], name)


@pytest.mark.parametrize("device", DEVICES)
def test_packed_attention_many_empty_sequences(device):
    lens = [0] * 700 + [3] + [0] * 900 + [130, 0, 0, 1] + [0] * 40
    q, k, v, cu, do = pack(lens, 2, 1, 64, device, seed=14)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, cu)
    grads = torch.autograd.grad(o, leaves, do)
    want = packed64(q, k, v, cu, 0.125, do)
    for name, got in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)):
        close(got, *want[name], name)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,cut", [(0, [0]), (0, [0, 0, 0]), (9, [0]), (9, [9]), (9, [4, 4])], ids=str)
def test_packed_attention_nothing(M, cut, device):
    """No rows, no sequences, or rows of no sequence: zeros, and zero gradients."""
    g = torch.Generator().manual_seed(14)
    leaves = [torch.randn(M, h, 64, generator=g).to(BF16).to(device).requires_grad_() for h in (4, 2, 2)]
    cu = torch.tensor(cut, dtype=torch.int32, device=device)
    o = ops.packed_attention(*leaves, cu)
    assert o.shape == (M, 4, 64) and (o == 0).all()
    for d, x in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), leaves):
        assert d.shape == x.shape and (d == 0).all()
    check_errors(device)


@pytest.mark.gpu
def test_packed_attention_captured():
    """A captured call reads the lengths of the time of its replay; the backward pass is captured with it."""
    q, k, v, cu, do = pack([100, 200, 57], 4, 2, 64, "cuda", seed=11)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        o = ops.packed_attention(*leaves, cu)
        return (o, *torch.autograd.grad(o, leaves, do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for cut in ([0, 100, 300, 357], [0, 1, 1, 340], [0, 356, 356, 357]):
        cu.copy_(torch.tensor(cut, dtype=torch.int32))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------- paged cache
WRITES = [([3], [0], 16), ([1, 1, 1], [0, 15, 16], 16), ([20, 0, 33], [10, 5, 0], 16), ([70, 5], [60, 127], 64), ([300], [7], 32)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("lens,pos,page", WRITES, ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_paged_cache_write(lens, pos, page, layout, dtype, d, device):
    H, B = 3, len(lens)
    W = max(-(-(a + n) // page) for a, n in zip(pos, lens)) + 1
    P = B * W + 2
    pages = make_pages(P, H, page, d, dtype, layout, device)
    table = make_table(B, W, P, device)
    _, k, v, cu, _ = pack(lens, 1, H, d, device, seed=2, pad=2)
    before = [None if t is None else t.clone() for t in pages]
    ops.paged_cache_write(k, v, *pages[:2], table, torch.tensor(pos, dtype=torch.int32, device=device), cu, *pages[2:])
    rows, codes = [], []
    for x in (k, v):
        c, s = ops.ref.quantise_rows(x.cpu()) if dtype == E4M3 else (x.cpu(), None)
        rows.append(c)
        codes.append(s)
    for i in range(2):
        want, scale = raw(before[i].cpu()).clone(), None if before[2] is None else raw(before[2 + i].cpu()).clone()
        for b in range(B):
            for n in range(lens[b]):
                t, r = pos[b] + n, int(cu[b]) + n
                want[int(table[b, t // page]), :, t % page] = raw(rows[i][r])
                if scale is not None:
                    scale[int(table[b, t // page]), :, t % page] = raw(codes[i][r])
        assert torch.equal(raw(pages[i].cpu()), want)
        if scale is not None:
            assert torch.equal(raw(pages[2 + i].cpu()), scale)


@pytest.mark.parametrize("device", DEVICES)
def test_paged_cache_write_leaves_out(device):
    """Rows that the table has no page for, and those in front of row 0, go nowhere."""
    P, W, page = 4, 2, 16
    pages = make_pages(P, 2, page, 64, BF16, "head", device)
    before = [t.clone() for t in pages[:2]]
    table = torch.tensor([[0, -1], [7, 3], [1, 2]], dtype=torch.int32, device=device)
    pos = torch.tensor([10, 12, -3], dtype=torch.int32, device=device)
    _, k, v, cu, _ = pack([12, 30, 5], 1, 2, 64, device, seed=3)
    ops.paged_cache_write(k, v, *pages[:2], table, pos, cu)
    for new, old, x in zip(pages, before, (k, v)):
        old = old.clone()
        old[0, :, 10:16] = x[0:6].transpose(0, 1)      # then page -1
        old[3, :, 0:16] = x[16:32].transpose(0, 1)     # page 7 is none; rows past the table
        old[1, :, 0:2] = x[45:47].transpose(0, 1)
        assert torch.equal(new, old)
    one = torch.tensor([0, 40, 17], dtype=torch.int32, device=device)   # one row each: page 0, past the table, page 2
    ops.paged_cache_write(k[:3], v[:3], *pages[:2], table, one)
    assert torch.equal(pages[0][0, :, 0], k[0]) and torch.equal(pages[0][2, :, 1], k[2])


ATTN = [(1, 1, 128, 16), (4, 2, 128, 16), (3, 3, 64, 16), (8, 1, 64, 32), (12, 1, 128, 64), (48, 2, 64, 16), (16, 1, 128, 16), (6, 2, 128, 128)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("hq,hkv,d,page", ATTN, ids=str)
def test_paged_attention(hq, hkv, d, page, layout, dtype, device):
    lens = [0, 1, 15, 16, 17, 200, 333, 129]
    B, W = len(lens), -(-333 // page)
    P = B * W + 1
    pages = make_pages(P, hkv, page, d, dtype, layout, device)
    table = make_table(B, W, P, device, seed=1)
    for b, n in enumerate(lens):      # nothing behind the last page is an entry, nothing behind the last row a number
        table[b, -(-n // page):] = -1 if b % 2 else 2 ** 30
        if n % page:
            p = int(table[b, n // page])
            for t in pages[:2]:
                raw(t)[p, :, n % page:] = 0x7f if dtype == E4M3 else math.nan
    g = torch.Generator().manual_seed(2)
    q = torch.randn(B, hq * d * 2, generator=g).to(BF16).to(device)[:, :hq * d].unflatten(-1, (hq, d))
    ln = torch.tensor(lens, dtype=torch.int32, device=device)
    o = ops.paged_attention(q, *pages[:2], table, ln, None, *pages[2:])
    want, bound = paged64(q, *pages[:2], table, ln, d ** -0.5, *pages[2:])
    close(o, want, bound, "o")
    assert (o[0] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.9])
def test_paged_attention_scale(scale, device):
    pages = make_pages(8, 1, 16, 64, BF16, "head", device)
    table = make_table(2, 4, 8, device)
    q = torch.randn(2, 3, 64, generator=torch.Generator().manual_seed(3)).to(BF16).to(device)
    ln = torch.tensor([60, 33], dtype=torch.int32, device=device)
    close(ops.paged_attention(q, *pages[:2], table, ln, scale), *paged64(q, *pages[:2], table, ln, scale, None, None), "o")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_paged_attention_not_finite(dtype, device):
    """NaN in a seen row reaches its sequence; a page shared by two sequences is seen by both up to their lengths;
    entries that are no page hide their rows; scores of -inf alone give NaN."""
    pages = make_pages(6, 1, 16, 64, dtype, "head", device)
    nan = 0x7f if dtype == E4M3 else math.nan
    table = torch.tensor([[0, 1], [0, 2], [3, 9], [-5, 4], [-1, -1], [5, 5]], dtype=torch.int32, device=device)
    raw(pages[1])[0, :, 12, 5] = nan
    lens = torch.tensor([13, 12, 32, 20, 32, 18], dtype=torch.int32, device=device)
    q = torch.randn(6, 2, 64, generator=torch.Generator().manual_seed(4)).to(BF16).to(device)
    o = ops.paged_attention(q, *pages[:2], table, lens, None, *pages[2:])
    want, bound = paged64(q, *pages[:2], table, lens, 0.125, *pages[2:])
    assert torch.isnan(want[0, :, 5]).all() and (want[4] == 0).all()
    close(o, want, bound, "o")
    if dtype == BF16:
        q.abs_()
        pages[0][:, :, :, 0] = -math.inf
        o = ops.paged_attention(q, *pages[:2], table, lens)
        assert torch.isnan(o[[0, 1, 2, 3, 5]]).all() and (o[4] == 0).all()
        pages[0][0, :, 3, 0] = 0.0      # all scores but one are -inf: that row alone
        o = ops.paged_attention(q[:2], *pages[:2], table[:2], lens[:2])
        assert torch.equal(o[1], pages[1][0, :, 3].expand(2, -1))
    else:
        raw(pages[3])[3, :, 2] = 255
        o = ops.paged_attention(q, *pages[:2], table, lens, None, *pages[2:])
        assert torch.isnan(o[2]).all() and torch.isfinite(o[1]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_paged_attention_zero_rows(device):
    """Rows of zeros have the least scale; next to rows of ordinary size they count with their weight."""
    pages = make_pages(4, 1, 16, 64, E4M3, "head", device)
    table = make_table(1, 4, 4, device)
    for i in (0, 3):
        raw(pages[1])[int(table[0, i])] = 0
        raw(pages[3])[int(table[0, i])] = 10
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(5)).to(BF16).to(device)
    ln = torch.tensor([64], dtype=torch.int32, device=device)
    close(ops.paged_attention(q, *pages[:2], table, ln, None, *pages[2:]), *paged64(q, *pages[:2], table, ln, 0.125, *pages[2:]), "o")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("B,hq,hkv,n", [(1, 8, 1, 20001), (3, 4, 4, 5000), (1, 32, 8, 3001)])
def test_paged_attention_long(B, hq, hkv, n, dtype):
    """Sequences cut into many pieces, against packed rows attended in 64 bits."""
    page, d = 32, 128
    W = -(-n // page)
    pages = make_pages(B * W, hkv, page, d, dtype, "head", "cuda")
    table = make_table(B, W, B * W, "cuda", seed=4)
    lens = torch.tensor([n, n // 3, 40][:B], dtype=torch.int32, device="cuda")
    q = torch.randn(B, hq, d, generator=torch.Generator().manual_seed(6)).to(BF16).cuda()
    o = ops.paged_attention(q, *pages[:2], table, lens, None, *pages[2:])
    for b in range(B):
        m = int(lens[b])
        kk, vv = (values(c, s)[table[b].long()].transpose(0, 1).reshape(hkv, -1, d)[:, :m] for c, s in ((pages[0], pages[2]), (pages[1], pages[3])))
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q[b].double().view(hkv, -1, d), kk) * d ** -0.5, -1)
        want, a = p @ vv, p @ vv.abs()
        # weights to bf16 2^-8, or f16 2^-11 with its least steps, 2^-25 of the largest weight times 448; scores as in packed64
        close(o[b], want.reshape(hq, d), (2.0 ** -8 * want.abs() + 2.0 ** -7.9 * a + 2.0 ** -16 * m * p.amax(-1, keepdim=True)).reshape(hq, d), "o")


@pytest.mark.parametrize("device", DEVICES)
def test_paged_refuses(device):
    kp, vp, ks, vs = make_pages(4, 2, 16, 64, E4M3, "head", device)
    table = make_table(2, 2, 4, device)
    lens = torch.tensor([3, 20], dtype=torch.int32, device=device)
    q = torch.zeros(2, 4, 64, dtype=BF16, device=device)
    k = torch.zeros(2, 2, 64, dtype=BF16, device=device)
    odd = make_pages(4, 2, 24, 64, BF16, "head", device)
    for args in [(q, kp, vp, table, lens), (q, kp, vp, table.long(), lens, None, ks, vs), (q, kp, vp, table, lens.long(), None, ks, vs),
                 (q[:, :3], kp, vp, table, lens, None, ks, vs), (q[:1], kp, vp, table, lens, None, ks, vs), (q, *odd[:2], table, lens),
                 (q, kp, vp, table, lens, math.nan, ks, vs), (q[..., :32], kp, vp, table, lens, None, ks, vs)]:
        with pytest.raises(RuntimeError):
            ops.paged_attention(*args)
    for args in [(k, k, kp, vp, table, lens), (k, k, kp, vp, table, lens[:1], None, ks, vs), (k[:1], k[:1], kp, vp, table, lens, None, ks, vs),
                 (k, k, kp, vp, table, lens, lens, ks, vs), (k[:, :1], k[:, :1], kp, vp, table, lens, None, ks, vs),
                 (k, k[:1], kp, vp, table, lens, None, ks, vs), (k, k, *odd[:2], table, lens)]:
        with pytest.raises(RuntimeError):
            ops.paged_cache_write(*args)


@pytest.mark.parametrize("device", DEVICES)
def test_paged_nothing(device):
    """No pages, no table entries, no sequences, no rows."""
    kp, vp, _, _ = make_pages(3, 2, 16, 64, BF16, "head", device)
    before = kp.clone()
    q = torch.ones(2, 4, 64, dtype=BF16, device=device)
    ln = torch.tensor([5, 40], dtype=torch.int32, device=device)
    empty = torch.zeros(2, 0, dtype=torch.int32, device=device)
    assert (ops.paged_attention(q, kp, vp, empty, ln) == 0).all()
    table = torch.tensor([[0], [2]], dtype=torch.int32, device=device)
    assert (ops.paged_attention(q, kp[:0], vp[:0], table, ln) == 0).all()
    assert ops.paged_attention(q[:0], kp, vp, table[:0], ln[:0]).shape == (0, 4, 64)
    assert torch.equal(ops.paged_attention(q, kp, vp, table, ln * 0 - 3), torch.zeros_like(q))
    long, full = (ops.paged_attention(q, kp, vp, table, ln * 0 + n) for n in (1000, 16))   # past the table: as much as it has
    assert torch.equal(long, full)
    k = torch.ones(2, 2, 64, dtype=BF16, device=device)
    ops.paged_cache_write(k, k, kp, vp, empty, ln)
    ops.paged_cache_write(k[:0], k[:0], kp, vp, table, ln, torch.zeros(3, dtype=torch.int32, device=device))
    ops.paged_cache_write(k, k, kp, vp, table[:0], ln[:0], torch.zeros(1, dtype=torch.int32, device=device))
    assert torch.equal(kp, before)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_paged_integers_at_their_ends(dtype, device):
    """Lengths, positions and table entries at the ends of their type reach no row but their own."""
    top, least = 2 ** 31 - 1, -2 ** 31
    pages = make_pages(3, 2, 16, 64, dtype, "head", device)
    before = [None if t is None else raw(t).clone() for t in pages]
    _, k, v, cu, _ = pack([4, 4, 2, 3], 1, 2, 64, device, seed=15)
    table = torch.tensor([[0, 1], [1, 2], [top, 0], [2, least]], dtype=torch.int32, device=device)
    pos = torch.tensor([top, least, 0, 16], dtype=torch.int32, device=device)
    ops.paged_cache_write(k, v, *pages[:2], table, pos, cu, *pages[2:])   # past every row, in front of row 0, no pages
    ops.paged_cache_write(k[:4], v[:4], *pages[:2], table, pos, None, *pages[2:])
    assert all(t is None or torch.equal(raw(t), b) for t, b in zip(pages, before))
    q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(16)).to(BF16).to(device)
    lens = torch.tensor([top, least, top, top], dtype=torch.int32, device=device)
    got = ops.paged_attention(q, *pages[:2], table, lens, None, *pages[2:])
    assert (got[1] == 0).all()
    seen = torch.tensor([[0, 1], [1, 2], [0, 0], [2, 0]], dtype=torch.int32, device=device)
    few = torch.tensor([32, 0, 16, 16], dtype=torch.int32, device=device)
    close(got, *paged64(q, *pages[:2], seen, few, 0.125, *pages[2:]), "o")
    check_errors(device)


@pytest.mark.gpu
def test_paged_step_captured():
    """A decode step, rows written and attended, captured once and replayed as the sequences grow."""
    B, H, d, page, W = 3, 2, 64, 16, 6
    pages = make_pages(B * W, H, page, d, BF16, "head", "cuda")
    table = make_table(B, W, B * W, "cuda")
    lens = torch.tensor([0, 30, 47], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.empty(B, H * (2 if i == 0 else 1), d, dtype=BF16, device="cuda") for i in range(3))

    def step():
        ops.paged_cache_write(k, v, *pages[:2], table, lens)
        lens.add_(1)
        return ops.paged_attention(q, *pages[:2], table, lens)
    keep = lens.clone()
    step()
    lens.copy_(keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lens.copy_(keep)
    for _ in range(20):
        for t in (q, k, v):
            t.normal_(generator=g)
        graph.replay()
        close(out, *paged64(q, *pages[:2], table, lens, 0.125, None, None), "o")
    assert torch.equal(lens, keep + 20)


# ------------------------------------------------------------------------------- scores
def make_logits(N, V, dtype, device, seed=0, strided=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(N, V, generator=g) * 3
    if V > 8:
        z[torch.arange(N)[:, None], torch.randint(0, V, (N, 3), generator=g)] += 6
    if strided:
        full = torch.zeros(N, V + 8 - V % 8)
        full[:, :V] = z
        return full.to(dtype).to(device)[:, :V], g
    return z.to(dtype).to(device), g


SIZES = [(3, 1, 1), (5, 2, 2), (4, 31, 31), (7, 257, 5), (2, 1000, 32), (33, 8192, 5), (1, 8191, 20), (2, 50000, 8)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("N,V,top", SIZES, ids=str)
def test_token_logprobs(N, V, top, dtype, strided, device):
    z, g = make_logits(N, V, dtype, device, strided=strided)
    z = z.detach().requires_grad_()
    tokens = torch.randint(0, V, (N,), generator=g).to(device)
    tokens[::5] = -1
    tokens[1::7] = V
    a, b = torch.randn(N, generator=g).to(device), torch.randn(N, generator=g).to(device)
    got = ops.token_logprobs(z, tokens, top)
    dz, = torch.autograd.grad(got[:2], (z,), (a, b))
    want = scores64(z.detach(), tokens, top, a, b)
    assert torch.equal(got[2].cpu(), want["top_tokens"][0].cpu())
    for x, name in ((got[0], "logprob"), (got[1], "entropy"), (got[3], "top_logprobs")):
        close(x.detach(), *want[name], name)
    value, bound = want["dlogits"]
    assert dz.dtype == dtype and dz.shape == z.shape
    close(dz, value, bound + torch.finfo(dtype).eps / 2 * value.abs(), "dlogits")
    with torch.no_grad():
        plain = ops.token_logprobs(z, tokens.int(), top)
    assert all(torch.equal(x, y) for x, y in zip(plain, got))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("N,V,top", [(1, 131072, 32), (8, 131072, 8), (300, 131072, 1), (2, 300001, 5), (600, 65536, 0), (5000, 1001, 5)], ids=str)
def test_token_logprobs_large(N, V, top, dtype):
    z, g = make_logits(N, V, dtype, "cuda")
    z = z.detach().requires_grad_()
    tokens = torch.randint(0, V, (N,), generator=g).cuda()
    a, b = torch.randn(N, generator=g).cuda(), torch.randn(N, generator=g).cuda()
    got = ops.token_logprobs(z, tokens, top)
    dz, = torch.autograd.grad(got[:2], (z,), (a, b))
    want = scores64(z.detach(), tokens, top, a, b)
    assert torch.equal(got[2], want["top_tokens"][0])
    for x, name in ((got[0], "logprob"), (got[1], "entropy"), (got[3], "top_logprobs")):
        close(x.detach(), *want[name], name)
    value, bound = want["dlogits"]
    close(dz, value, bound + torch.finfo(dtype).eps / 2 * value.abs(), "dlogits")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_token_logprobs_ties(dtype, device):
    """Equal logits: the lowest token first, however many there are."""
    V = 20000
    z = torch.zeros(6, V, dtype=dtype)
    z[1, 7000:] = 1
    z[2] = torch.arange(V) // 4000
    z[3, ::2] = -0.0                                       # equal to 0
    z[4] = -math.inf
    z[4, [5, 9]] = 2
    at = torch.arange(V) // (8 if dtype == BF16 else 4) % 256 < 32   # some threads' shares are all above the others'
    z[5] = torch.where(at, torch.arange(V).float().remainder(97) + 50, -1.0).to(dtype)
    z = z.to(device)
    tokens = torch.tensor([0, 0, 19999, 4, 5, 3], device=device)
    got = ops.token_logprobs(z, tokens, 32)
    want = scores64(z, tokens, 32)
    assert torch.equal(got[2].cpu(), want["top_tokens"][0].cpu())
    for x, name in ((got[0], "logprob"), (got[1], "entropy"), (got[3], "top_logprobs")):
        close(x, *want[name], name)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_token_logprobs_not_finite(dtype, device):
    low = torch.finfo(dtype).min
    z = torch.randn(8, 300, generator=torch.Generator().manual_seed(1)).to(dtype)
    z[0, 10:] = -math.inf
    z[1, 10:] = low
    z[2, 7] = math.nan
    z[3] = -math.inf
    z[4, 9] = math.inf
    z[5] = low
    z[6, :] = -math.inf
    z[6, 299] = 5
    z[7, 3] = -math.nan
    z = z.to(device).requires_grad_()
    tokens = torch.tensor([3, 200, 1, 1, 9, 0, 299, 1], device=device)
    got = ops.token_logprobs(z, tokens, 3)
    lp, ent, tok, top = (t.detach().cpu() for t in got)
    want = scores64(z.detach()[[0, 1, 5, 6]], tokens[[0, 1, 5, 6]], 3)
    for x, name in ((lp, "logprob"), (ent, "entropy"), (top, "top_logprobs")):
        close(x[[0, 1, 5, 6]], *want[name], name)
    assert torch.equal(tok[[0, 1, 5, 6]], want["top_tokens"][0].cpu())
    assert torch.isnan(lp[[2, 3, 4, 7]]).all() and torch.isnan(ent[[2, 3, 4, 7]]).all() and torch.isnan(top[[2, 3, 4, 7]]).all()
    assert tok[2, 0] == 7 and tok[7, 0] == 3 and tok[4, 0] == 9 and tok[3].tolist() == [0, 1, 2]
    dz, = torch.autograd.grad((got[0].sum() + got[1].sum()), (z,))
    assert torch.isfinite(dz[[0, 1, 5, 6]]).all() and (dz[0, 10:] == 0).all() and (dz[6, :299] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_token_logprobs_shapes(device):
    z, g = make_logits(6, 40, torch.float32, device)
    z = z.view(2, 3, 40)
    tokens = torch.randint(0, 40, (2, 3), generator=g).to(device)
    got = ops.token_logprobs(z, tokens, 2)
    flat = ops.token_logprobs(z.view(6, 40), tokens.view(6), 2)
    assert [tuple(t.shape) for t in got] == [(2, 3), (2, 3), (2, 3, 2), (2, 3, 2)]
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, flat))
    one = ops.token_logprobs(z[0, 0], tokens[0, 0], 1)
    assert one[0].shape == () and torch.equal(one[0], got[0][0, 0])
    none = ops.token_logprobs(z[:0], tokens[:0], 4)
    assert [tuple(t.shape) for t in none] == [(0, 3), (0, 3), (0, 3, 4), (0, 3, 4)]
    z = z.detach().requires_grad_()       # one of the two gradients alone
    lp, ent, _, _ = ops.token_logprobs(z, tokens)
    a, = torch.autograd.grad(lp.sum(), (z,), retain_graph=True)
    b, = torch.autograd.grad(ent.sum(), (z,))
    one, zero = torch.ones(2, 3, device=device), torch.zeros(2, 3, device=device)
    for x, gh in ((a, (one, zero)), (b, (zero, one))):
        value, bound = scores64(z.detach(), tokens, 0, *gh)["dlogits"]
        close(x, value, bound + 2.0 ** -23 * value.abs(), "dlogits")


@pytest.mark.parametrize("device", DEVICES)
def test_token_logprobs_edges(device):
    """Tokens at the ends of their type, which are outside the vocabulary; rows and tokens shared or cut out of others."""
    z, g = make_logits(4, 40, torch.float32, device)
    for t in (torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 32 + 1, 3], device=device), torch.tensor([2 ** 31 - 1, -2 ** 31, 40, 3], dtype=torch.int32, device=device)):
        lp = ops.token_logprobs(z, t)[0]
        assert (lp[:3] == 0).all() and lp[3] == ops.token_logprobs(z[3], t[3])[0] and lp[3] < 0
    tokens = torch.randint(0, 40, (3, 5), generator=g).to(device)
    whole = z[0].expand(3, 4, 40).contiguous()
    for a, b in zip(ops.token_logprobs(z[0].expand(3, 4, 40), tokens[:, 1:], 3), ops.token_logprobs(whole, tokens[:, 1:].contiguous(), 3)):
        assert torch.equal(a, b)
    one = z[:1].clone().requires_grad_()       # a row that four tokens share: the sum of their gradients
    da, = torch.autograd.grad(ops.token_logprobs(one.expand(4, 40), tokens[0, 1:])[0].sum(), (one,))
    each = z[:1].expand(4, 40).contiguous().requires_grad_()
    db, = torch.autograd.grad(ops.token_logprobs(each, tokens[0, 1:])[0].sum(), (each,))
    value = db.double().sum(0, keepdim=True)
    close(da, value, 4 * 2.0 ** -24 * db.double().abs().sum(0, keepdim=True), "dlogits")   # a sum of four in any order
    none = z[:0].clone().requires_grad_()
    dn, = torch.autograd.grad(ops.token_logprobs(none, tokens[0, :0])[0].sum(), (none,))
    assert dn.shape == (0, 40)


def test_token_logprobs_differences():
    z, g = make_logits(4, 50, torch.float32, "cpu")
    z.requires_grad_()
    tokens = torch.randint(0, 50, (4,), generator=g)
    a, b = torch.randn(4, generator=g), torch.randn(4, generator=g)
    dz, = torch.autograd.grad(ops.token_logprobs(z, tokens)[:2], (z,), (a, b))
    step = torch.randn(z.shape, generator=g)
    y = [ops.token_logprobs(z.detach() + s * 2.0 ** -8 * step, tokens)[:2] for s in (1, -1)]
    slope = float(sum(((u - w).double() * c).sum() for u, w, c in zip(*y, (a, b))) * 2.0 ** 7)
    size = float((dz.double().abs() * step.abs()).sum())
    assert abs(slope - float((dz.double() * step).sum())) <= 2.0 ** -9 * size


@pytest.mark.parametrize("device", DEVICES)
def test_token_logprobs_refuses(device):
    z, g = make_logits(4, 40, torch.float32, device)
    t = torch.zeros(4, dtype=torch.long, device=device)
    for args in [(z.double(), t), (z, t[:3]), (z, t.float()), (z, t, 33), (z, t, -1), (z[:, :5], t, 6), (z.T.contiguous().T, t), (z[:, :0], t)]:
        with pytest.raises(RuntimeError):
            ops.token_logprobs(*args)


@pytest.mark.gpu
def test_other_stream():
    """Calls on a stream of their own, next to work on the current one."""
    q, k, v, cu, _ = pack([200, 30], 2, 1, 64, "cuda", seed=12)
    z, _ = make_logits(20, 8192, torch.float32, "cuda")
    t = torch.arange(20, device="cuda")
    want = ops.packed_attention(q, k, v, cu), *ops.token_logprobs(z, t, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.packed_attention(q, k, v, cu), *ops.token_logprobs(z, t, 4)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
