"""Speculative-decoding operators at the ends of their number formats: NaN codes and scales, infinite
scores, rows near the least and the greatest numbers."""
import math

import pytest
import torch

from tests._specutil import BF16, E4M3, attention64, make_cache, quant_row, raw
from trainium_frontier_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
# nodes and query heads a key/value head: 1, 8, 16, 17, 120 and 256 query rows, for every kernel and tile form
ROWS = [(1, 1), (4, 2), (2, 8), (1, 17), (6, 20), (4, 64)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def attend(q, cache, lens, parents, scale=None):
    """tree_attention against the formula in 64 bits, infinities and NaN included."""
    kc, vc, ks, vs = cache
    device, D = kc.device, q.shape[-1]
    o = ops.tree_attention(q.to(device), kc, vc, i32(lens, device), None if parents is None else parents.to(device), scale, ks, vs)
    o = o.double().cpu()
    want, bound = attention64(q, kc, vc, lens, parents, D ** -0.5 if scale is None else scale, ks, vs)
    assert torch.equal(torch.isnan(o), torch.isnan(want)), (torch.isnan(o).sum(), torch.isnan(want).sum())
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(o), inf) and torch.equal(o[inf], want[inf])
    fine = torch.isfinite(want)
    err = (o - want).abs()
    assert bool((err <= bound)[fine].all()), float((err / bound)[fine].max())
    return want


def queries(B, N, Hq, D, seed=4):
    return torch.randn(B, N, Hq, D, generator=gen(seed)).to(BF16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,G", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_value_row_reaches_all_that_see_it(device, N, G, D):
    """Quantised value rows with the scale NaN: the newest token's, by itself among its neighbours or
    not, and a run of 16 context rows."""
    lens = [0, 16, 37, 128, 192]
    cache = make_cache(len(lens) + 1, 2, 270, D, E4M3, "head", device, gen(D))
    for b, ln in enumerate(lens):
        raw(cache[3])[b, 0, ln + N - 1] = 255
    raw(cache[3])[-1, 1, 16:32] = 255
    want = attend(queries(len(lens) + 1, N, 2 * G, D), cache, lens + [200], None)
    assert bool(want[:-1, N - 1, :G].isnan().all()) and bool(want[-1, :, G:].isnan().all())
    assert bool(want[:-1, :, G:].isfinite().all()) and bool(want[:-1, :N - 1].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("N,G", ROWS)
def test_a_nan_value_counts_however_small_its_weight(device, dtype, N, G):
    """64 neighbouring context rows whose weights are below 2^-300 of the others', one of them with a
    NaN value: a product with NaN is NaN."""
    D, T = 64, 270
    cache = make_cache(1, 1, T, D, dtype, "head", device, gen(1))
    kc, vc, ks, vs = cache
    if dtype == E4M3:
        raw(kc)[:, :, 64:128] = 0xd0          # -8
        raw(ks)[:, :, 64:128] = 127
        raw(vs)[:, :, 70] = 255
    else:
        kc[:, :, 64:128] = -8.0
        vc[:, :, 70, 3:] = math.nan
    q = (queries(1, N, G, D).abs() * 0.25 + 4).to(BF16)
    par = torch.arange(-1, N - 1, dtype=torch.int32)[None]
    if N > 2:
        par[0, 1] = -2                        # and the nodes behind it: unused, zero all the same
    want = attend(q, cache, [130], par)
    assert bool(want[0, 0, :, 3:].isnan().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,G", ROWS)
def test_scores_of_minus_infinity_alone(device, N, G):
    """Where every visible score is -inf the softmax is 0 / 0; beside a finite one they count nothing,
    and unused nodes stay zero."""
    D, T = 128, 1300
    lens = [0, 3, 1000, 1000, 1000]
    kc, vc, _, _ = cache = make_cache(5, 1, T, D, BF16, "head", device, gen(2))
    kc[0, 0, 0, 0] = -math.inf                # node 0
    kc[1, 0, :4, 0] = -math.inf               # the context and node 0
    kc[2, 0, :, 0] = -math.inf                # everything: a NaN row over many tiles
    kc[3, 0, :, 0] = -math.inf
    kc[3, 0, 700, 0] = 1.0                    # all but one
    kc[4, 0, :, 0] = -math.inf
    par = torch.arange(-1, N - 1, dtype=torch.int32).expand(5, N).contiguous()
    if N > 1:
        par[4, -1] = -2
    q = queries(5, N, G, D)
    q[..., 0] = q[..., 0].abs() + 1
    want = attend(q, cache, lens, par)
    assert bool(want[[0, 1, 2], 0].isnan().all()) and bool(want[2].isnan().all()) and bool(want[3].isfinite().all())
    if N > 1:
        assert bool(want[0, 1:].isfinite().all()) and bool((want[4, -1] == 0).all())


def nan_codes(device, N, G, D, code):
    """e4m3's two NaN codes, single ones under ordinary scales, in key and value rows of the context, of
    drafted nodes and of rows that no node sees."""
    B, T = 6, 280
    lens = [130, 130, 125, 125, 60, 0]
    cache = make_cache(B, 1, T, D, E4M3, "head", device, gen(3))
    kc, vc = raw(cache[0]), raw(cache[1])
    vc[0, 0, 7, 5] = code
    vc[0, 0, 129, D - 1] = code
    kc[1, 0, 66, D - 2] = code
    vc[2, 0, 125, 9] = code                   # node 0, seen by all nodes below it
    vc[2, 0, 125 + N - 1, D - 3] = code       # the last one, seen by itself
    kc[3, 0, 125 + N - 1, 1] = code
    vc[4, 0, 60 + N:, ::3] = code             # behind the nodes
    kc[4, 0, 60 + N:, ::3] = code
    vc[5, 0, N - 1, 2] = code
    par = torch.arange(-1, N - 1, dtype=torch.int32).expand(B, N).contiguous()
    par[:, -1] = -1                           # a root of its own
    if N > 2:
        par[4, 1] = -2
        vc[4, 0, 61, :] = code                # an unused node's
        kc[4, 0, 61, :] = code
    want = attend(queries(B, N, G, D), cache, lens, par)
    assert bool(want[1].isnan().all()) and bool(want[4].isfinite().all())
    assert bool(want[2, 0, :, 9].isnan().all()) and bool(want[5, N - 1, :, 2].isnan().all())
    if N > 1:
        assert bool(want[2, 0, :, D - 3].isfinite().all()) and bool(want[3, 0].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,G", ROWS[:3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_nan_codes_with_few_rows(device, N, G, D, code):
    nan_codes(device, N, G, D, code)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,G", ROWS[3:])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_nan_codes_with_many_rows(device, N, G, D, code):
    nan_codes(device, N, G, D, code)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("N,G", ROWS)
@pytest.mark.parametrize("qe,ke,scale", [(-120, 100, 2.0 ** 17), (-122, 117, None), (-110, 105, None), (110, -112, None)])
def test_queries_and_keys_of_opposite_sizes(device, dtype, N, G, qe, ke, scale):
    """Queries near the least (greatest) numbers over keys whose sizes make up for it, so that the
    scores are ordinary ones."""
    B, T, D, lens = 2, 300, 64, [257, 20]
    kc, vc, ks, vs = ops.kv_cache_alloc(B, 1, T, D, dtype, device=device)
    k = (torch.randn(B, T, 1, D, generator=gen(1)) * 2.0 ** ke).to(BF16).to(device)
    v = torch.randn(B, T, 1, D, generator=gen(2)).to(BF16).to(device)
    ops.kv_cache_write(k, v, kc, vc, i32([0, 0], device), None, ks, vs)
    q = (torch.randn(B, N, G, D, generator=gen(3)) * 2.0 ** qe).to(BF16)
    attend(q, (kc, vc, ks, vs), lens, None, scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [1, 3, 200])
def test_rows_near_the_greatest_bf16(device, D, N):
    """A finite row reads back finite: a value that would round to 2^128 is held as 1.875 * 2^127."""
    x = torch.randn(1, N, 1, D, generator=gen(N)).to(BF16).float()
    top = torch.tensor([1.9921875, 1.9375, 1.9296875, 1.75, 1.875, -1.9921875, -1.9375, 1.0]) * 2.0 ** 127
    x[..., :8] = top
    x[:, 0, :, 8:] *= 2.0 ** 126
    x = x.to(BF16)
    assert bool(x.isfinite().all())
    kc, vc, ks, vs = ops.kv_cache_alloc(1, 1, N, D, E4M3, device=device)
    ops.kv_cache_write(x.to(device), x.neg().to(device), kc, vc, i32([0], device), None, ks, vs)
    got = ops.kv_cache_read(kc, vc, i32([N], device), N, ks, vs)
    for y, rows in zip(got, (x, x.neg())):
        for n in range(N):
            codes, scale = quant_row(rows[0, n, 0])
            want = torch.tensor(codes, dtype=torch.float64).clamp(-240, 240) * scale
            assert scale == 2.0 ** 120 and torch.equal(y[0, n, 0].double().cpu(), want)
    if N == 1:
        for G in (1, 17):
            attend(queries(1, 1, G, D) * 2.0 ** -126, (kc, vc, ks, vs), [0], None)


@pytest.mark.parametrize("device", DEVICES)
def test_broadcast_scales_are_read_and_not_written(device):
    """One scale for all rows of a cache may be read; a row's own scale cannot be stored in it."""
    B, H, T, D, N = 2, 2, 40, 64, 3
    kc, vc, ks, vs = make_cache(B, H, T, D, E4M3, "head", device, gen(1))
    one = ks[:, :, :1].expand(B, H, T)
    lens = i32([30, 5], device)
    attend(queries(B, N, 4, D), (kc, vc, one, one), [30, 5], None)
    full = one.contiguous()
    for a, b in zip(ops.kv_cache_read(kc, vc, lens, T, one, one), ops.kv_cache_read(kc, vc, lens, T, full, full)):
        assert torch.equal(a, b)
    x = torch.zeros(B, N, H, D, dtype=BF16, device=device)
    heads = ks[:, :1].expand(B, H, T)
    path, count = i32([[0, 2, -1]] * B, device), i32([2, 2], device)
    before = raw(one).clone(), raw(kc).clone()
    for s in (one, heads):
        with pytest.raises(RuntimeError, match="scales"):
            ops.kv_cache_write(x, x, kc, vc, lens, None, s, s)
        with pytest.raises(RuntimeError, match="scales"):
            ops.kv_cache_commit(kc, vc, lens, path, count, s, s)
    assert torch.equal(raw(one), before[0]) and torch.equal(raw(kc), before[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,G", ROWS)
def test_key_scales_of_the_least_byte(device, N, G):
    """Scale byte 0 is 2^-127, for keys as for values."""
    T, D = 200, 64
    cache = make_cache(1, 1, T, D, E4M3, "head", device, gen(6))
    kc, _, ks, _ = cache
    codes = torch.randint(0x28, 0x7f, (T, D), generator=gen(7)) + 128 * torch.randint(0, 2, (T, D), generator=gen(8))
    raw(kc)[0, 0] = codes.to(torch.uint8).to(device)   # 2^-2 and more: exact in bf16 under this scale
    raw(ks)[0, 0, ::2] = 0
    raw(ks)[0, 0, 1::2] = 1
    attend(queries(1, N, G, D) * 2.0 ** 118, cache, [150], None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,G", ROWS)
def test_a_scale_of_zero(device, N, G):
    """Every visible row weighs the same, and 0 times an infinite score is NaN."""
    D, T = 64, 300
    kc, _, _, _ = cache = make_cache(3, 1, T, D, BF16, "head", device, gen(2))
    kc[1, 0, 70, 0] = math.inf
    kc[2, 0, 200 + N - 1, 0] = -math.inf
    q = queries(3, N, G, D)
    q[..., 0] = q[..., 0].abs() + 1
    par = torch.arange(-1, N - 1, dtype=torch.int32).expand(3, N).contiguous()
    par[:, -1] = -1
    want = attend(q, cache, [200, 200, 200], par, 0.0)
    assert bool(want[0].isfinite().all()) and bool(want[1].isnan().all()) and bool(want[2, -1].isnan().all())
    assert bool(want[2, :-1].isfinite().all())
