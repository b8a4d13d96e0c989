"""Packed attention at the ends of what it takes: first tokens, values that are no number; what its gradients' D is summed from."""
import math

import pytest
import torch

from _packutil import close, pack, packed64
from trainium_frontier_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HEADS = [(1, 1, 128), (4, 2, 128), (3, 1, 64), (10, 10, 64)]


def forward_backward(q, k, v, cu, do):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = ops.packed_attention(*leaves, cu)
    return (o.detach(), *torch.autograd.grad(o, leaves, do))


# ------------------------------------------------------------------------------- first tokens
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", [[1], [1] * 40, [1, 0, 300, 1, 129, 2, 128]], ids=lambda x: "-".join(map(str, x[:5])))
def test_first_tokens_have_no_gradient_through_their_weight(lens, heads, device):
    """A sequence's first token sees itself alone: its weight is 1 whatever its score, so its query's gradient is 0, and so is
    what it adds to its key's."""
    hq, hkv, d = heads
    q, k, v, cu, do = pack(lens, hq, hkv, d, device, seed=21)
    q, k = 3 * q, 3 * k                      # scores of ordinary models' sizes, some tens
    first = cu[:-1].long()[cu[1:] > cu[:-1]]
    _, dq, _, _ = forward_backward(q, k, v, cu, do)
    assert (dq[first] == 0).all()
    only = torch.zeros_like(do)              # no other token has a gradient to hand on
    only[first] = do[first]
    _, dq, dk, dv = forward_backward(q, k, v, cu, only)
    assert (dq == 0).all() and (dk == 0).all()
    want = torch.zeros(dv.shape, dtype=torch.float64, device=device)
    want[first] = do[first].double().unflatten(1, (hkv, -1)).sum(2)
    # weights of 1 to 2^-8 (bf16) at most, one rounding of the sum
    assert ((dv.double() - want).abs() <= 2.0 ** -7 * do.double().abs().unflatten(1, (hkv, -1)).sum(2) * 1.01).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["q", "k", "do"])
def test_first_tokens_keep_what_is_no_number(which, device):
    q, k, v, cu, do = pack([1, 5, 1], 2, 1, 64, device, seed=22)
    {"q": q, "k": k, "do": do}[which][0, :, 3] = math.nan
    _, dq, dk, _ = forward_backward(q, k, v, cu, do)
    assert torch.isnan(dq[0]).any() and torch.isnan(dk[0]).any()
    assert torch.isfinite(dq[1:]).all() and torch.isfinite(dk[1:]).all() and (dq[[1, 6]] == 0).all() and (dk[6] == 0).all()


# ------------------------------------------------------------------------------- values that are no number
def with_bad_values(q, k, v, cu, scale, bad):
    """(output, bound) in 64 bits where v holds infinities and NaN at `bad` (its finite rest in v)."""
    want, bound = packed64(q, k, torch.where(bad, torch.zeros_like(v), v), cu, scale)["o"]
    g = q.shape[1] // k.shape[1]
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        odd = v[a:b].double().masked_fill(~bad[a:b], 0.0)
        up, down, nan = ((f(odd).cumsum(0) > 0).repeat_interleave(g, 1) for f in (
            lambda x: (x == math.inf).int(), lambda x: (x == -math.inf).int(), lambda x: torch.isnan(x).int()))
        w = want[a:b]
        w[up] = math.inf
        w[down] = -math.inf
        w[nan | (up & down)] = math.nan
    return want, bound


@pytest.mark.parametrize("device,lens", [("cpu", [300, 1, 140]), pytest.param("cuda", [3000, 1, 700, 130], marks=pytest.mark.gpu),
                                         pytest.param("cuda", [90, 128, 257, 3] * 6, marks=pytest.mark.gpu)], ids=str)
@pytest.mark.parametrize("heads", [(4, 2, 128), (3, 3, 64), (5, 1, 128)], ids=str)
@pytest.mark.parametrize("many", [False, True])
def test_values_that_are_no_number_reach_who_sees_them(many, heads, lens, device):
    """Tokens anywhere in long and short sequences: infinities and NaN of values reach the dimensions of the tokens that see
    them, and nothing else; all other entries are as exact as ever."""
    hq, hkv, d = heads
    q, k, v, cu, _ = pack(lens, hq, hkv, d, device, seed=23)
    v = v.clone()
    g = torch.Generator().manual_seed(24)
    M = sum(lens)
    at = torch.randint(0, M, (M // 3 if many else 9,), generator=g)
    at[:2] = torch.tensor([lens[0] - 1, lens[0] // 2])      # a sequence's last token, seen by itself alone
    which = torch.randint(0, 3, at.shape, generator=g)
    dim = torch.randint(0, d // 4, at.shape, generator=g)
    for i, x in enumerate((math.inf, -math.inf, math.nan)):
        m = which == i
        v[at[m].to(device), i % hkv, dim[m].to(device)] = x
    bad = ~torch.isfinite(v)
    close(ops.packed_attention(q, k, v, cu), *with_bad_values(q, k, v, cu, d ** -0.5, bad), "o")


@pytest.mark.parametrize("device", DEVICES)
def test_no_weight_and_infinite_values(device):
    """All scores -inf: the weights are no numbers, whatever the values are."""
    q, k, v, cu, _ = pack([40], 2, 1, 64, device, seed=25)
    q, k, v = q.abs(), k.clone(), v.clone()
    k[:30, :, 0] = -math.inf
    v[3, 0, 5] = math.inf
    o = ops.packed_attention(q, k, v, cu)
    assert torch.isnan(o[3:30]).any(-1).all() and torch.isnan(o[3:30, :, 5]).all() and torch.isnan(o[:3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(2, 1, 128), (3, 3, 64)], ids=str)
def test_values_of_nan_cost_no_more_than_a_few_numbers(heads):
    """A model that has diverged is as quick as one that has not: within 4 times (rows of NaN are 128 a tile at most, some
    100 cycles each, next to a step's 3700 of which a sequence of 16384 has 64 a tile on average)."""
    q, k, v, cu, _ = pack([16384], *heads, "cuda", seed=26)

    def us(v):
        for _ in range(2):
            ops.packed_attention(q, k, v, cu)
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        for _ in range(3):
            ops.packed_attention(q, k, v, cu)
        b.record()
        b.synchronize()
        return a.elapsed_time(b)
    nan = torch.full_like(v, math.nan)
    assert us(nan) < 4 * us(v)
    assert torch.isnan(ops.packed_attention(q, k, nan, cu)).all()


# ------------------------------------------------------------------------------- what D is summed from
# The gradients' D_i = dO_i . o_i is not taken of the rounded output: in a sequence's first 128 rows it is the sum of the 32-bit
# weights times dP, and behind them the output's product with its rest, to 16 bits.  (The bounds of packed64's gradients are
# wider: they would admit a D of the rounded output.)  Values of 16 +- 1 show it: dP - D is of size sqrt(128) = 11.3 (64: 8), and so
# are sums of dO.  A rounding of o to steps of 2^-3 is off by 0.036 (rms), independently in each dimension: D by 0.036 * 11.3, ds
# and with it dq and dk by 3.6e-2 of their size.  Weights rounded to bf16 (1.66e-3 rms) move all dimensions of o
# by 16 * 1.66e-3 sqrt(sum p^2), D by 11.3 times that, ds by 2.7e-2 sqrt(sum p^2); sum p^2 is some e / n among n keys: 1e-2 for
# n = 20, 2.7e-3 for n = 256.  The rounding of ds and that of the result are 1.66e-3 each: 2.4e-3 in all.
def offset_values(lens, heads, device, seed):
    q, k, v, cu, do = pack(lens, *heads, device, seed=seed)
    return q, k, (16 + v.float()).to(v.dtype), cu, do


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads", [(4, 2, 128), (3, 1, 64)], ids=str)
def test_gradients_of_short_sequences_take_d_from_their_weights(heads, device):
    """Nearer than weights or an output of 8 bits allow: 5e-3 lies between the 2.4e-3 of the two last roundings and 1e-2."""
    q, k, v, cu, do = offset_values([20, 3, 128, 9, 2, 60, 14, 31] * 4, heads, device, 27)
    _, dq, dk, _ = forward_backward(q, k, v, cu, do)
    want = packed64(q, k, v, cu, heads[2] ** -0.5, do)
    few = torch.cat([torch.arange(a, b) for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]) if b - a <= 20]).to(device)
    for got, name in ((dq, "dq"), (dk, "dk")):
        assert rel(got, want[name][0]) < 5e-3, name
        assert rel(got[few], want[name][0][few]) < 5e-3, name + " of up to 20 rows"


@pytest.mark.parametrize("device,n", [("cpu", 400), pytest.param("cuda", 1500, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("heads", [(4, 2, 128), (3, 1, 64)], ids=str)
def test_gradients_of_long_sequences_take_d_from_the_output_and_its_rest(heads, device, n):
    """8e-3: above the 2.4e-3 and 2.7e-3 of all that is rounded to 8 bits, below the 3.6e-2 of a rounded output."""
    q, k, v, cu, do = offset_values([n, 256], heads, device, 28)
    _, dq, dk, _ = forward_backward(q, k, v, cu, do)
    want = packed64(q, k, v, cu, heads[2] ** -0.5, do)
    for a, b in ((128, n), (n + 128, n + 256)):
        assert rel(dq[a:b], want["dq"][0][a:b]) < 8e-3
    assert rel(dk, want["dk"][0]) < 8e-3


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(4, 2, 128), (3, 1, 64)], ids=str)
def test_the_rest_of_the_output(heads):
    """The output with its rest is off by what rounded weights cost (2.7e-3 and less from 256 keys on), the output alone by 0.036."""
    from trainium_frontier_b200.ops._ext import C, err_word
    q, k, v, cu, _ = offset_values([1200, 700], heads, "cuda", 29)
    out, _, low = C().packed_attention_fwd(q, k, v, cu, heads[2] ** -0.5, True, err_word(q.device))
    want = packed64(q, k, v, cu, heads[2] ** -0.5)["o"][0]
    for a, b in ((256, 1200), (1456, 1900)):
        alone = float((out.double() - want)[a:b].square().mean().sqrt())
        both = float((out.double() + low.double() - want)[a:b].square().mean().sqrt())
        assert both < 6e-3 and 0.02 < alone
