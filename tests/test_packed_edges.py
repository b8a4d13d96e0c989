"""Packed attention at the ends of what it takes: first tokens."""
import math

import pytest
import torch

from _packutil import BF16, pack
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
