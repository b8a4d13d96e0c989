"""Backward attention: weights are stored over scores in TMEM by warps that share lanes.  What a warp stores has to lie over
columns that it alone has read, since nothing holds it back until the other one has read its own."""
import re
from pathlib import Path

import pytest
import torch

KERNELS = Path(__file__).resolve().parents[1] / "trainium_frontier_b200" / "csrc" / "kernels"


def kernel_source(file, name):
    text = (KERNELS / file).read_text()
    start = text.index(f"    {name}(")
    return text[start:text.index("\n}\n", start)]


def columns(pattern, text, env):
    """Columns that the calls of `pattern` (name, width, base, offset) reach, for every h2 of their loops."""
    got = set()
    for width, at in re.findall(pattern, text):
        for h2 in (0, 1) if "h2" in at else (0,):
            first = eval(at, {}, dict(env, h2=h2))
            got |= set(range(first, first + int(width)))
    return got


@pytest.mark.parametrize("file,name,base,halves,share", [
    ("attention_sm100.cu", "fa_bwd2_kernel", "tR0", 2, "half"),
    ("packed_attention.cu", "packed_dkv_kernel", "tS", 4, "quarter"),
    ("packed_attention.cu", "packed_dkv_kernel", "tP", 4, "quarter"),
])
def test_weights_are_stored_over_columns_of_their_own(file, name, base, halves, share):
    text = kernel_source(file, name)
    reads, writes = [], []
    for i in range(halves):
        env = {share: i, "cb": i * (128 // halves)}
        assert re.search(rf"cb = {share} \* {128 // halves}\b", text)
        reads.append(columns(rf"tmem_ld_32x32b_x(\d+)\({base} \+ lane_off \+ ([^,]+),", text, env))
        writes.append(columns(rf"tmem_st_32x32b_x(\d+)\({base} \+ lane_off \+ ([^,]+),", text, env))
        assert len(reads[i]) == 128 // halves and len(writes[i]) == 64 // halves
    for i in range(halves):
        for j in range(halves):
            assert i == j or not writes[i] & (reads[j] | writes[j]), f"{share} {i} stores over columns that {share} {j} reads"


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_of_keys_and_values_repeat(causal):
    """dK and dV are sums in TMEM, in order: the same bits in every run."""
    from trainium_frontier_b200.ops.flash_attention import flash_bwd, flash_fwd
    B, T, H, D = 4, 2048, 10, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(B * T, H * D, dtype=torch.bfloat16, device="cuda", generator=g) for _ in range(4))
    o, lse = flash_fwd(q, k, v, B, T, H, D, D ** -0.5, causal)
    runs = [flash_bwd(q, k, v, o, do, lse, B, T, H, D, D ** -0.5, causal)[1:] for _ in range(20)]
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(run, runs[0]))
