"""Models over packed attention and the paged decoder: what is saved comes back, and what the decoders sample."""
import pytest
import torch

from test_paged_generator import DEVICES, make_model, make_prompts
from trainium_frontier_b200 import checkpoint as ckpt
from trainium_frontier_b200.inference.paged import PagedGenerator
from trainium_frontier_b200.inference.speculative import SpeculativeGenerator


@torch.no_grad()
def logits(m, idx):
    return m(idx.to(m.get_device())).float().cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kv", [0, 2])
def test_a_saved_model_with_packed_documents_comes_back(kv, device, tmp_path):
    """The same logits after saving and loading, and no later token is seen."""
    m = make_model(device, kv, doc_mask=True, doc_mask_packed=True)
    path = tmp_path / "final.pt"
    ckpt.save_checkpoint(path, m, {"step": 1})
    back = ckpt.load_for_eval(str(path), device)
    assert back.rc.doc_mask and back.rc.doc_mask_packed
    idx = torch.randint(1, 300, (2, 100), generator=torch.Generator().manual_seed(5))
    idx[0, [0, 40, 41]] = 0
    later = idx.clone()
    later[:, 60:] = 7
    got = logits(back, idx)
    assert torch.equal(got, logits(m, idx))
    assert torch.equal(got[:, :60], logits(back, later)[:, :60])


def test_warm_start_says_that_documents_are_masked_in_another_way(tmp_path, capsys):
    path = tmp_path / "final.pt"
    ckpt.save_checkpoint(path, make_model("cpu", doc_mask=True, doc_mask_packed=True), {"step": 1})
    capsys.readouterr()
    ckpt.warm_start_from(str(path), make_model("cpu", doc_mask=True))
    assert "doc_mask_packed mismatch" in capsys.readouterr().out
    ckpt.warm_start_from(str(path), make_model("cpu", doc_mask=True, doc_mask_packed=True))
    assert "mismatch" not in capsys.readouterr().out


# ------------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("temperature", [1e-300, 1e-46, 1e-39, 1e-30, 1e-6])
def test_temperatures_near_zero_are_greedy(temperature):
    """However small the temperature: the likeliest token (on the CPU; logits over it would be infinite)."""
    m = make_model("cpu")
    g = PagedGenerator(m, 2, 64)
    prompts = make_prompts([9, 30])
    got = g.generate(prompts, 8, temperature, generator=torch.Generator().manual_seed(1))
    want = g.generate(prompts, 8)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.logprobs, want.logprobs)


@pytest.mark.parametrize("temperature", [1e30, 1e300, float("inf")])
def test_any_token_at_great_temperatures(temperature):
    m = make_model("cpu")
    got = PagedGenerator(m, 2, 64).generate(make_prompts([9, 30]), 30, temperature, generator=torch.Generator().manual_seed(1))
    assert int(got.tokens.min()) >= 0 and int(got.tokens.max()) < 300 and torch.isfinite(got.logprobs).all()
    assert got.tokens.unique().numel() > 40      # 60 draws out of 300 alike: 54 different ones are expected


def test_a_model_of_nan_is_sampled_without_a_fault():
    """Weights that are no number: some token of the vocabulary, its log probability NaN (on the CPU; a draw from
    probabilities of NaN would be a device-side assertion)."""
    m = make_model("cpu")
    m.lm_head.weight.data[7] = float("nan")
    for temperature in (0.0, 0.7):
        got = PagedGenerator(m, 2, 64).generate(make_prompts([3, 5]), 4, temperature, generator=torch.Generator().manual_seed(1))
        assert int(got.tokens.min()) >= 0 and int(got.tokens.max()) < 300 and torch.isnan(got.logprobs).all()


@pytest.mark.parametrize("prompt", [torch.tensor([1.5, 2.0]), torch.tensor([True, False]), [3.0, 4.0]], ids=["float", "bool", "list"])
def test_prompts_are_integers(prompt):
    with pytest.raises(ValueError):
        PagedGenerator(make_model("cpu"), 2, 64).generate([prompt], 2)


def test_prompts_of_any_integers():
    m = make_model("cpu")
    p = make_prompts([5])[0]
    want = PagedGenerator(m, 2, 64).generate([p], 4)
    for q in (p.tolist(), p.int(), p.short(), p.numpy()):
        assert torch.equal(PagedGenerator(m, 2, 64).generate([q], 4).tokens, want.tokens)


@pytest.mark.parametrize("temperature", [1e-300, 1e-46, 1e-39, 1e-6])
def test_speculative_decoding_near_temperature_zero_is_greedy(temperature):
    """The other decoder that samples: logits over such a temperature were infinite, and every token 0."""
    g = SpeculativeGenerator(make_model("cpu"), 2, 64)
    p = torch.stack([x[:9] for x in make_prompts([9, 30])]).int()
    assert torch.equal(g.generate(p, 8, temperature, generator=torch.Generator().manual_seed(1)), g.generate(p, 8))
