"""Models over packed attention and the paged decoder: what is saved comes back, and what the decoder samples."""
import pytest
import torch

from test_paged_generator import DEVICES, make_model
from trainium_frontier_b200 import checkpoint as ckpt


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
