"""Packed prompts, the paged cache and token scores together: ``PagedGenerator``, and document masking through
packed attention."""
import pytest
import torch

from trainium_frontier_b200.config import GPTConfig, RunConfig, validate
from trainium_frontier_b200.inference.generate import generate_reference
from trainium_frontier_b200.inference.paged import PagedGenerator
from trainium_frontier_b200.models import gpt
from trainium_frontier_b200.models.gpt import GPT

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make_model(device, n_kv_heads=0, seed=3, heads=4, dim=64, layers=3, **flags):
    """A model whose tokens depend on all of their context: weights of ordinary size everywhere."""
    torch.manual_seed(seed)
    cfg = GPTConfig(sequence_len=256, vocab_size=300, n_layer=layers, n_head=heads, n_embd=heads * dim, n_kv_heads=n_kv_heads)
    m = GPT(cfg, RunConfig(**flags))
    m.init_weights()
    g = torch.Generator().manual_seed(seed)
    for p in m.parameters():
        if p.dim() == 2:
            p.data.copy_(torch.randn(p.shape, generator=g) * p.shape[1] ** -0.5)
    m.lm_head.weight.data.mul_(6)
    m = m.to(device)
    if device == "cuda":
        m.set_compute_dtype(torch.bfloat16)
    return m


def make_prompts(lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 300, (n,), generator=g) for n in lens]


@torch.no_grad()
def full_logits(m, tokens):
    """Logits [T, V] of one text by the model's own forward."""
    return m(tokens[None].to(m.get_device()).to(torch.int32))[0].float()


@pytest.mark.parametrize("n_kv_heads", [0, 2])
def test_generation_is_that_of_recomputation(n_kv_heads):
    """fp32 on the CPU: greedy tokens, log probabilities, entropies and alternatives of every step against a
    full forward of the text so far."""
    m = make_model("cpu", n_kv_heads)
    prompts = make_prompts([1, 17, 33, 5])
    g = PagedGenerator(m, 4, 64, page=16)
    out = g.generate(prompts, 12, top=3)
    for b, p in enumerate(prompts):
        text = torch.cat([p, out.tokens[b].long()])
        logits = full_logits(m, text)[p.numel() - 1:-1].double()
        lp = torch.log_softmax(logits, -1)
        best = lp.topk(3, -1)
        # fp32 through three layers: 2^-24 of the values a step, some 2^10 steps
        assert torch.equal(out.tokens[b].long(), logits.argmax(-1))
        assert torch.equal(out.top_tokens[b].long(), best.indices)
        for got, want in ((out.top_logprobs[b], best.values), (out.logprobs[b], best.values[:, 0]), (out.entropy[b], -(lp.exp() * lp).sum(-1))):
            assert float((got.double() - want).abs().max()) < 2.0 ** -10
    one = [generate_reference(m, p[None].to(torch.int32), 12)[0] for p in prompts]
    assert torch.equal(out.tokens.long(), torch.stack(one).long())


@pytest.mark.gpu
@pytest.mark.parametrize("n_kv_heads,kv_dtype,dim", [(0, None, 64), (2, None, 64), (1, None, 128), (2, torch.float8_e4m3fn, 64)])
def test_generation_gpu(n_kv_heads, kv_dtype, dim):
    """bf16 on the GPU: the log probabilities of the tokens that were taken against a full forward in fp32
    through the oracle, and each taken token is near the likeliest."""
    m = make_model("cuda", n_kv_heads, dim=dim)
    prompts = make_prompts([1, 17, 130, 5, 64])
    g = PagedGenerator(m, 8, 200, page=32, kv_dtype=kv_dtype)
    out = g.generate(prompts, 20, top=4)
    again = g.generate(prompts, 20, top=4)
    assert torch.equal(out.tokens, again.tokens)
    alone = PagedGenerator(m, 1, 200, page=16, kv_dtype=kv_dtype).generate(prompts[2:3], 1, top=4)
    assert (alone.logprobs[0, 0] - out.logprobs[2, 0]).abs() < 0.2
    m32 = make_model("cpu", n_kv_heads, dim=dim)
    # bf16 activations and weights (2^-8 each) through three layers onto logits of size 6: some 0.1; e4m3 rows (2^-4) more
    tol = 0.3 if kv_dtype is None else 1.0
    for b, p in enumerate(prompts):
        text = torch.cat([p, out.tokens[b].long().cpu()])
        lp = torch.log_softmax(full_logits(m32, text)[p.numel() - 1:-1].double(), -1)
        own = lp.gather(1, out.tokens[b].long().cpu()[:, None])[:, 0]
        assert float((own - out.logprobs[b].cpu()).abs().max()) < tol
        assert float((lp.amax(-1) - own).max()) < tol
        assert torch.equal(out.top_tokens[b, :, 0], out.tokens[b])


@pytest.mark.parametrize("device", DEVICES)
def test_sampling(device):
    m = make_model(device)
    prompts = make_prompts([9, 30])
    g = PagedGenerator(m, 2, 64)
    gen = lambda s: torch.Generator(device=device).manual_seed(s)  # noqa: E731
    a, b, c = (g.generate(prompts, 10, 1.0, generator=gen(s)) for s in (1, 1, 2))
    assert torch.equal(a.tokens, b.tokens) and not torch.equal(a.tokens, c.tokens)
    assert int(a.tokens.min()) >= 0 and int(a.tokens.max()) < 300 and (a.logprobs <= 0).all()


def test_refusals():
    m = make_model("cpu")
    g = PagedGenerator(m, 2, 64, pages=5)
    ok = make_prompts([10, 20])
    for prompts, n, kw in [([], 1, {}), (make_prompts([1, 1, 1]), 1, {}), (make_prompts([60]), 5, {}), (ok, 0, {}), (ok, 40, {}),
                           ([torch.tensor([300])], 1, {}), ([torch.tensor([-1])], 1, {}), ([torch.zeros(2, 3, dtype=torch.long)], 1, {}),
                           ([torch.zeros(0, dtype=torch.long)], 1, {}), (ok, 1, dict(top=33))]:
        with pytest.raises(ValueError):
            g.generate(prompts, n, **kw)
    with pytest.raises(ValueError):
        PagedGenerator(m, 1, 257)
    with pytest.raises(NotImplementedError):
        PagedGenerator(make_model("cpu", gated_mlp=True), 1, 64)


@pytest.mark.parametrize("temperature", [-1.0, float("nan")])
def test_refuses_temperatures(temperature):
    with pytest.raises(ValueError):
        PagedGenerator(make_model("cpu"), 2, 64).generate(make_prompts([3]), 2, temperature=temperature)


def test_refuses_packed_documents_without_document_masking():
    with pytest.raises(ValueError):
        validate(RunConfig(doc_mask_packed=True))
    validate(RunConfig(doc_mask_packed=True, doc_mask=True))


# ------------------------------------------------------------------------------- document masking
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("flags", [dict(), dict(n_kv_heads=2), dict(window_pattern="LS")], ids=str)
def test_document_mask_packed(flags, device, monkeypatch):
    """The same loss and gradients as with dense masks that hide later tokens too, and no later token is seen."""
    dense = gpt.doc_boundary_mask
    monkeypatch.setattr(gpt, "doc_boundary_mask", lambda idx, bos=0: dense(idx, bos) + torch.full(
        (idx.shape[1],) * 2, float("-inf"), device=idx.device).triu(1))
    kv = flags.get("n_kv_heads", 0)
    rc = {k: v for k, v in flags.items() if k != "n_kv_heads"}
    idx = torch.randint(1, 300, (3, 128), generator=torch.Generator().manual_seed(4))
    idx[0, [0, 40, 41]] = 0
    idx[1, 100] = 0
    idx = idx.to(device).to(torch.int32)
    tgt = idx.roll(-1, 1).long()
    got = []
    for packed in (False, True):
        m = make_model(device, kv, doc_mask=True, doc_mask_packed=packed, **rc)
        if device == "cuda":
            for p in m.parameters():
                p.grad = torch.zeros_like(p)
        loss = m(idx, tgt)
        loss.backward()
        got.append((float(loss.detach()), [p.grad.float().clone() for p in m.parameters() if p.grad is not None]))
        if packed:
            with torch.no_grad():
                later = idx.clone()
                later[:, 90:] = 5
                assert torch.equal(m(idx)[:, :90], m(later)[:, :90])
    (la, ga), (lb, gb) = got
    # fp32: 2^-24 a sum; bf16: 2^-8 a value, averaged over the tokens
    tol = 1e-5 if device == "cpu" else 2e-2
    assert abs(la - lb) < tol * abs(la)
    for x, y in zip(ga, gb):
        assert float((x - y).norm()) <= (1e-4 if device == "cpu" else 6e-2) * float(x.norm()) + 1e-9


def test_documents_of_rows():
    from trainium_frontier_b200.models.gpt import PackedDocs
    idx = torch.tensor([[5, 0, 7, 0], [0, 1, 2, 3]])
    assert PackedDocs(idx).cu_seqlens.tolist() == [0, 1, 3, 4, 8]
