"""KV-cache greedy decoding (prefill + graph-captured decode) vs full recomputation."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dev, depth=2, n_embd=256, head_dim=128, seq=512):
    from trainium_frontier_b200.config import preset
    from trainium_frontier_b200.models.gpt import GPT
    cfg = preset("tiny", depth=depth, n_embd=n_embd, head_dim=head_dim, seq_len=seq)
    torch.manual_seed(5)
    m = GPT(cfg.model_config(), cfg)
    m.init_weights()
    with torch.no_grad():  # a non-degenerate random model (zero-init projections otherwise)
        for b in m.transformer.h:
            b.mlp.c_proj.weight.normal_(0, 0.02)
        m.lm_head.weight.normal_(0, 0.05)
    m.set_compute_dtype(torch.bfloat16)
    return m.to(dev).eval()


@pytest.mark.parametrize("use_graph", [False, True])
def test_cached_decode_matches_recompute(cuda_device, use_graph):
    from trainium_frontier_b200.inference.generate import Generator, generate_reference
    from trainium_frontier_b200.ops._ext import check_errors
    m = _model(cuda_device)
    B, T, N = 4, 128, 16
    prompts = torch.randint(1, 8192, (B, T), device=cuda_device, dtype=torch.int32)
    ref = generate_reference(m, prompts, N)
    gen = Generator(m, B, T + N + 8)
    out = gen.generate(prompts, N, use_graph=use_graph)
    check_errors()
    agree = (out.long() == ref.long()).float().mean().item()
    # bf16 logits of two different kernel paths may break near-ties differently late in the
    # sequence; the first tokens must agree exactly
    assert torch.equal(out[:, :4].long(), ref[:, :4].long())
    assert agree > 0.9, agree


def test_decode_attention_kernel(cuda_device):
    from trainium_frontier_b200.ops._ext import C
    torch.manual_seed(0)
    B, Tm, H, D, L = 3, 300, 4, 128, 257
    q = torch.randn(B, H * D, device=cuda_device).to(torch.bfloat16)
    kc = torch.randn(B, Tm, H * D, device=cuda_device).to(torch.bfloat16)
    vc = torch.randn(B, Tm, H * D, device=cuda_device).to(torch.bfloat16)
    ln = torch.tensor([L], dtype=torch.int32, device=cuda_device)
    out = torch.empty(B, H * D, dtype=torch.bfloat16, device=cuda_device)
    C().decode_attn(q, kc, vc, ln, H, D, D ** -0.5, out)
    qf = q.float().view(B, H, 1, D)
    kf = kc[:, :L].float().view(B, L, H, D).transpose(1, 2)
    vf = vc[:, :L].float().view(B, L, H, D).transpose(1, 2)
    ref = torch.softmax(qf @ kf.transpose(-1, -2) * D ** -0.5, -1) @ vf
    assert (out.float().view(B, H, D) - ref.squeeze(2)).abs().max().item() < 2e-2


@pytest.mark.parametrize("layout", ["token", "head"])
def test_split_decode_attention_kernel(cuda_device, layout):
    """Cache length split over CTAs per (batch, head), partials combined by the last CTA;
    repeated calls check that the arrival counters are left zeroed.  Token-major
    [B, T, H*D] and head-major [B, H, T, D] caches."""
    from trainium_frontier_b200.ops._ext import C
    torch.manual_seed(1)
    B, Tm, H, D, splits = 3, 640, 4, 128, 5
    q = torch.randn(B, H * D, device=cuda_device).to(torch.bfloat16)
    kc = torch.randn(B, Tm, H * D, device=cuda_device).to(torch.bfloat16)
    vc = torch.randn(B, Tm, H * D, device=cuda_device).to(torch.bfloat16)
    if layout == "head":
        kcs = kc.view(B, Tm, H, D).transpose(1, 2).contiguous()
        vcs = vc.view(B, Tm, H, D).transpose(1, 2).contiguous()
    else:
        kcs, vcs = kc, vc
    ws = torch.zeros(B * H * splits * (D + 4), device=cuda_device)
    cnt = torch.zeros(B * H, dtype=torch.int32, device=cuda_device)
    for L, pdl in ((1, False), (77, True), (513, False), (640, True)):
        ln = torch.tensor([L], dtype=torch.int32, device=cuda_device)
        out = torch.empty(B, H * D, dtype=torch.bfloat16, device=cuda_device)
        C().decode_attn_split(q, kcs, vcs, ln, H, D, D ** -0.5, out, ws, cnt, splits, pdl)
        qf = q.float().view(B, H, 1, D)
        kf = kc[:, :L].float().view(B, L, H, D).transpose(1, 2)
        vf = vc[:, :L].float().view(B, L, H, D).transpose(1, 2)
        ref = torch.softmax(qf @ kf.transpose(-1, -2) * D ** -0.5, -1) @ vf
        assert (out.float().view(B, H, D) - ref.squeeze(2)).abs().max().item() < 2e-2, L
        assert int(cnt.abs().sum()) == 0


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
def test_speculative_greedy_decoding(cuda_device, kv, head_dim):
    """Speculative greedy decoding against plain greedy decoding by recomputation: a draft that
    knows the answer on one branch of its tree, and the draft by rule."""
    from trainium_frontier_b200.inference.generate import generate_reference
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    from trainium_frontier_b200.ops._ext import check_errors
    m = _model(cuda_device, head_dim=head_dim)
    B, T, N = 4, 128, 24
    prompts = torch.randint(1, 8192, (B, T), device=cuda_device, dtype=torch.int32)
    ref = generate_reference(m, prompts, N)
    full = torch.cat([prompts.long(), ref.long(), torch.zeros(B, 8, device=cuda_device, dtype=torch.long)], 1)

    def oracle(text, lens):
        tok = torch.randint(0, 8192, (B, 5), device=cuda_device).to(torch.int32)
        for k, node in enumerate((2, 3, 5)):
            tok[:, node - 1] = full.gather(1, (lens.long() + k).clamp_max(full.shape[1] - 1)[:, None])[:, 0].to(torch.int32)
        return tok, torch.tensor([[0, 0, 2, 2, 3]] * B, dtype=torch.int32, device=cuda_device), None
    for draft in (oracle, None):
        g = SpeculativeGenerator(m, B, 256, draft, kv)
        out = g.generate(prompts, N)
        check_errors()
        assert out.shape == (B, N)
        if kv == torch.bfloat16:
            # bf16 logits of two kernel paths may break near-ties differently late in the sequence
            assert torch.equal(out[:, :4].long(), ref[:, :4].long())
            agree = (out.long() == ref.long()).float().mean().item()
            assert agree > 0.9, agree
            assert draft is None or g.rounds < N // 2
    sampled = SpeculativeGenerator(m, B, 256, None, kv).generate(prompts, 8, 1.0)
    check_errors()
    assert int(sampled.min()) >= 0 and int(sampled.max()) < 8192


@pytest.mark.parametrize("head_dim", [64, 128])
def test_speculative_decoding_where_attention_decides(cuda_device, head_dim):
    """Attention projections that are not zero, a wide tree whose last nodes hold the right tokens
    and a cache that ends with the text.  The new tokens against the same model's probabilities by
    recomputation: each is the largest or nearer to it than the two paths' bf16 rounding."""
    from trainium_frontier_b200.inference.generate import generate_reference
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    from trainium_frontier_b200.ops._ext import check_errors
    m = _model(cuda_device, head_dim=head_dim)
    with torch.no_grad():
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, 0.2)
    B, T, N = 3, 128, 10
    prompts = torch.randint(1, 8192, (B, T), device=cuda_device, dtype=torch.int32)
    other = prompts.clone()
    other[:, :T - 1] = torch.randint(1, 8192, (B, T - 1), device=cuda_device, dtype=torch.int32)
    ref = generate_reference(m, prompts, N)
    assert not torch.equal(generate_reference(m, other, N), ref)
    full = torch.cat([prompts.long(), ref.long(), torch.zeros(B, 8, device=cuda_device, dtype=torch.long)], 1)

    def draft(text, lens):
        tok = torch.full((B, 63), 3, dtype=torch.int32, device=cuda_device)
        for k in range(2):
            tok[:, 61 + k] = full.gather(1, (lens.long() + k).clamp_max(full.shape[1] - 1)[:, None])[:, 0].to(torch.int32)
        return tok, torch.tensor([[0] * 62 + [62]] * B, dtype=torch.int32, device=cuda_device), None
    g = SpeculativeGenerator(m, B, T + N, draft)
    out = g.generate(prompts, N).long()
    check_errors()
    text = torch.cat([prompts.long(), out], 1)
    with torch.no_grad():
        z = m(torch.nn.functional.pad(text, (0, 256 - T - N)).to(torch.int32))[:, T - 1:T + N - 1].double()
    gap = z.amax(-1) - z.gather(-1, out[..., None])[..., 0]
    # a logit is a product of n_embd terms of a normed state and weights of 0.05, each state off by
    # some roundings of 2^-8 in either path: sqrt(256) * 0.05 * 2^-8 * 8 roundings * 2 paths, four times over
    assert float(gap.max()) <= 4 * 256 ** 0.5 * 0.05 * 2 ** -8 * 16, gap


@pytest.mark.parametrize("T", [1, 100, 130])
def test_speculative_prompts_of_any_length_use_the_kernels(cuda_device, T, monkeypatch):
    """Prompts that are no multiple of 128 tokens: no library attention is called, and the new tokens
    are the largest of the same model's logits by recomputation, or nearer to them than the two
    paths' bf16 rounding."""
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    from trainium_frontier_b200.ops import reference
    from trainium_frontier_b200.ops._ext import check_errors
    m = _model(cuda_device, head_dim=128)
    with torch.no_grad():
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, 0.2)
    B, N = 3, 8
    prompts = torch.randint(1, 8192, (B, T), device=cuda_device, dtype=torch.int32)

    def library(*a, **k):
        raise AssertionError("library attention")
    with monkeypatch.context() as mp:
        mp.setattr(reference.F, "scaled_dot_product_attention", library)
        out = SpeculativeGenerator(m, B, T + N).generate(prompts, N).long()
    check_errors()
    text = torch.cat([prompts.long(), out], 1)
    with torch.no_grad():
        z = m(torch.nn.functional.pad(text, (0, 256 - T - N)).to(torch.int32))[:, T - 1:T + N - 1].double()
    gap = z.amax(-1) - z.gather(-1, out[..., None])[..., 0]
    # a logit is a product of n_embd terms of a normed state and weights of 0.05, each state off by
    # some roundings of 2^-8 in either path: sqrt(256) * 0.05 * 2^-8 * 8 roundings * 2 paths, four times over
    assert float(gap.max()) <= 4 * 256 ** 0.5 * 0.05 * 2 ** -8 * 16, gap


@pytest.mark.parametrize("head_dim", [64, 128])
def test_speculative_decoding_over_a_quantised_cache(cuda_device, head_dim):
    """Over an e4m3 cache, with right tokens on scattered nodes of a small and of a wide tree: the new
    tokens against logits by recomputation on the CPU with quantised keys and values."""
    import copy

    from tests._specutil import quantised_logits
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    from trainium_frontier_b200.ops._ext import check_errors
    m = _model(cuda_device, head_dim=head_dim)
    with torch.no_grad():
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, 0.2)
    plain = copy.deepcopy(m).cpu()
    plain.set_compute_dtype(torch.float32)
    B, T, N = 3, 128, 10
    prompts = torch.randint(1, 8192, (B, T), device=cuda_device, dtype=torch.int32)
    e4m3 = torch.float8_e4m3fn

    def nothing(text, lens):
        none = torch.empty(B, 0, dtype=torch.int32, device=cuda_device)
        return none, none, None
    one = SpeculativeGenerator(m, B, T + N, nothing, e4m3)
    full = torch.cat([prompts.long(), one.generate(prompts, N).long(), torch.zeros(B, 8, device=cuda_device, dtype=torch.long)], 1)

    def draft_of(n, at, parents):
        def draft(text, lens):
            tok = torch.full((B, n), 3, dtype=torch.int32, device=cuda_device)
            for k, node in enumerate(at):
                tok[:, node - 1] = full.gather(1, (lens.long() + k).clamp_max(full.shape[1] - 1)[:, None])[:, 0].to(torch.int32)
            return tok, torch.tensor([parents] * B, dtype=torch.int32, device=cuda_device), None
        return draft
    for draft in (nothing, draft_of(9, (3, 6, 8), [0, 0, 0, 3, 3, 3, 6, 6, 8]), draft_of(63, (62, 63), [0] * 62 + [62])):
        g = SpeculativeGenerator(m, B, T + N, draft, e4m3)
        out = g.generate(prompts, N).long()
        check_errors()
        assert draft is nothing or g.rounds < N - 1
        text = torch.cat([prompts.long(), out], 1).cpu()
        z = quantised_logits(plain, text, T)[:, T - 1:-1].double()
        gap = z.amax(-1) - z.gather(-1, out.cpu()[..., None])[..., 0]
        # a logit is a product of n_embd terms of a normed state and weights of 0.05, each state off by some
        # roundings of 2^-8: sqrt(256) * 0.05 * 2^-8 * 8 roundings, four times over.  A rounding that moves a
        # key or value entry by 2^-9 of it moves its code by a whole step, 2^-3, in 2^-9 / 2^-3 of the cases:
        # 2^-6 by root mean square, four roundings' worth, twice a block (keys and values), 2 blocks
        assert float(gap.max()) <= 4 * 256 ** 0.5 * 0.05 * 2 ** -8 * (8 + 4 * 2 * 2), gap
