"""Full-recompute greedy decoding on the CPU oracle path."""
import torch

from trainium_frontier_b200.config import preset
from trainium_frontier_b200.inference.generate import generate_reference
from trainium_frontier_b200.models.gpt import GPT


def test_generate_reference_shapes_and_determinism():
    cfg = preset("tiny", depth=2)
    torch.manual_seed(0)
    m = GPT(cfg.model_config(), cfg)
    m.init_weights()
    p = torch.randint(1, 8192, (2, 16))
    a = generate_reference(m, p, 5)
    b = generate_reference(m, p, 5)
    assert a.shape == (2, 5) and torch.equal(a, b)


def _small_model(seed=0):
    cfg = preset("tiny", depth=2)
    torch.manual_seed(seed)
    m = GPT(cfg.model_config(), cfg)
    m.init_weights()
    with torch.no_grad():   # a non-degenerate random model (zero-init projections otherwise)
        for b in m.transformer.h:
            b.mlp.c_proj.weight.normal_(0, 0.02)
        m.lm_head.weight.normal_(0, 0.05)
    return m.eval()


def test_speculative_greedy_is_greedy():
    """Whatever the draft proposes -- the right tokens, wrong ones, a tree of both, nothing --
    greedy speculative decoding gives plain greedy decoding's tokens."""
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator, ngram_draft
    m = _small_model()
    p = torch.randint(1, 8192, (3, 16))
    n = 12
    want = generate_reference(m, p, n)

    def oracle(text, lens):     # right tokens on one branch (node 2, 3, 5), wrong ones beside it
        full = torch.cat([p, want], 1)
        tok = torch.randint(0, 8192, (3, 5), dtype=torch.int32)
        for b in range(3):
            rest = full[b, int(lens[b]):][:3].tolist()
            for k, node in enumerate((2, 3, 5)):
                if k < len(rest):
                    tok[b, node - 1] = rest[k]
        return tok, torch.tensor([[0, 0, 2, 2, 3]] * 3, dtype=torch.int32), None

    def nothing(text, lens):
        return torch.full((3, 2), -1, dtype=torch.int32), torch.full((3, 2), -2, dtype=torch.int32), None
    for draft, most in ((oracle, 4), (nothing, n - 1), (ngram_draft(4), n - 1)):
        g = SpeculativeGenerator(m, 3, 64, draft)
        assert torch.equal(g.generate(p, n).long(), want.long())
        assert g.rounds <= most


def test_speculative_sampling_draws_from_the_target():
    """Sampled with a draft distribution that is not the target's: the first two tokens'
    frequencies over many sequences follow the target's within 5 standard deviations."""
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    m = _small_model(1)
    M = 600
    p = torch.randint(1, 8192, (1, 4)).expand(M, 4).contiguous()
    with torch.no_grad():
        law = torch.softmax(m(p[:1])[0, -1] / 0.1, -1)
    g = torch.Generator().manual_seed(3)

    def draft(text, lens):
        q = torch.softmax(torch.randn(1, 1, 8192, generator=g), -1).expand(M, 3, 8192).contiguous()
        tok = torch.multinomial(q[:, :2].reshape(-1, 8192), 1, generator=g).view(M, 2).to(torch.int32)
        return tok, torch.tensor([[0, 1]] * M, dtype=torch.int32), q
    out = SpeculativeGenerator(m, M, 16, draft).generate(p, 3, 0.1, g)
    top = law.argmax()
    share, want = (out[:, 0] == top).double().mean(), law[top].double()
    assert abs(share - want) <= 5 * (want * (1 - want) / M).sqrt()


def _attending_model():
    m = _small_model()
    with torch.no_grad():   # the tokens depend on the attention
        for b in m.transformer.h:
            b.attn.c_proj.weight.normal_(0, 0.2)
    return m


def test_speculative_greedy_depends_on_the_cache():
    """Plain greedy tokens where the attention decides them, with drafts by rule and with right
    and wrong branches."""
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator, ngram_draft
    m = _attending_model()
    p = torch.randint(1, 8192, (2, 10))
    full = torch.cat([p, generate_reference(m, p, 12)], 1)
    other = p.clone()
    other[:, :9] = torch.randint(1, 8192, (2, 9))   # the same last token: only attention tells the texts apart
    assert not torch.equal(generate_reference(m, other, 4), full[:, 10:14])

    def draft(text, lens):
        tok = torch.full((2, 5), 3, dtype=torch.int32)
        for b in range(2):
            for k, t in enumerate(full[b, int(lens[b]):][:3].tolist()):
                tok[b, (1, 2, 4)[k]] = t
        return tok, torch.tensor([[0, 0, 2, 2, 3]] * 2, dtype=torch.int32), None
    for d in (draft, ngram_draft(4)):
        assert torch.equal(SpeculativeGenerator(m, 2, 40, d).generate(p, 12).long(), full[:, 10:].long())


def test_speculative_tree_reaches_past_the_end():
    """The right tokens on the last nodes of a wide tree, and no room beyond the text's end: the
    tree's rows go past it, and greedy decoding still gives plain greedy decoding's tokens."""
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    m = _attending_model()
    p = torch.randint(1, 8192, (2, 10))
    for n in (2, 3, 4, 9):
        full = torch.cat([p, generate_reference(m, p, n)], 1)

        def draft(text, lens):
            tok = torch.full((2, 63), 3, dtype=torch.int32)
            for b in range(2):
                rest = full[b, int(lens[b]):][:2].tolist()
                for k, t in enumerate(rest):
                    tok[b, 61 + k] = t
            return tok, torch.tensor([[0] * 62 + [62]] * 2, dtype=torch.int32), None
        assert torch.equal(SpeculativeGenerator(m, 2, 10 + n, draft).generate(p, n).long(), full[:, 10:].long())


def test_speculative_tokens_outside_the_vocabulary():
    """A draft's tokens outside the vocabulary are read nowhere and never accepted."""
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    m = _attending_model()
    p = torch.randint(1, 8192, (2, 10))
    for bad in (8192, 2 ** 31 - 1, -5):
        draft = lambda text, lens: (torch.full((2, 2), bad, dtype=torch.int32),  # noqa: E731
                                    torch.tensor([[0, 1]] * 2, dtype=torch.int32), None)
        assert torch.equal(SpeculativeGenerator(m, 2, 32, draft).generate(p, 4).long(), generate_reference(m, p, 4).long())


def test_speculative_quantised_cache_runs():
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    m = _small_model()
    p = torch.randint(1, 8192, (2, 9))
    out = SpeculativeGenerator(m, 2, 40, kv_dtype=torch.float8_e4m3fn).generate(p, 10)
    assert out.shape == (2, 10) and int(out.min()) >= 0


def test_speculative_refusals():
    import pytest

    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    m = _small_model()
    with pytest.raises(ValueError):
        SpeculativeGenerator(m, 2, m.config.sequence_len + 1)
    g = SpeculativeGenerator(m, 2, 32)
    with pytest.raises(ValueError):
        g.generate(torch.ones(1, 4, dtype=torch.long), 2)
    with pytest.raises(ValueError):
        g.generate(torch.ones(2, 30, dtype=torch.long), 8)
    with pytest.raises(ValueError):
        g.generate(torch.ones(2, 3, dtype=torch.long), 0)


def test_ngram_draft():
    from trainium_frontier_b200.inference.speculative import ngram_draft
    text = torch.zeros(4, 12, dtype=torch.long)
    text[0, :8] = torch.tensor([5, 6, 7, 8, 5, 6, 9, 9])     # ends in a pair never seen before
    text[1, :9] = torch.tensor([1, 2, 3, 4, 1, 2, 7, 1, 2])  # latest earlier "1 2" is at 4
    text[2, :1] = 3                                          # shorter than the order
    text[3, :12] = 4                                         # one token over and over, to the end of the row
    lens = torch.tensor([8, 9, 1, 12], dtype=torch.int32)
    tok, par, q = ngram_draft(3)(text, lens)
    assert q is None
    assert tok.tolist() == [[-1] * 3, [7, 1, 2], [-1] * 3, [4, -1, -1]]
    assert par.tolist() == [[-2] * 3, [0, 1, 2], [-2] * 3, [0, -2, -2]]


def test_speculative_sampling_follows_the_target_token_by_token(monkeypatch):
    """Sampled with a draft whose distributions overlap the target's (two siblings and a child, drawn
    from flattened rows of the same model): the second and third tokens follow the target's law given
    the most common tokens before them.  Each share of a token is within 5 standard deviations,
    sqrt(p (1 - p) / n), of p, over the tokens that are expected 10 times or more."""
    from trainium_frontier_b200 import ops
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    m = _attending_model()
    M, T, n, temp = 800, 4, 4, 0.12
    p = torch.randint(1, 8192, (1, T), generator=torch.Generator().manual_seed(4)).expand(M, T).contiguous()
    g = torch.Generator().manual_seed(3)
    rows = torch.arange(M)

    def law(text, at, t):
        with torch.no_grad():
            return torch.softmax(m(text)[torch.arange(len(text)), at] / t, -1)

    def draft(text, lens):
        ln = lens.long()
        q = torch.full((M, 4, 8192), 1 / 8192)    # no token was drawn from the rows of nodes 2 and 3
        q[:, 0] = law(text, ln - 1, 2 * temp)
        tok = torch.empty(M, 3, dtype=torch.int32)
        tok[:, :2] = torch.multinomial(q[:, 0], 2, replacement=True, generator=g)
        longer = text.clone()
        longer[rows, ln] = tok[:, 0].long()
        q[:, 1] = law(longer, ln, 2 * temp)       # node 1's children
        tok[:, 2] = torch.multinomial(q[:, 1], 1, generator=g)[:, 0]
        return tok, torch.tensor([[0, 0, 1]] * M, dtype=torch.int32), q
    taken, verify = [], ops.verify_tree

    def counting(*a):
        res = verify(*a)
        if a[0].shape[1] > 1:
            taken.append(res)
        return res
    monkeypatch.setattr(ops, "verify_tree", counting)
    out = SpeculativeGenerator(m, M, T + n + 2, draft).generate(p, n, temp, g).long()
    counts = torch.stack([c for _, c, _ in taken])
    assert int((counts == 1).sum()) > M // 10 and int((counts == 2).sum()) > M // 10 and int((counts == 3).sum()) > M // 10
    second = torch.cat([path[count > 1][:, 1] for path, count, _ in taken])
    assert int((second == 2).sum()) > M // 50   # the first sibling rejected, the second one accepted
    text, some, checked = p[:1], out, []
    for i in range(3):
        want = law(text, torch.tensor([T + i - 1]), temp)[0].double()
        share = torch.bincount(some[:, i], minlength=8192).double() / len(some)
        seen = want * len(some) >= 10
        checked.append(int(seen.sum()))
        assert bool(((share - want).abs() <= 5 * (want * (1 - want) / len(some)).sqrt())[seen].all()), i
        top = share.argmax()
        some = some[some[:, i] == top]
        text = torch.cat([text, top.view(1, 1)], 1)
    assert min(checked) >= 2


def test_speculative_quantised_cache_reads_what_it_wrote():
    """Over an e4m3 cache one token a round gives the tokens of a recomputation with quantised keys and
    values.  A node reads the same rows in a tree, so trees with the right tokens on scattered nodes,
    and the draft by rule, give the same, in fewer rounds."""
    from tests._specutil import quantised_logits
    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator, ngram_draft
    m = _attending_model()
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():   # value rows of very unequal sizes, and so of unequal scales
        for b in m.transformer.h:
            b.attn.c_v.weight.mul_(torch.exp2(torch.randint(-3, 4, b.attn.c_v.weight.shape[:1], generator=g).float())[:, None])
        m.transformer.wte.weight.mul_(torch.exp2(torch.randint(-3, 4, (1, m.transformer.wte.weight.shape[1]), generator=g).float()))
    p = torch.randint(1, 8192, (3, 10), generator=g)
    n, e4m3 = 14, torch.float8_e4m3fn

    def nothing(text, lens):
        return torch.empty(3, 0, dtype=torch.int32), torch.empty(3, 0, dtype=torch.int32), None
    want = SpeculativeGenerator(m, 3, 32, nothing, e4m3).generate(p, n)
    assert not torch.equal(want.long(), generate_reference(m, p, n))      # the rounding of the cache matters here
    full = torch.cat([p, want.long()], 1)
    assert torch.equal(quantised_logits(m, full, 10)[:, 9:-1].argmax(-1), want.long())

    def draft(text, lens):
        tok = torch.full((3, 9), 3, dtype=torch.int32)
        for b in range(3):
            for k, t in enumerate(full[b, int(lens[b]):][:3].tolist()):
                tok[b, (2, 5, 7)[k]] = t                                  # nodes 3, 6 and 8
        return tok, torch.tensor([[0, 0, 0, 3, 3, 3, 6, 6, 8]] * 3, dtype=torch.int32), None
    for d, most in ((draft, 5), (ngram_draft(4), n - 1)):
        s = SpeculativeGenerator(m, 3, 32, d, e4m3)
        assert torch.equal(s.generate(p, n), want)
        assert s.rounds <= most


def test_speculative_prompts_outside_the_vocabulary_are_refused():
    import pytest

    from trainium_frontier_b200.inference.speculative import SpeculativeGenerator
    g = SpeculativeGenerator(_small_model(), 2, 32)
    for bad in (8192, -1, 2 ** 31 - 1):
        p = torch.ones(2, 4, dtype=torch.int32)
        p[1, 2] = bad
        with pytest.raises(ValueError, match="prompts"):
            g.generate(p, 2)
