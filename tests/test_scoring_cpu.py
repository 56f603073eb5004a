"""Scoring of sequences and log-probabilities of generated tokens on CPU ranks: against the softmax of the logits, the same on every grid."""

import pytest
import torch

from _dist import run_cached, run_distributed

LENGTHS = [18, 7]


def _model(family, grid, world):
    from axonn_b200 import axonn as ax
    from axonn_b200.models import GPT, GPTConfig, Llama, LlamaConfig

    r, c, d = grid
    ax.init(G_inter=1, G_data=world // (r * c * d), G_intra_r=r, G_intra_c=c, G_intra_d=d)
    torch.manual_seed(4)
    shape = dict(n_layers=2, hidden=64, n_heads=4, ffn=128, vocab=96, seq_len=40)
    model = GPT(GPTConfig(**shape), dtype=torch.float32) if family == "gpt" else Llama(LlamaConfig(n_kv_heads=2, **shape), dtype=torch.float32)
    with torch.no_grad():
        model.head.proj.weight.mul_(30)
    return model


def _tokens():
    return torch.randint(0, 96, (2, 18), generator=torch.Generator().manual_seed(3))


def _lists(told):
    return [None if t is None else (t if t.dtype == torch.int64 else t.detach().double()).tolist() for t in told]


def _score(rank, world, family, grid):
    from axonn_b200.models import score_tokens

    model, tokens = _model(family, grid, world), _tokens()
    whole = score_tokens(model, tokens, entropy=True, top=3)
    cut = score_tokens(model, tokens, LENGTHS, temperature=0.7)
    assert whole.log_probs.shape == (2, 17) and whole.top_tokens.shape == (2, 17, 3) and cut.entropy is None and cut.top_tokens is None
    if grid == (1, 1, 1):
        log_p = model(tokens).detach().double()[:, :-1].log_softmax(-1)
        want = log_p.gather(-1, tokens[:, 1:, None])[..., 0]
        # logits of 30 or so in 32 bits, twice evaluated
        assert (whole.log_probs - want).abs().max() < 30 * 2.0 ** -20 and (whole.entropy + (log_p.exp() * log_p).sum(-1)).abs().max() < 30 * 2.0 ** -20
        assert torch.equal(whole.top_tokens, log_p.topk(3).indices)
        log_p = (model(tokens).detach().double()[:, :-1] / 0.7).log_softmax(-1)
        want = log_p.gather(-1, tokens[:, 1:, None])[..., 0]
        for r, n in enumerate(LENGTHS):
            assert (cut.log_probs[r, :n - 1] - want[r, :n - 1]).abs().max() < 30 * 2.0 ** -19 and cut.log_probs[r, n - 1:].eq(0).all()
        # the sum's gradient is that of the cross-entropy of the same tokens
        g1 = torch.autograd.grad(-score_tokens(model, tokens).log_probs.sum() / 34, list(model.parameters()))
        logits = model(tokens)[:, :-1]
        g2 = torch.autograd.grad(torch.nn.functional.cross_entropy(logits.reshape(34, -1), tokens[:, 1:].reshape(-1)), list(model.parameters()))
        for a, b in zip(g1, g2):
            assert (a - b).norm() <= 1e-4 * b.norm() + 1e-9
    return _lists(whole) + _lists(cut)


@pytest.mark.parametrize("family", ["gpt", "llama"])
def test_scores(family):
    run_cached(_score, 1, family, (1, 1, 1))


def test_scores_are_the_same_on_a_grid():
    ref = run_cached(_score, 1, "gpt", (1, 1, 1))[0]
    for grid, world in (((2, 1, 1), 2), ((2, 2, 1), 4)):
        for got in run_distributed(_score, world, "gpt", grid):
            for a, b in zip(got, ref):
                assert (a is None) == (b is None)
                if a is not None:
                    a, b = torch.tensor(a), torch.tensor(b)
                    assert torch.equal(a, b) if a.dtype == torch.int64 else torch.allclose(a, b, rtol=0, atol=2e-3)


def _generate(rank, world, family, grid):
    from axonn_b200.models import greedy_generate, score_tokens

    model, prompts = _model(family, grid, world), _tokens()[:, :9]
    plain = greedy_generate(model, prompts, 6)
    out, told = greedy_generate(model, prompts, 6, alternatives=4)
    assert torch.equal(out, plain) and told.log_probs.shape == (2, 6) and told.top_tokens.shape == (2, 6, 4) and told.entropy is None
    assert torch.equal(told.top_tokens[..., 0], out[:, 9:]) and torch.equal(told.top_log_probs[..., 0], told.log_probs)
    scored = score_tokens(model, out).log_probs[:, 8:].detach()
    assert (told.log_probs - scored).abs().max() < 30 * 2.0 ** -19
    bare = greedy_generate(model, prompts, 6, alternatives=0)[1]
    assert torch.equal(bare.log_probs, told.log_probs) and bare.top_tokens is None
    eos = int(out[0, 10])                                 # the first row ends with its second new token
    ended, part = greedy_generate(model, prompts, 6, eos_id=eos, alternatives=2)
    n = part.log_probs.shape[1]
    assert ended.shape[1] == 9 + n and torch.equal(part.log_probs[0, :2], told.log_probs[0, :2])
    assert part.log_probs[0, 2:].eq(0).all() and part.top_tokens[0, 2:].eq(-1).all()
    cached, near = greedy_generate(model, prompts, 6, cache_dtype=torch.int8, alternatives=4)
    assert cached.shape == out.shape and near.log_probs.shape == (2, 6) and near.log_probs.le(0).all() and torch.equal(near.top_tokens[..., 0], cached[:, 9:])
    none = greedy_generate(model, prompts, 0, cache_dtype=torch.int8, alternatives=4)[1]
    assert none.log_probs.shape == (2, 0) and none.top_tokens.shape == (2, 0, 4)
    assert model.training
    return out.tolist()


@pytest.mark.parametrize("family", ["gpt", "llama"])
def test_generated_tokens(family):
    run_distributed(_generate, 1, family, (1, 1, 1))


def test_generated_tokens_on_a_grid():
    run_distributed(_generate, 2, "llama", (2, 1, 1))


def _refusals(rank, world):
    from axonn_b200.models import greedy_generate, score_tokens

    model, tokens = _model("gpt", (1, 1, 1), 1), _tokens()
    for bad in (lambda: score_tokens(model, tokens.int()), lambda: score_tokens(model, tokens[:, :1]), lambda: score_tokens(model, tokens[0]),
                lambda: score_tokens(model, tokens, [18]), lambda: score_tokens(model, tokens, top=33),
                lambda: greedy_generate(model, tokens, 2, alternatives=33), lambda: greedy_generate(model, tokens, 2, alternatives=-1)):
        with pytest.raises(ValueError):
            bad()


def test_refusals():
    run_distributed(_refusals, 1)
