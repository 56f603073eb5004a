"""Calls of the vocabulary's operators, and of the layers and functions on them, at the ends of what they take: on the CPU."""

import shutil

import pytest
import torch

from axonn_b200 import ops
from axonn_b200.ops import _lib

from _dist import run_distributed
from _vocabulary_ends import COLD, HOT, check_ends_of_temperature, ends_of_temperature


def _grid(world, depth=1):
    from axonn_b200 import axonn as ax

    ax.init(G_inter=1, G_data=world // depth, G_intra_r=1, G_intra_c=1, G_intra_d=depth)


def _rows_outside(rank, world):
    """A device whose lookups look at no index (on a GPU torch's ends the program) is never asked for rows that the table has not got."""
    from axonn_b200.intra_layer import Embedding

    _grid(world)
    for scale in (1.0, 2.0):
        layer = Embedding(40, 8, expert_mode=True, scale=scale)
        there = layer.rows(23, 17, "cpu")
        for device in ("cpu", "meta"):
            layer = layer.to(device)
            for grad in (False, True):
                with torch.set_grad_enabled(grad):
                    for first, count in ((24, 17), (-1, 2), (40, 1), (1 << 40, 3)):
                        with pytest.raises(IndexError):
                            layer.rows(first, count, device)
                        with pytest.raises(IndexError), torch.device("meta"):       # whatever the default device is
                            layer.rows(first, count, device)
                    assert layer.rows(23, 17, device).shape == (17, 8) and layer.rows(0, 40, device).shape == (40, 8)
                    for first in (0, 40, 50):
                        assert layer.rows(first, 0, device).shape == (0, 8)
    assert there.shape == (17, 8)


def test_rows_that_the_table_has_not_got():
    run_distributed(_rows_outside, 1)


def _model(family, vocab=96, seq_len=40):
    from axonn_b200.models import GPT, GPTConfig, Llama, LlamaConfig

    torch.manual_seed(4)
    shape = dict(n_layers=2, hidden=64, n_heads=4, ffn=128, vocab=vocab, seq_len=seq_len)
    return GPT(GPTConfig(**shape), dtype=torch.float32) if family == "gpt" else Llama(LlamaConfig(n_kv_heads=2, **shape), dtype=torch.float32)


def _scores_of_long_sequences(rank, world):
    """A model that has learned its positions refuses more of them before it looks any up; rotary ones go on."""
    from axonn_b200.models import score_tokens

    _grid(world)
    g = torch.Generator().manual_seed(0)
    for family in ("gpt", "llama"):
        model = _model(family, seq_len=12)
        for length in (11, 12, 13, 20):
            tokens = torch.randint(0, 96, (2, length), generator=g)
            if family == "gpt" and length > 12:
                model.pos_emb.register_forward_pre_hook(lambda *_: pytest.fail("positions are looked up"))
                with pytest.raises(ValueError, match="12"):
                    score_tokens(model, tokens)
                with pytest.raises(ValueError, match="12"):
                    score_tokens(model, tokens, lengths=[12, 3])
            else:
                assert score_tokens(model, tokens).log_probs.shape == (2, length - 1)


def test_scores_of_long_sequences():
    run_distributed(_scores_of_long_sequences, 1)


def _padding_outside_the_table(rank, world, family):
    """What stands behind the rows' ends is no token: any number may, and the results do not see it."""
    from axonn_b200.models import beam_generate, greedy_generate, score_tokens

    _grid(world)
    model, g = _model(family), torch.Generator().manual_seed(0)
    tokens, lengths = torch.randint(0, 96, (3, 14), generator=g), torch.tensor([14, 5, 1])
    behind = torch.arange(14) >= lengths[:, None]
    calls = [lambda t: score_tokens(model, t, lengths, entropy=True, top=3), lambda t: score_tokens(model, t, lengths.tolist()),
             lambda t: (greedy_generate(model, t, 4, cache_dtype=torch.int8, prompt_lengths=lengths),),
             lambda t: beam_generate(model, t, 4, 3, cache_dtype=torch.int8, prompt_lengths=lengths)]
    for call in calls:
        want = call(tokens.masked_fill(behind, 0))
        for pad in (-1, -100, 96, 1 << 40, 7):
            given = tokens.masked_fill(behind, pad)
            kept = given.clone()
            got = call(given)
            assert torch.equal(given, kept)
            for a, b in zip(got, want):
                assert (a is None) == (b is None) and (a is None or torch.equal(a, b)), pad
    for bad in (lambda: score_tokens(model, tokens.masked_fill(tokens == tokens[0, 3], 96), lengths),
                lambda: score_tokens(model, tokens.masked_fill(behind, -1))):
        with pytest.raises(IndexError):                   # within the rows there are tokens only
            bad()


@pytest.mark.parametrize("family", ["gpt", "llama"])
def test_padding_outside_the_table(family):
    run_distributed(_padding_outside_the_table, 1, family)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("temperature", [COLD, HOT])
def test_ends_of_the_temperature(dtype, temperature):
    check_ends_of_temperature(*ends_of_temperature(dtype, "cpu"), temperature)


def test_temperatures_that_are_refused():
    """32 bits hold neither the factor 1 / temperature nor that with log2 e at some positive numbers: NaN for a maximum, for what is masked."""
    logits, tokens = ends_of_temperature(torch.float32, "cpu")
    for temperature in (1e-39, 3e-39, 1e-38, COLD / 2, 2 * HOT, 9e37, 1e38, 3e38, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_log_probs(logits, tokens, temperature=temperature)


@pytest.mark.skipif(not (_lib.available() or shutil.which("nvcc")), reason="native library not built")
def test_factors_that_the_launchers_refuse():
    """Addresses that are never used: the calls are refused on the host."""
    L, p = _lib.lib(), 4096
    for scale in (2.0 ** 101, 2.0 ** -101, 3e38, 1e-39, float("inf"), float("nan"), 0.0, -1.0):
        for call in (lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, p, p, p, 1, 1, 8, 0, 8, 0, scale, -100, 1, 0, None),
                     lambda: L.axb_token_log_probs_bwd(p, 8, 8, p, 1, 1, p, p, p, p, p, p, 1, 1, 8, 0, 8, 0, scale, -100, 0, None)):
            assert call() == -1 and b"scale" in L.axb_last_error()


def test_batched_gradients():
    """Of a lookup as of torch.nn.functional.embedding; of log-probabilities they are refused."""
    tokens, w = torch.tensor([1, 4, 1, 0]), torch.randn(6, 3, requires_grad=True)
    dy = torch.randn(5, 4, 3)
    (got,) = torch.autograd.grad(ops.embedding(tokens, w, 2.0, 4), w, dy, is_grads_batched=True)
    want = torch.zeros(5, 6, 3).index_add(1, tokens[[0, 2, 3]], 2 * dy[:, [0, 2, 3]])
    assert torch.equal(got, want)
    z = torch.randn(4, 9, requires_grad=True)
    for entropy in (False, True):
        r = ops.token_log_probs(z, tokens, entropy=entropy)
        with pytest.raises(RuntimeError, match="batched gradients"):
            torch.autograd.grad(r.entropy if entropy else r.log_probs, z, torch.randn(3, 4), is_grads_batched=True)


def _scaled_layers(rank, world, depth):
    """The scale on every way that rows are looked up: the table gathered over depth ranks or not, torch's own lookup where a layer asks for
    what the package's does not do, rows fetched from the owning ranks (a stub here)."""
    from axonn_b200.intra_layer import Embedding, embedding
    from axonn_b200.intra_layer.communication import _gather

    _grid(world, depth)
    g = torch.Generator().manual_seed(5)
    table, tokens = torch.randn(12, 8, generator=g), torch.randint(0, 12, (3, 7), generator=g)
    dy = torch.randn(3, 7, 8, generator=g)
    for kw in (dict(), dict(padding_idx=3), dict(scale_grad_by_freq=True), dict(dtype=torch.float64)):
        layer = Embedding(12, 8, expert_mode=True, scale=2.5, **kw)
        layer.load_state_dict({"weight": table.to(layer.weight.dtype)})
        want = torch.nn.Embedding(12, 8, _weight=table.to(layer.weight.dtype).clone(), **{k: v for k, v in kw.items() if k != "dtype"})
        out, ref = layer(tokens), want(tokens) * 2.5
        assert torch.equal(out, ref)
        out.backward(dy.to(out.dtype))
        ref.backward(dy.to(ref.dtype))
        grad = layer.weight.grad if depth == 1 else _gather(layer.weight.grad, 0, layer.depth_group)
        # every depth rank has the same tokens here, and their gradients are summed
        assert torch.allclose(grad.view(12, 8), depth * want.weight.grad, rtol=1e-6, atol=1e-6)
        assert torch.equal(layer.rows(2, 5, "cpu"), want.weight.detach()[2:7] * 2.5)
    with torch.no_grad():
        long = Embedding(12, 8, expert_mode=True, scale=2.5, max_norm=1.0)
        long.load_state_dict({"weight": table})
        assert torch.equal(long(tokens), torch.nn.functional.embedding(tokens, table.clone(), max_norm=1.0) * 2.5)
    layer = Embedding(12, 8, expert_mode=True, scale=2.5)
    layer._p2p_rows, kept = (lambda x: True), embedding._EmbeddingRowsP2P
    embedding._EmbeddingRowsP2P = type("Fetched", (), {"apply": staticmethod(lambda x, *_: table[x])})
    try:
        assert torch.equal(layer(tokens), table[tokens] * 2.5)
    finally:
        embedding._EmbeddingRowsP2P = kept


@pytest.mark.parametrize("depth", [1, 2])
def test_scaled_layers(depth):
    run_distributed(_scaled_layers, depth, depth)
