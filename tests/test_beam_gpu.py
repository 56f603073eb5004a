"""The selection kernel of beam search against the 64-bit form on the CPU."""

import pytest
import torch

from axonn_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _same(logits, scores, done=None, eos=None):
    want = ops.beam_select(logits, scores, done, eos)
    got = ops.beam_select(logits.to(DEV), scores.to(DEV), None if done is None else done.to(DEV), eos)
    assert torch.equal(got.tokens.cpu(), want.tokens) and torch.equal(got.parents.cpu(), want.parents)
    if done is None:
        assert got.done is None
    else:
        assert torch.equal(got.done.cpu(), want.done)
    # rounded once to 32 bits; the sum's relative error in 32 bits (V 2^-24 at worst, 2^-20 of what is met) is the logarithm's absolute one
    finite = want.scores.isfinite()
    assert torch.equal(got.scores.cpu()[~finite], want.scores[~finite])
    assert bool(((got.scores.cpu() - want.scores).abs()[finite] <= 2.0 ** -23 * want.scores[finite].abs() + 2.0 ** -20).all())
    return got


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 4, 255), (3, 2, 257), (2, 5, 2048), (1, 8, 2049), (2, 4, 32000), (1, 32, 1000),
                                   (3, 7, 50304), (1, 4, 128256), (40, 8, 4001), (2, 32, 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_select(B, K, V, dtype):
    """One value to many parts, odd vocabularies, fewer tokens than beams; 16-bit logits have many equal values."""
    g = torch.Generator().manual_seed(V + K)
    logits = (torch.randn(B, K, V, generator=g) * 2).to(dtype)
    scores = -10 * torch.rand(B, K, generator=g)
    _same(logits, scores)
    done = torch.rand(B, K, generator=g) < 0.4
    _same(logits, scores, done, V // 2)
    scores[:, 1:] = float("-inf")                      # the first step
    _same(logits, scores, torch.zeros(B, K, dtype=torch.bool), 0)


@pytest.mark.parametrize("V", [700, 701, 5000])
def test_ties_go_to_the_lowest_beam_and_token(V):
    """Equal rows have equal sums, however they are aligned, and equal values the order of (beam, token)."""
    logits = torch.zeros(2, 4, V).bfloat16()
    got = _same(logits, torch.zeros(2, 4))
    assert got.parents.tolist() == [[0] * 4] * 2 and got.tokens.tolist() == [[0, 1, 2, 3]] * 2
    row = (torch.randn(V, generator=torch.Generator().manual_seed(0)) * 2).round().bfloat16()
    row[5], row[V - 3] = 20.0, -0.0
    got = _same(row.expand(2, 4, V).contiguous(), torch.zeros(2, 4))
    assert got.parents.tolist() == [[0, 1, 2, 3]] * 2 and got.tokens.tolist() == [[5] * 4] * 2
    row = torch.full((V,), -5.0)                       # zeros of both signs are equal
    row[3::5], row[::7] = 0.0, -0.0
    _same(row.expand(1, 6, V).contiguous(), torch.tensor([[0.0, -1, -2, -3, -4, -5]]))


def test_values_that_are_no_numbers():
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(6, 3, 300, generator=g)
    scores = -torch.rand(6, 3, generator=g)
    logits[0, 1, 7], logits[1, 0, 299], logits[2, 2] = nan, inf, -inf
    logits[3, :, 2:] = -inf                            # six values, then -inf in the order of the tokens
    logits[4] = -inf
    scores[5] = torch.tensor([nan, -inf, inf])
    _same(logits, scores)
    done = torch.zeros(6, 3, dtype=torch.bool)
    done[:, 1] = True
    scores[5] = torch.tensor([-inf, -inf, nan])
    _same(logits, scores, done, 4)
    got = _same(logits[4:5], scores[4:5], done[4:5], 4)
    assert got.tokens[0, 0] == 4 and got.parents[0, 0] == 1 and got.tokens[0, 1:].tolist() == [0, 1]


def test_logits_of_all_sizes():
    """Rows whose maximum grows along the row, falls along it, and large values: the sums' references move."""
    V = 40000
    up = torch.linspace(-3e4, 3e4, V)
    rows = torch.stack([up, up.flip(0), torch.full((V,), -3e38), torch.full((V,), 3e38), up * 1e30])
    _same(rows[None].contiguous(), torch.tensor([[-1.0, -2.0, 1.0, -3.0, -4.0]]))


def test_views_of_larger_tensors():
    """The last position of [prompts, beams, S, V] logits (copied), rows off 16 bytes."""
    g = torch.Generator().manual_seed(0)
    wide = torch.randn(2, 3, 4, 1000, generator=g).bfloat16()
    scores = -torch.rand(2, 3, generator=g)
    want = _same(wide[:, :, -1].contiguous(), scores)
    got = ops.beam_select(wide.to(DEV)[:, :, -1], scores.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))
    off = torch.empty(6001, dtype=torch.bfloat16, device=DEV)[1:].view(2, 3, 1000).copy_(wide[:, :, -1])
    got = ops.beam_select(off, scores.to(DEV))
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.parents, want.parents)


def test_select_in_graphs_on_two_streams():
    torch.manual_seed(0)
    logits = [torch.randn(2, 4, 30011, device=DEV) for _ in range(2)]
    scores = torch.zeros(2, 4, device=DEV)
    want = [ops.beam_select(x, scores) for x in logits]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x in logits:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.beam_select(x, scores))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o[:3], w[:3]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_masked_by_the_lowest_value(dtype):
    """Banned tokens as the type's lowest value or -inf, all of a row or of a part of it, in the first parts and the last."""
    low = torch.finfo(dtype).min
    logits = (torch.randn(2, 4, 20000, generator=torch.Generator().manual_seed(0)) * 2).to(dtype)
    logits[0, 0], logits[0, 1, :9000], logits[0, 2, 9000:], logits[0, 3, 1:] = low, low, low, low
    logits[1, 0], logits[1, 1, :9000], logits[1, 2, 9000:], logits[1, 3, 1:] = float("-inf"), float("-inf"), float("-inf"), float("-inf")
    _same(logits, torch.tensor([[0.0, -1.0, -2.0, -3.0]] * 2))
    _same(logits[:, :1].contiguous(), torch.zeros(2, 1))
    _same(logits[:1, :1].repeat(1, 32, 1).contiguous(), -torch.rand(1, 32, generator=torch.Generator().manual_seed(1)))
