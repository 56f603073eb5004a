"""``token_log_probs`` on the CPU: results, gradients, refusals, and a vocabulary that is split over ranks."""

import math

import pytest
import torch

from axonn_b200 import ops

from _dist import run_distributed
from _vocabulary import check_gradient, check_told, told, told_gradient

INF, NAN = float("inf"), float("nan")


def _case(shape, dtype, seed=0, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    logits = (3 * torch.randn(shape, generator=g)).to(dtype)
    tokens = torch.randint(0, shape[-1], shape[:-1], generator=g)
    tokens[torch.rand(shape[:-1], generator=g) < ignored] = -100
    return logits, tokens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,top", [((7,), 3), ((1, 1), 1), ((4, 33), 0), ((3, 5, 100), 32), ((2, 3, 2, 17), 5), ((0, 9), 2), ((2, 0, 9), 2)])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_told(shape, top, dtype, temperature):
    logits, tokens = _case(shape, dtype)
    logits.requires_grad_()
    got = ops.token_log_probs(logits, tokens, entropy=True, top=top, temperature=temperature)
    want = told(logits, tokens, top, temperature)
    check_told(got, want, shape[-1], top)
    assert (got.top_tokens is None) == (top == 0)
    d = [torch.randn(t.shape) for t in got[:3] if t is not None]
    (grad,) = torch.autograd.grad([t for t in got[:3] if t is not None], logits, d)
    check_gradient(grad, *told_gradient(logits, tokens, d[0], d[1], d[2] if top else None, temperature), shape[-1], want["log_p"])


def test_gradients_by_differences():
    """The sum of everything that can be differentiated, moved along a direction: 32-bit results, so a large step of central differences."""
    logits, tokens = _case((3, 19), torch.float32)
    a, b, c = torch.randn(3), torch.randn(3), torch.randn(3, 4)

    def value(z):
        w = told(z, tokens, 4, 0.7)
        return (w["log_probs"] * a).sum() + (w["entropy"] * b).sum() + (w["top_log_probs"] * c).sum()

    logits = logits.sort(-1).values                       # the order of the alternatives stays
    logits += torch.arange(19) * 0.1
    logits.requires_grad_()
    r = ops.token_log_probs(logits, tokens, entropy=True, top=4, temperature=0.7)
    ((r.log_probs * a).sum() + (r.entropy * b).sum() + (r.top_log_probs * c).sum()).backward()
    u = torch.randn(3, 19, dtype=torch.float64)
    step = 1e-4                                           # third derivatives of size 10: 1e-7 off
    z = logits.detach().double()
    by = (value(z + step * u) - value(z - step * u)) / (2 * step)
    assert abs(float((logits.grad * u).sum()) - float(by)) < 1e-4 * (1 + abs(float(by)))


def test_rows_without_a_distribution_and_masks():
    logits = torch.zeros(6, 8)
    logits[0] = -INF
    logits[1, 3] = NAN
    logits[2, 5] = INF
    logits[3, 1:] = -INF
    logits[4] = torch.finfo(torch.float32).min
    logits[5, ::2] = torch.finfo(torch.float32).min
    tokens = torch.tensor([0, 1, 5, 0, 7, 1])
    got = ops.token_log_probs(logits, tokens, entropy=True, top=8)
    check_told(got, told(logits, tokens, 8), 8, 8)
    assert got.log_probs[:3].isnan().all() and got.log_probs[3] == 0 and got.entropy[3] == 0
    assert abs(float(got.log_probs[4]) + math.log(8)) < 1e-6
    assert got.top_tokens[3].tolist() == list(range(8)) and got.top_log_probs[3, 1:].eq(-INF).all()
    assert got.top_tokens[1, 0] == 3                       # a NaN is the largest
    none = ops.token_log_probs(logits, entropy=True)
    assert none.log_probs is None and none.top_tokens is None and torch.equal(none.entropy.nan_to_num(), got.entropy.nan_to_num())


def test_tokens_outside_the_vocabulary():
    logits = torch.randn(4, 5, requires_grad=True)
    r = ops.token_log_probs(logits, torch.tensor([5, -1, -100, 2]), entropy=True)
    assert r.log_probs.isnan().tolist() == [True, True, False, False] and r.log_probs[2] == 0 and r.entropy.isfinite().all()
    (g,) = torch.autograd.grad(r.log_probs.sum(), logits, retain_graph=True)
    assert g.isnan().all(-1).tolist() == [True, True, False, False] and g[2].eq(0).all()
    (g,) = torch.autograd.grad(r.entropy.sum(), logits)
    assert g.isfinite().all() and g[2].eq(0).all()
    r = ops.token_log_probs(logits, torch.tensor([0, 0, 1, 2]), ignore_index=0)
    assert r.log_probs[:2].eq(0).all()


def test_refusals():
    z, t = torch.randn(2, 5), torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: ops.token_log_probs(z.double(), t), lambda: ops.token_log_probs(z, t.int()), lambda: ops.token_log_probs(z, t[:1]),
                lambda: ops.token_log_probs(z), lambda: ops.token_log_probs(z, t, top=6), lambda: ops.token_log_probs(z, t, top=-1),
                lambda: ops.token_log_probs(torch.randn(1, 100), t[:1], top=33), lambda: ops.token_log_probs(z, t, temperature=0.0),
                lambda: ops.token_log_probs(z, t, temperature=NAN), lambda: ops.token_log_probs(z, t, temperature=-1.0),
                lambda: ops.token_log_probs(z, t, temperature=INF), lambda: ops.token_log_probs(z, t, temperature=1e-60),
                lambda: ops.token_log_probs(z[:, :0], t), lambda: ops.token_log_probs(torch.tensor(1.0), torch.tensor(0))):
        with pytest.raises(ValueError):
            bad()
    z.requires_grad_()
    r = ops.token_log_probs(z, t)
    (g,) = torch.autograd.grad(r.log_probs.square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


def _split(rank, world):
    import torch.distributed as dist

    g = torch.Generator().manual_seed(5)
    V = 24
    whole = torch.randn(9, V * world, generator=g).bfloat16()
    whole[:, 3] = whole[:, V * world - 2]                 # ties over ranks
    whole[1, :V] = -INF                                   # nothing in the first slice
    whole[2] = -INF
    whole[3, V + 2] = NAN
    whole[4, 1] = INF
    whole[5, 2:] = -INF
    tokens = torch.randint(0, V * world, (9,), generator=g)
    tokens[5], tokens[6], tokens[7], tokens[8] = 0, -100, V * world, V * world - 1
    mine = whole[:, rank * V:(rank + 1) * V].clone().requires_grad_()
    got = ops.token_log_probs(mine, tokens, entropy=True, top=7, temperature=0.9, group=dist.group.WORLD)
    want = told(whole, tokens, 7, 0.9)
    check_told(got, want, V * world, 7)
    d = [torch.randn(t.shape, generator=g) for t in got[:3]]
    (grad,) = torch.autograd.grad(got[:3], mine, d)
    full, size = told_gradient(whole, tokens, *d, temperature=0.9)
    cut = slice(rank * V, (rank + 1) * V)
    check_gradient(grad, full[:, cut], size[:, cut], V * world, want["log_p"][:, cut])


@pytest.mark.parametrize("world", [2, 3])
def test_vocabulary_split_over_ranks(world):
    run_distributed(_split, world)
