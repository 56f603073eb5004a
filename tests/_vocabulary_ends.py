"""Cases at the ends of what the vocabulary's operators take, for both devices."""

import torch

from axonn_b200 import ops

from _vocabulary import check_gradient, check_told, told, told_gradient

COLD, HOT = 2.0 ** -100, 2.0 ** 100


def ends_of_temperature(dtype, device):
    """Logits with a mask, and with the largest and the lowest numbers of the type."""
    g = torch.Generator().manual_seed(3)
    logits = (3 * torch.randn(4, 41, generator=g)).to(dtype)
    logits[1, ::2] = -float("inf")
    logits[2] = torch.finfo(dtype).min
    logits[2, 5] = torch.finfo(dtype).max
    tokens = torch.tensor([int(logits[0].float().argmax()), 3, 5, -100])
    return logits.to(device), tokens.to(device)


def check_ends_of_temperature(logits, tokens, temperature):
    """Results and gradients against 64 bits; what the gradient's type does not hold (2^100 in fp16, of which the largest is 65504) is
    infinite."""
    z = logits.requires_grad_()
    got = ops.token_log_probs(z, tokens, entropy=True, top=4, temperature=temperature)
    want = told(z, tokens, 4, temperature)
    check_told(got, want, 41, 4)
    d = [torch.ones_like(t) for t in got[:3]]
    (grad,) = torch.autograd.grad(got[:3], z, d)
    want_d, size = told_gradient(z, tokens, *d, temperature=temperature)
    held = want_d.to(z.dtype).double()
    assert torch.equal(grad.cpu().isinf(), held.isinf()) and torch.equal(grad.cpu().double()[held.isinf()], held[held.isinf()])
    check_gradient(grad.masked_fill(grad.isinf(), 0), want_d.masked_fill(held.isinf(), 0), size, 41, want["log_p"])
