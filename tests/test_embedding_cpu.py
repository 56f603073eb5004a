"""``embedding`` on the CPU: results, gradients and refusals, and what its launchers refuse."""

import shutil

import pytest
import torch

from axonn_b200 import ops
from axonn_b200.ops import _lib


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_lookup(dtype, index):
    w = torch.randn(6, 5).to(dtype).requires_grad_()
    tokens = torch.tensor([[1, 4, 1], [2, 0, 4]], dtype=index)
    out = ops.embedding(tokens, w)
    assert torch.equal(out, w[tokens.long()])
    scaled = ops.embedding(tokens, w, scale=2.5, padding_idx=-2)
    assert torch.equal(scaled, (w[tokens.long()].float() * 2.5).to(dtype))
    (g,) = torch.autograd.grad(scaled.sum(), w)
    assert torch.equal(g[:, 0].float(), torch.tensor([2.5, 5, 2.5, 0, 0, 0]))
    assert ops.embedding(tokens[:0], w).shape == (0, 3, 5) and ops.embedding(tokens[0, 0], w).shape == (5,)


def test_refusals():
    w, t = torch.randn(4, 8), torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: ops.embedding(t.float(), w), lambda: ops.embedding(t, w.double()), lambda: ops.embedding(t, w[0]),
                lambda: ops.embedding(t, w, float("inf")), lambda: ops.embedding(t, w, padding_idx=4), lambda: ops.embedding(t, w, padding_idx=-5)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        ops.embedding(t + 4, w)


@pytest.mark.skipif(not (_lib.available() or shutil.which("nvcc")), reason="native library not built")
def test_launchers_refuse():
    """Addresses that are never used: the calls are refused on the host."""
    L, p = _lib.lib(), 4096
    for call in (lambda: L.axb_embedding(p, 4, 1, p, 8, 0, 8, 1.0, p, -1, None, 0, None), lambda: L.axb_embedding(p, 2, 1, p, 8, 4, 8, 1.0, p, -1, None, 0, None),
                 lambda: L.axb_embedding(p, 8, 1 << 31, p, 8, 4, 8, 1.0, p, -1, p, 0, None), lambda: L.axb_embedding(p, 8, 1, p, 8, 4, 8, 1.0, p, -1, p, 3, None),
                 lambda: L.axb_embedding(p, 8, 1, p, 8, 4, 8, 1.0, p, -1, p + 4, 0, None), lambda: L.axb_embedding_grad(p, 8, p, -1, p, 8, 4, 8, 1.0, -1, p, p, 0, None),
                 lambda: L.axb_embedding_grad(p, 8, p, 1, p, 8, (1 << 30) + 1, 8, 1.0, -1, p, p, 0, None),
                 lambda: L.axb_embedding_grad(p, 8, p, 1, p, 8, 4, 8, 1.0, -1, p, p + 8, 0, None), lambda: L.axb_embedding_grad(p, 4, p + 8, 1, p, 8, 4, 8, 1.0, -1, p, p, 0, None),
                 lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, p, p, p, 1, 0, 8, 0, 8, 0, 1.0, -100, 1, 0, None),
                 lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, p, p, p, 1, 1, 8, 0, 8, 9, 1.0, -100, 1, 0, None),
                 lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, p, p, p, 1, 1, 80, 0, 80, 33, 1.0, -100, 1, 0, None),
                 lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, p, p, p, 1, 1, 8, 0, 8, 0, 0.0, -100, 1, 0, None),
                 lambda: L.axb_embedding_grad(p, 8, None, 300, p, 8, 4, 8, 1.0, -1, p, p, 0, None),
                 lambda: L.axb_embedding_grad(p, 8, p, 300, p, 8, 4, 8, 1.0, -1, p, None, 0, None),
                 lambda: L.axb_embedding_grad(p, 2, p, 30, p, 8, 4, 8, 1.0, -1, p, p, 0, None),
                 lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, p, p, p + 8, 1, 1, 8, 0, 8, 0, 1.0, -100, 1, 0, None),
                 lambda: L.axb_token_log_probs(p, 8, 8, p, 1, 1, p, p, None, p, p, 1, 1, 8, 0, 8, 2, 1.0, -100, 1, 0, None),
                 lambda: L.axb_token_log_probs_bwd(p, 8, 8, p, 1, 1, p, p, p, p, None, p, 1, 1, 8, 0, 8, 2, 1.0, -100, 0, None),
                 lambda: L.axb_token_log_probs_bwd(p, 8, 8, p, 1, 1, p, p, p, p, p, p, 1, 1, 8, 0, 8, 0, 1.0, -100, 3, None)):
        assert call() == -1 and _lib.lib().axb_last_error()
