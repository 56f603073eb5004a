"""Generation with a block cache on the GPU: the kernels' logits beside those of the same cache attended to in plain PyTorch, and beams
whose scores are those of their sequences evaluated on their own."""

import pytest
import torch
import torch.distributed as dist

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _grid():
    from axonn_b200 import axonn as ax

    if not dist.is_initialized():
        dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1)
    if not ax.is_initialized:
        ax.init(G_inter=1, G_data=1, G_intra_r=1, G_intra_c=1, G_intra_d=1)


def _model(family, head_dim):
    from axonn_b200.models import GPT, GPTConfig, Llama, LlamaConfig, Mixtral, MixtralConfig

    torch.manual_seed(0)
    h = 4 * head_dim
    shape = dict(n_layers=2, hidden=h, n_heads=4, ffn=2 * h, vocab=1000, seq_len=256)
    if family == "gpt":
        model = GPT(GPTConfig(**shape), dtype=torch.bfloat16)
    elif family == "llama":
        model = Llama(LlamaConfig(n_kv_heads=2, **shape), dtype=torch.bfloat16)
    else:
        model = Mixtral(MixtralConfig(n_kv_heads=1, n_experts=8, capacity_factor=4.0, **shape), dtype=torch.bfloat16)
    with torch.no_grad():
        model.head.proj.weight.mul_(10)
    return model.to(DEV).eval()


@torch.no_grad()
def _feed(model, cache, tokens, new, steps):
    """Logits of the prompt's last tokens and of the steps' tokens."""
    cache.plan(tokens.shape[1], new)
    out = [model(tokens, cache=cache)]
    for s in steps:
        cache.plan(s.shape[1])
        out.append(model(s, cache=cache))
    return torch.cat(out, 1).float()


@pytest.mark.parametrize("family,head_dim", [("gpt", 64), ("llama", 128), ("llama", 64), ("mixtral", 64)])
@pytest.mark.parametrize("dtype,block", [(torch.float8_e4m3fn, 64), (torch.int8, 16)])
def test_logits_of_cached_steps(family, head_dim, dtype, block, monkeypatch):
    """Two layers, in each of which the attention's outputs differ by a rounding to bf16 on either side (2^-8), and some six operations
    behind it that round what has changed (2^-8 each): at most 2 x 8 x 2^-8 of the logits' norm.  Steps of one token and of several."""
    from axonn_b200 import ops
    from axonn_b200.models import BlockCache
    from axonn_b200.ops import kv_cache

    model = _model(family, head_dim)
    torch.manual_seed(1)
    prompt, new = torch.randint(0, 1000, (3, 70), device=DEV), torch.tensor([70, 1, 37], dtype=torch.int32, device=DEV)
    steps = [torch.randint(0, 1000, (3, n), device=DEV) for n in (1, 1, 5, 1, 20, 1)]
    got = _feed(model, BlockCache(model, 3, 128, block, dtype), prompt, new, steps)

    def attend(q, layer, tables, lengths, new=None, scale=None):
        R, S, G, P, D = q.shape if q.ndim == 5 else (*q.shape[:2], layer.k.shape[1], q.shape[2] // layer.k.shape[1], q.shape[3])
        return kv_cache._attend_torch(q.reshape(R, S, G, P, D), layer, tables, lengths, new, D ** -0.5)
    monkeypatch.setattr(ops, "cached_attention", attend)
    want = _feed(model, BlockCache(model, 3, 128, block, dtype), prompt, new, steps)
    assert bool(got.isfinite().all()) and float((got - want).norm()) <= 2.0 ** -4 * float(want.norm())


@pytest.mark.parametrize("family,head_dim,eos", [("gpt", 64, None), ("llama", 128, 17), ("mixtral", 64, 5)])
def test_scores_of_beams_are_those_of_their_sequences(family, head_dim, eos):
    """Every beam's sequence evaluated on its own through a cache that no row goes on from another in: the same blocks' contents, so that
    logits differ by the roundings of products over other numbers of rows alone: sixteen values of size up to 16 in bf16, at most
    16 x 16 x 2^-8 = 1, and their logarithms' sums add what is met of it at random (a quarter)."""
    from axonn_b200.models import BlockCache, beam_generate

    model = _model(family, head_dim)
    torch.manual_seed(2)
    lengths, new, K = [40, 23], 16, 4
    prompts = torch.randint(0, 1000, (2, 40), device=DEV)
    seqs, scores = beam_generate(model, prompts, new, K, eos_id=eos, prompt_lengths=lengths, block_tokens=16)
    again, same = beam_generate(model, prompts, new, K, eos_id=eos, prompt_lengths=lengths, block_tokens=16)
    assert torch.equal(seqs, again) and torch.equal(scores, same)
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    for b, n in enumerate(lengths):
        assert len({tuple(s) for s in seqs[b].tolist()}) == K
        tail = seqs[b, :, n:n + new]
        logits = _feed(model, BlockCache(model, K, 64, 16), prompts[b, :n].expand(K, n).contiguous(),
                       torch.full((K,), n, dtype=torch.int32, device=DEV), [tail[:, i:i + 1].contiguous() for i in range(new - 1)])
        logp = logits.double().log_softmax(-1).gather(2, tail[..., None])[..., 0]
        for j in range(K):
            m = new
            if eos is not None and eos in tail[j].tolist():
                m = tail[j].tolist().index(eos) + 1
                assert all(t == eos for t in tail[j, m:].tolist())
            assert abs(float(logp[j, :m].sum()) - float(scores[b, j])) < 0.25


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_greedy_decoding_with_a_cache(dtype):
    """The first token is that of the prompt as it is; with an end token rows stop and are padded; heads that no kernel takes are refused."""
    from axonn_b200.models import greedy_generate

    model = _model("llama", 128)
    prompts = torch.randint(0, 1000, (2, 30), device=DEV)
    want = greedy_generate(model, prompts, 8)
    got = greedy_generate(model, prompts, 8, cache_dtype=dtype)
    assert got.shape == want.shape and torch.equal(got[:, :31], want[:, :31])
    eos = int(got[0, 33])
    stopped = greedy_generate(model, prompts, 8, eos_id=eos, cache_dtype=dtype)
    first = got[0, 30:].tolist().index(eos)
    assert torch.equal(stopped[0, :31 + first], got[0, :31 + first]) and bool((stopped[0, 31 + first:] == eos).all())
    with pytest.raises(ValueError, match="64 or 128"):
        greedy_generate(_model("gpt", 32), prompts, 2, cache_dtype=dtype)
