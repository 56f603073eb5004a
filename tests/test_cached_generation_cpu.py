"""Generation with a block cache on CPU ranks: the same tokens as re-evaluating every prefix where the cache holds 32-bit values, beam
search against a plain one, the same results on every grid, and what is refused."""

import math

import pytest
import torch

from _dist import run_cached, run_distributed


def _model(family, grid, world):
    from axonn_b200 import axonn as ax
    from axonn_b200.models import GPT, GPTConfig, Llama, LlamaConfig, Mixtral, MixtralConfig

    r, c, d = grid
    ax.init(G_inter=1, G_data=world // (r * c * d), G_intra_r=r, G_intra_c=c, G_intra_d=d)
    torch.manual_seed(4)
    if family == "gpt":
        model = GPT(GPTConfig(n_layers=2, hidden=64, n_heads=4, ffn=128, vocab=96, seq_len=40), dtype=torch.float32)
    elif family == "llama":
        model = Llama(LlamaConfig(n_layers=2, hidden=64, n_heads=4, n_kv_heads=2, ffn=128, vocab=96, seq_len=40), dtype=torch.float32)
    else:
        model = Mixtral(MixtralConfig(n_layers=2, hidden=64, n_heads=4, n_kv_heads=2, ffn=128, n_experts=4, vocab=96, seq_len=40,
                                      capacity_factor=4.0), dtype=torch.float32)
    with torch.no_grad():                               # logits that tell tokens apart
        model.head.proj.weight.mul_(30)
        if family == "gpt":
            model.pos_emb.weight.mul_(10)
    return model


def _lossless():
    """The cache in 32 bits: the same blocks, tables and slots, nothing rounded."""
    from axonn_b200 import ops
    from axonn_b200.models import cache, generate
    from axonn_b200.ops import kv_cache

    class Lossless(cache.BlockCache):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            k, v, ks, vs = self.blocks
            self.blocks = ops.BlockLayer(torch.full(k.shape, math.nan), torch.full(v.shape, math.nan), ks, vs)
            self._layers = [cache._LayerCache(self, i) for i in range(len(self._layers))]

    def store(qkv, layer, slots, positions=None, table=None):
        R, S, G, n, D = qkv.shape
        BT = layer.k.shape[2]
        q = qkv
        if table is not None:
            x = kv_cache._rotate_torch(qkv[:, :, :, :-1].reshape(R * S, -1, D), table, positions.reshape(-1).clamp(min=0)).view(R, S, G, n - 1, D)
            q = torch.cat([x, qkv[:, :, :, -1:]], 3)
        for r in range(R):
            for i in range(S):
                if slots[r, i] >= 0:
                    b, t = divmod(int(slots[r, i]), BT)
                    layer.k[b, :, t], layer.v[b, :, t] = q[r, i, :, -2], q[r, i, :, -1]
        return q[:, :, :, :-2]

    def attend(q, layer, tables, lengths, new=None, scale=None):
        return kv_cache._attend_torch(q, layer, tables, lengths, new, q.shape[-1] ** -0.5)
    ops.store_blocks, ops.cached_attention = store, attend
    ops.reorder_blocks = lambda blocks, *a: kv_cache._reorder_torch(blocks, *a)
    generate.BlockCache = Lossless


PROMPTS = [[5, 17, 9, 3, 60, 2, 2, 31, 7, 7, 1, 90, 44, 18, 6, 3, 3, 8], [64, 2, 2, 20, 11, 95, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0]]
LENGTHS = [18, 6]


def _greedy(rank, world, family, grid):
    from axonn_b200.models import greedy_generate

    model = _model(family, grid, world)
    prompts = torch.tensor(PROMPTS)
    want = greedy_generate(model, prompts, 12)
    ragged = [greedy_generate(model, prompts[r:r + 1, :n], 12)[0] for r, n in enumerate(LENGTHS)]
    eos = int(want[0, 22])
    stopped = greedy_generate(model, prompts, 12, eos_id=eos)
    rounded = {dtype: greedy_generate(model, prompts, 12, cache_dtype=dtype) for dtype in (torch.float8_e4m3fn, torch.int8)}
    for out in rounded.values():                        # the first token comes from the prompt as it is
        assert out.shape == want.shape and torch.equal(out[:, :19], want[:, :19]) and model.training
    _lossless()
    for block in (16, 32):
        assert torch.equal(greedy_generate(model, prompts, 12, cache_dtype=torch.int8, block_tokens=block), want)
        assert torch.equal(greedy_generate(model, prompts, 12, eos_id=eos, cache_dtype=torch.int8, block_tokens=block), stopped)
        out = greedy_generate(model, prompts, 12, cache_dtype=torch.int8, prompt_lengths=LENGTHS, block_tokens=block)
        for r, n in enumerate(LENGTHS):
            assert torch.equal(out[r, :n + 12], ragged[r]) and not bool(out[r, n + 12:].any())
    assert torch.equal(greedy_generate(model, prompts, 100, cache_dtype=torch.int8), greedy_generate(model, prompts, 100))      # to the model's length
    assert torch.equal(greedy_generate(model, prompts, 0, cache_dtype=torch.int8), prompts)
    return want.tolist()


@pytest.mark.parametrize("family", ["gpt", "llama", "mixtral"])
def test_greedy_decoding_with_a_cache(family):
    run_cached(_greedy, 1, family, (1, 1, 1))


def test_greedy_decoding_with_a_cache_on_a_grid():
    ref = run_cached(_greedy, 1, "llama", (1, 1, 1))[0]
    for got in run_distributed(_greedy, 2, "llama", (2, 1, 1)):
        assert got == ref


def _plain_beams(model, prompt, steps, K, eos):
    """Beam search over whole prefixes, in 64 bits: [(score, tokens, done)], best first."""
    rows = [(0.0, list(prompt), False)]
    for _ in range(steps):
        found = []
        for j, (score, seq, done) in enumerate(rows):
            if done:
                found.append((score, j, eos, True))
                continue
            logp = model(torch.tensor([seq])).detach()[0, -1].double().log_softmax(-1)
            found += [(score + float(logp[t]), j, t, t == eos) for t in logp.topk(K + 1)[1].tolist()]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        rows = [(s, rows[j][1] + [t], d) for s, j, t, d in found[:K]]
        if all(d for _, _, d in rows):
            break
    return rows


def _beams(rank, world, family, grid, K):
    from axonn_b200.models import beam_generate, greedy_generate

    model = _model(family, grid, world)
    prompts = torch.tensor(PROMPTS)
    single = grid == (1, 1, 1)
    eos = int(greedy_generate(model, prompts, 4)[1, 20])
    rounded = beam_generate(model, prompts, 6, K, eos_id=eos, prompt_lengths=LENGTHS)
    assert rounded[0].shape[:2] == (2, K) and bool((rounded[1][:, :-1] >= rounded[1][:, 1:]).all()) and model.training
    _lossless()
    results = []
    for end in (None, eos):
        for block in (16, 32):
            seqs, scores = beam_generate(model, prompts, 6, K, eos_id=end, prompt_lengths=LENGTHS, block_tokens=block)
            results.append((seqs.tolist(), [[round(s, 3) for s in row] for row in scores.tolist()]))
            if not single:
                continue
            model.eval()
            for r, n in enumerate(LENGTHS):
                want = _plain_beams(model, PROMPTS[r][:n], 6, K, end)
                for (score, seq, _), got, value in zip(want, seqs[r].tolist(), scores[r].tolist()):
                    # a sum of six logarithms of 32-bit logits (up to 30): 6 x 30 x 2^-20
                    assert got[:len(seq)] == seq and abs(value - score) < 2e-4
                    assert all(t == (end or 0) for t in got[len(seq):])
            model.train()
    if single:
        # longer sequences count more with a penalty: sums over the numbers of new tokens
        plain, scores = beam_generate(model, prompts, 6, K, eos_id=eos, prompt_lengths=LENGTHS)
        by_length, normed = beam_generate(model, prompts, 6, K, eos_id=eos, prompt_lengths=LENGTHS, length_penalty=1.0)
        for r, n in enumerate(LENGTHS):
            def size(seq):
                new = seq[n:n + 6]
                return new.index(eos) + 1 if eos in new else len(new)
            want = sorted((s / size(seq) for s, seq in zip(scores[r].tolist(), plain[r].tolist())), reverse=True)
            assert normed[r].tolist() == pytest.approx(want, rel=1e-5)
        one = beam_generate(model, prompts, 12, 1)[0][:, 0]
        assert torch.equal(one, greedy_generate(model, prompts, 12))
        seqs, scores = beam_generate(model, prompts, 100, 2)
        assert seqs.shape == (2, 2, 40)
        assert beam_generate(model, prompts, 0, 2)[0].shape == (2, 2, 18)
    return results


@pytest.mark.parametrize("family,K", [("gpt", 4), ("llama", 3)])
def test_beam_search(family, K):
    run_cached(_beams, 1, family, (1, 1, 1), K)


def test_beam_search_is_the_same_on_a_grid():
    """Vocabulary and KV heads split over the row group, hidden over the column group."""
    ref = run_cached(_beams, 1, "gpt", (1, 1, 1), 4)[0]
    for got in run_distributed(_beams, 4, "gpt", (2, 2, 1), 4):
        for (seqs, scores), (want, want_scores) in zip(got, ref):
            assert seqs == want
            for a, b in zip(scores, want_scores):
                assert a == pytest.approx(b, abs=2e-3)


def _refusals(rank, world):
    from axonn_b200.models import BlockCache, beam_generate, greedy_generate

    model = _model("llama", (1, 1, 1), 1)
    prompts = torch.tensor(PROMPTS)
    for words, call in (("need a cache", lambda: greedy_generate(model, prompts, 2, prompt_lengths=LENGTHS)),
                        ("prompt_lengths", lambda: greedy_generate(model, prompts, 2, cache_dtype=torch.int8, prompt_lengths=[18])),
                        ("prompt_lengths", lambda: greedy_generate(model, prompts, 2, cache_dtype=torch.int8, prompt_lengths=[18, 0])),
                        ("prompt_lengths", lambda: beam_generate(model, prompts, 2, 2, prompt_lengths=[19, 1])),
                        ("starts from a prompt", lambda: beam_generate(model, prompts[:, :0], 2, 2)),
                        ("of which the model takes", lambda: beam_generate(model, prompts.repeat(1, 3), 2, 2)),
                        ("beams", lambda: beam_generate(model, prompts, 2, 33)),
                        ("beams", lambda: beam_generate(model, prompts, 2, 0)),
                        ("blocks hold", lambda: greedy_generate(model, prompts, 2, cache_dtype=torch.int8, block_tokens=24)),
                        ("expand", lambda: BlockCache(model, 2, 20).reorder(torch.zeros(1, 2, dtype=torch.int32)))):
        with pytest.raises(ValueError, match=words):
            call()
        assert model.training
    with pytest.raises(TypeError, match="codes"):
        greedy_generate(model, prompts, 2, cache_dtype=torch.uint8)


def test_refusals():
    run_distributed(_refusals, 1)


def _shared_blocks(rank, world):
    """A cache through its public calls: full blocks of a prompt are shared by its beams, every row writes into blocks of its own."""
    from axonn_b200.models import BlockCache

    model = _model("llama", (1, 1, 1), 1).eval()
    cache = BlockCache(model, 2, 40, 16, torch.int8, beams=3, prompt_tokens=18)
    with torch.no_grad():
        cache.plan(18, torch.tensor(LENGTHS, dtype=torch.int32))
        model(torch.tensor(PROMPTS), cache=cache)
        cache.expand(3)
        assert cache.lengths.tolist() == [18] * 3 + [6] * 3
        for step in range(20):
            t = cache.tables
            held = [-(-n // 16) for n in cache.lengths.tolist()]
            writing = [int(t[r, n // 16]) for r, n in enumerate(cache.lengths.tolist()) if n % 16]
            own = writing + cache.spare.tolist()
            assert len(set(own)) == len(own) and min(own) >= 0
            for r, n in enumerate(held):
                assert bool((t[r, :n] >= 0).all())
            if step == 0:
                assert t[0, 0] == t[1, 0] == t[2, 0]
            cache.plan(1)
            model(torch.randint(0, 96, (6, 1)), cache=cache)
            cache.reorder(torch.randint(0, 3, (2, 3)).int())
    assert cache.lengths.tolist() == [38] * 3 + [26] * 3 and int(cache.taken) <= cache.free.numel()


def test_beams_share_what_is_full():
    run_distributed(_shared_blocks, 1)


def _ends_of_a_cache(rank, world):
    """Tokens past the cache's end get no place; beams that no blocks were set aside for are refused, prompts longer than was said end."""
    from axonn_b200.models import BlockCache

    model = _model("gpt", (1, 1, 1), 1).eval()
    with torch.no_grad():
        cache = BlockCache(model, 2, 20, 16, torch.int8)
        cache.plan(18, torch.tensor(LENGTHS, dtype=torch.int32))
        model(torch.tensor(PROMPTS), cache=cache)
        cache.plan(5)                                   # the last block has places for 32
        assert cache.lengths.tolist() == [20, 11] and cache.new.tolist() == [2, 5]
        assert cache.step.slots[0, 2:].tolist() == [-1] * 3 and int(cache.positions.max()) == 19
        assert bool(model(torch.tensor(PROMPTS)[:, :5], cache=cache).isfinite().all())
        cache.plan(1)
        assert cache.lengths.tolist() == [20, 12] and cache.new.tolist() == [0, 1]
        assert bool(model(torch.zeros(2, 1, dtype=torch.long), cache=cache).isfinite().all())
        with pytest.raises(ValueError, match="targets"):
            model(torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1, dtype=torch.long), cache)
        with pytest.raises(ValueError, match="go on once"):
            cache.expand(2)
        with pytest.raises(ValueError, match="40 positions"):
            BlockCache(model, 1, 41)
        beams = BlockCache(model, 1, 40, 16, torch.int8, beams=2, prompt_tokens=2)
        with pytest.raises(ValueError, match="go on once"):
            beams.expand(3)
        for n in (18, 18):
            beams.plan(n)
            model(torch.tensor(PROMPTS)[:1], cache=beams)
        beams.expand(2)
        with pytest.raises(ValueError, match="go on once"):
            beams.expand(2)
        for _ in range(10):
            beams.plan(1)
            assert bool(model(torch.zeros(2, 1, dtype=torch.long), cache=beams).isfinite().all())
            beams.reorder(torch.tensor([[1, 0]], dtype=torch.int32))
        assert int(beams.taken) <= beams.free.numel() and int(beams.tables.max()) < beams.free.numel()


def test_ends_of_a_cache():
    run_distributed(_ends_of_a_cache, 1)
