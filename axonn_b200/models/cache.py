"""Key/value cache of a model in blocks of 8-bit codes, for generation (``models/generate.py``).

The state that the operators of ``ops/kv_cache.py`` work on: codes and scales of all layers, the rows' block tables and
lengths, and the list that blocks are taken from.  Every rank of a tensor-parallel group holds the KV heads of its own
attention layers; tables and lengths are the same everywhere.
"""

import torch

from .. import ops


class _LayerCache:
    """One attention layer's part of a cache, in the step that ``BlockCache.plan`` has prepared."""

    def __init__(self, cache, index):
        self._cache = cache
        self._layer = ops.BlockLayer(*(t[index] for t in cache.blocks))

    @property
    def starting(self):
        return self._cache.starting

    @property
    def max_tokens(self):
        return self._cache.max_tokens

    def store(self, qkv, rope_table=None):
        step = self._cache.step
        return ops.store_blocks(qkv, self._layer, step.slots, step.positions, rope_table)

    def attend(self, q):
        c = self._cache
        return ops.cached_attention(q, self._layer, c.tables, c.lengths, c.new)


class BlockCache:
    """Cache for ``rows`` sequences of up to ``max_tokens`` tokens of ``model`` (``GPT``, ``Llama``, ``Mixtral``).

    ``plan(tokens, new)`` places the next tokens of every row, ``model(tokens, cache=cache)`` evaluates them and returns the logits
    of each row's last one; tokens past ``max_tokens`` get no place, and ``lengths`` tells how many have one.  ``expand(beams)`` lets
    every row go on as ``beams`` rows, which ``reorder(parents)`` lets go on from one another; ``prompt_tokens`` (``None``: up to
    ``max_tokens``) are stored before that, whose full blocks are shared, and ``beams`` here sets blocks aside for it.  ``dtype``: ``torch.float8_e4m3fn`` or ``torch.int8``."""

    def __init__(self, model, rows, max_tokens, block_tokens=64, dtype=torch.float8_e4m3fn, beams=None, prompt_tokens=None):
        attn = [blk.attn for blk in model.blocks]
        device = next(model.parameters()).device
        per = lambda n: -(-n // block_tokens)  # noqa: E731
        if hasattr(model, "pos_emb") and max_tokens > model.cfg.seq_len:
            raise ValueError(f"{max_tokens} tokens for a model that has learned {model.cfg.seq_len} positions")
        self.block_tokens, self.max_tokens, self.beams = block_tokens, max_tokens, beams
        width = per(max_tokens)
        blocks = rows * width
        if beams is not None:
            # the prompts' blocks, and for every beam two to start with and those that it fills
            prompt = max_tokens if prompt_tokens is None else prompt_tokens
            blocks = rows * per(prompt) + rows * beams * (per(max_tokens - prompt) + 3)
        shape = (len(attn), blocks, attn[0].groups_l)
        self.blocks = ops.BlockLayer(*(torch.zeros(*shape, block_tokens, attn[0].head_dim, dtype=torch.uint8, device=device).view(dtype)
                                       for _ in range(2)), *(torch.ones(shape, device=device) for _ in range(2)))
        self.tables = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        self.taken = torch.zeros(1, dtype=torch.int32, device=device)
        self.free = torch.arange(blocks, dtype=torch.int32, device=device)
        self.spare = None
        self.starting = True           # the step at hand is the rows' first
        self.step = self.new = None
        self._layers = [_LayerCache(self, i) for i in range(len(attn))]

    def layer(self, i):
        return self._layers[i]

    def plan(self, tokens, new=None):
        """Place the next ``tokens`` tokens of every row, the first ``new[r]`` (int32; ``None``: all) of which are there."""
        if new is None:
            new = torch.full_like(self.lengths, tokens)
        if self.max_tokens % self.block_tokens:                         # the last block has more places
            new = torch.minimum(new, (self.max_tokens - self.lengths).clamp(min=0))
        before = self.lengths
        self.starting = self.step is None
        self.step = ops.plan_blocks(self.lengths, new, self.tables, self.free, self.taken, tokens, self.block_tokens)
        self.lengths, self.taken = self.step.lengths, self.step.taken
        self.new = self.lengths - before

    @property
    def positions(self):
        """Positions of the step's tokens (0 where there is none)."""
        return self.step.positions.clamp(min=0).long()

    def last(self, y):
        """Of ``y [rows, tokens, hidden]`` every row's last new token."""
        if y.shape[1] == 1:
            return y
        at = (self.new.long() - 1).clamp(min=0)
        return y.gather(1, at[:, None, None].expand(-1, 1, y.shape[2]))

    def expand(self, beams):
        """Every row goes on as ``beams`` rows: full blocks are shared, the unfinished one is copied for each."""
        if self.beams is None or not 1 <= beams <= self.beams or self.spare is not None:
            raise ValueError(f"rows go on once, as up to {self.beams or 'beams='} rows that the cache was made for, not {beams}")
        rows = self.tables.shape[0]
        n = rows * beams
        at = self.taken.long() + torch.arange(2 * n, device=self.free.device)
        last = self.free.numel() - 1
        own, spare = torch.where(at <= last, self.free[at.clamp(max=last)], -1).view(2, n)      # a prompt longer than was said: none is left
        self.taken = (self.taken + 2 * n).clamp(max=last + 1)
        tables, lengths = self.tables.repeat_interleave(beams, 0), self.lengths.repeat_interleave(beams, 0)
        # the first of a row's beams keeps the row's blocks; each other one gets a block of its own, filled as that of a row that moves
        current = lengths[:, None] // self.block_tokens == torch.arange(tables.shape[1], device=tables.device)
        other = (torch.arange(n, device=tables.device) % beams != 0)[:, None]
        self.tables, self.lengths, self.spare = torch.where(current & other, own[:, None], tables), lengths, spare.contiguous()
        self.reorder(torch.zeros(rows, beams, dtype=torch.int32, device=tables.device))

    def reorder(self, parents):
        """Row ``j`` of the beams of ``b`` goes on from row ``parents[b, j]`` (int32) of them."""
        if self.spare is None:
            raise ValueError("rows go on from one another after expand()")
        self.tables, self.lengths, self.spare = ops.reorder_blocks(self.blocks, self.tables, self.lengths, self.spare, parents)
