"""Prefill + greedy decode of a fixed batch, with a HIP-graph-capturable decode step.

The counterpart of the reference runtime's prefill-then-decode loop
(`src/torch_llm/inference/runtime.py:174-330`) for one fixed batch, reduced to
what drives the FP8 paged KV-cache path:

* `prefill(prompts)` reserves every sequence's whole lifetime in the
  `PageAllocator` (reference full-lifetime reservation), runs the packed prompts
  through the model (prompt attention, then the bulk quantized cache write) and
  samples the first token (argmax at temperature 0, reference `sampling.py`);
* `step()` is one decode step over the batch with no host synchronization: the
  write locations `block_table[slot, pos // BS]`, `pos % BS` (reference
  `page_allocator.py:225-245`), the context lengths (committed + 1, reference
  `:347`) and the next positions are all computed on the device from buffers
  that live as long as the decoder, so the step can be captured once in a HIP
  graph and replayed (`capture()`, `generate()`).

Unlike the reference runtime, the allocator's committed lengths are not advanced
by every step (that would be host work inside the captured step): `generate()`
commits the tokens it wrote when it returns, and a caller driving `step()` itself
commits with `commit(steps)`.

A prefix that all sequences share (a system prompt, or one prompt to be answered many times) is kept
once: with `prefix_len`, `prefill(prompts, prefix)` runs it through the model as a request of its own
and the prompts and every later step behind it (`kernals/shared_prefix_attention.py`). With
`logprobs`, every step records the log probability of the token it chose, the entropy and that many
alternatives (`kernals/token_logprobs.py`) in `scores`, rows in decode order like `history`.

Drafted continuations, from whatever proposes them, are checked in one pass with `verify(drafts)`
(`kernals/draft_tree.py`): every sequence gains the tokens of the path that the model would have chosen
step by step, and its choice behind them.
"""

from __future__ import annotations

import torch as t

from aiproj_amd.inference.page_allocator import CacheContainer, PageAllocator
from aiproj_amd.inference.paged_kv_cache import PagedKVCache
from aiproj_amd.kernals.draft_tree import DraftTree, accept_draft
from aiproj_amd.kernals.shared_prefix_attention import SharedPrefix
from aiproj_amd.kernals.token_logprobs import MAX_TOP, TokenLogprobs, token_logprobs
from aiproj_amd.model.transformer import StepMeta, TransformerLM


class GreedyDecoder:
    def __init__(self, model: TransformerLM, batch: int, max_len: int, cache_dtype=t.float8_e4m3fn,
                 block_size: int = 16, device="cuda", prefix_len: int = 0, logprobs: int | None = None):
        cfg = model.cfg
        if prefix_len < 0 or (prefix_len and prefix_len + max_len > cfg.max_seq_len):
            raise ValueError("GreedyDecoder: prefix_len and max_len together are at most the model's max_seq_len")
        if logprobs is not None and not 0 <= logprobs <= min(MAX_TOP, cfg.vocab_size):
            raise ValueError(f"GreedyDecoder: logprobs is a number of alternatives up to {MAX_TOP}")
        self.model = model
        self.batch = batch
        self.block_size = block_size
        self.max_len = max_len
        pages = batch * (-(-max_len // block_size)) + -(-prefix_len // block_size)
        self.allocator = PageAllocator(pages, block_size, batch + (prefix_len > 0), max(max_len, prefix_len), device)
        self.prefix_len = prefix_len          # tokens reserved for the prefix; after prefill, those it has
        self.prefix = None
        self.logprobs = logprobs
        self.scores = None
        self.caches = [PagedKVCache(pages, block_size, cfg.num_kv_heads, cfg.head_dim, device, cache_dtype)
                       for _ in range(cfg.num_layers)]
        self.device = t.device(device)
        self.slots = None
        # Decode-step state, updated in place by every step (graph-stable addresses).
        self.tokens = t.zeros(batch, dtype=t.int64, device=device)
        self.positions = t.zeros(batch, dtype=t.int64, device=device)
        self.context_lengths = t.zeros(batch, dtype=t.int32, device=device)
        self.history = None
        self.steps_left = 0
        self.step_index = t.zeros(1, dtype=t.int64, device=device)
        self.graph = None

    def _prefill_prefix(self, prefix: t.Tensor | None):
        """The shared prefix [P] int64 into the cache, as request `batch`."""
        if prefix is not None and prefix.ndim != 1:
            raise ValueError("GreedyDecoder: a prefix is a vector of tokens")
        given = 0 if prefix is None else prefix.shape[0]
        if given > self.prefix_len:
            raise ValueError(f"GreedyDecoder: a prefix of {given} tokens, {self.prefix_len} are reserved")
        self.prefix_len = given
        if given == 0:
            return
        slot = self.allocator.allocate_request(self.batch, given)
        positions = t.arange(given, device=self.device)
        cu = t.tensor([0, given], dtype=t.int32, device=self.device)
        ctx = self.allocator.create_container(t.tensor([slot], dtype=t.int64, device=self.device), cu, positions, validate=False)
        self.model(prefix.to(self.device), StepMeta("prefill", positions, ctx, cu_seqlens=cu, max_seqlen=given), self.caches)
        self.allocator.advance(self.batch, given)
        self.prefix = SharedPrefix.one(slot, given, self.batch, self.device)

    def prefill(self, prompts: t.Tensor, prefix: t.Tensor | None = None) -> t.Tensor:
        """prompts [B, P] int64, behind `prefix` [N] int64 if given -> first sampled tokens [B] (also the next
        step's input)."""
        batch, length = prompts.shape
        assert batch == self.batch and length < self.max_len
        self._prefill_prefix(prefix)
        slots = [self.allocator.allocate_request(i, self.max_len) for i in range(batch)]
        self.slots = t.tensor(slots, dtype=t.int64, device=self.device)
        positions = t.arange(length, device=self.device).repeat(batch)
        cu = t.arange(batch + 1, device=self.device, dtype=t.int32) * length
        ctx = self.allocator.create_container(self.slots, cu, positions, validate=False)
        meta = StepMeta("prefill", positions + self.prefix_len, ctx, cu_seqlens=cu, max_seqlen=length, prefix=self.prefix)
        logits = self.model(prompts.reshape(-1).to(self.device), meta, self.caches)
        self.allocator.advance_batch(list(range(batch)), [length] * batch)
        self.tokens.copy_(logits.argmax(-1))
        self.positions.fill_(length)
        self.context_lengths.fill_(length + 1)
        # Every later token of every sequence, in decode order (fixed address).
        self.history = t.zeros(self.max_len - length, batch, dtype=t.int64, device=self.device)
        if self.logprobs is not None:
            shape = self.history.shape
            self.scores = TokenLogprobs(t.zeros(shape, device=self.device), t.zeros(shape, device=self.device),
                                        t.zeros((*shape, self.logprobs), device=self.device),
                                        t.zeros((*shape, self.logprobs), dtype=t.int64, device=self.device))
        self.step_index.zero_()
        self.steps_left = self.max_len - length
        return self.tokens.clone()

    def step(self) -> t.Tensor:
        """One decode step: logits [B, vocab]; the argmax becomes the next input token.
        Writes the new token's K/V at `positions`, so at most `max_len - prompt` steps."""
        table = self.allocator.block_table
        blocks = table[self.slots, self.positions // self.block_size]
        offsets = self.positions % self.block_size
        # The new token of every sequence is written at its last attended position.
        ctx = CacheContainer(self.slots, blocks, offsets, self.context_lengths, table, appends_last_position=True)
        # Positions count from the prefix's first token.
        at = self.positions + self.prefix_len if self.prefix is not None else self.positions
        meta = StepMeta("decode", at, ctx, prefix=self.prefix)
        logits = self.model(self.tokens, meta, self.caches)
        nxt = logits.argmax(-1)
        self.history.index_copy_(0, self.step_index, nxt.unsqueeze(0))
        if self.scores is not None:
            for kept, got in zip(self.scores, token_logprobs(logits, nxt, self.logprobs)):
                kept.index_copy_(0, self.step_index, got.unsqueeze(0))
        self.step_index.add_(1)
        self.tokens.copy_(nxt)
        self.positions.add_(1)
        self.context_lengths.add_(1)
        return logits

    def capture(self):
        """Capture one decode step in a HIP graph. Capture records without running,
        so the decoder state is unchanged; every replay is one more step."""
        self.graph = t.cuda.CUDAGraph()
        with t.cuda.graph(self.graph):
            self.logits = self.step()
        return self.graph

    def generate(self, steps: int, use_graph: bool = True) -> t.Tensor:
        """`steps` decode steps -> their tokens [steps, B]. With `use_graph`, the first
        step runs eagerly (warm-up), the step is captured, and the rest are replays."""
        assert 0 < steps <= self.steps_left
        start = int(self.step_index.item())
        for i in range(steps):
            if not use_graph:
                self.step()
            elif self.graph is None:
                self.step()
                self.capture()
            else:
                self.graph.replay()
        self.steps_left -= steps
        self.commit(steps)
        return self.history[start:start + steps]

    def commit(self, steps: int):
        """Advance the allocator's committed lengths (host and device) by the `steps`
        tokens each sequence's decode steps wrote into the cache."""
        self.allocator.advance_batch(list(range(self.batch)), [steps] * self.batch)

    def verify(self, drafts: list[tuple[list[int], list[int]]]) -> list[list[int]]:
        """One pass over the model's choice and a tree of guesses behind it, for each sequence: `drafts[i]` is the guessed
        tokens and the number of the node that each follows, 0 the last chosen token and n the n-th guess. Returns what each
        sequence gains: the guesses that the model agrees with, and its next choice. The tokens are committed, and step,
        generate or verify go on behind them; `history` has steps only. Reads the result on the host."""
        if self.prefix is not None or self.logprobs is not None:
            raise ValueError("GreedyDecoder: verify takes neither a shared prefix nor logprobs")
        if self.slots is None or len(drafts) != self.batch:
            raise ValueError("GreedyDecoder: verify takes a draft for each sequence, after prefill")
        if any(len(guesses) != len(above) or any(p < 0 for p in above) for guesses, above in drafts):
            raise ValueError("GreedyDecoder: a draft is guesses and the node that each follows")
        if any(not 0 <= x < self.model.cfg.vocab_size for guesses, _ in drafts for x in guesses):
            raise ValueError("GreedyDecoder: a guess is a token of the model's vocabulary")
        sizes = [1 + len(guesses) for guesses, _ in drafts]
        lengths = [self.allocator.get_seq_len(i) for i in range(self.batch)]
        if any(n + size > self.max_len for n, size in zip(lengths, sizes)):
            raise ValueError(f"GreedyDecoder: a draft passes the {self.max_len} tokens that are reserved")
        parents = [[-1, *above] for _, above in drafts]
        tree = DraftTree.from_parents(parents, self.device)
        if self.positions.tolist() != lengths:
            raise ValueError("GreedyDecoder: commit the steps before a draft")
        nodes, depths, tokens = t.tensor([[i for n in sizes for i in range(n)], [d for own in DraftTree.depths(parents) for d in own],
                                          [x for guesses, _ in drafts for x in (0, *guesses)]], device=self.device)
        tokens[tree.starts[:-1].long()] = self.tokens
        held = self.allocator.seq_lens[self.slots].long().repeat_interleave(t.tensor(sizes, device=self.device), output_size=len(nodes))
        ctx = self.allocator.create_container(self.slots, tree.starts, held + nodes, validate=False)
        logits = self.model(tokens, StepMeta("verify", held + depths, ctx, tree=tree), self.caches)
        got = accept_draft(tokens, logits.argmax(-1), tree, self.caches, ctx)
        self.tokens.copy_(got.next_tokens)
        self.positions.add_(got.counts)
        self.context_lengths.add_(got.counts)
        counts, path, last = got.counts.tolist(), got.path.tolist(), got.next_tokens.tolist()
        self.allocator.advance_batch(list(range(self.batch)), counts)
        self.steps_left = min(self.steps_left, self.max_len - max(n + c for n, c in zip(lengths, counts)))
        return [[*(drafts[i][0][node - 1] for node in path[i][1:counts[i]]), last[i]] for i in range(self.batch)]
