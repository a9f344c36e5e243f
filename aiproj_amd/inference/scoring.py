"""Scores of many continuations of one prompt.

`score_continuations(model, prompt, continuations, top=0)` gives the log probability of every token
of every continuation, with the entropy and `top` alternatives at its place. The prompt is run through
the model once; the continuations follow packed, in passes of up to 16384 tokens, in which each attends the prompt's
keys and values in the paged cache (`kernals/shared_prefix_attention.py`) and its own, and a pass's logits are
scored in one launch (`kernals/token_logprobs.py`). The reference has no counterpart.
"""

from __future__ import annotations

import torch as t

from aiproj_amd.inference.page_allocator import PageAllocator
from aiproj_amd.inference.paged_kv_cache import PagedKVCache
from aiproj_amd.kernals.shared_prefix_attention import SharedPrefix
from aiproj_amd.kernals.token_logprobs import TokenLogprobs, token_logprobs
from aiproj_amd.model.transformer import StepMeta, TransformerLM


# A pass holds the logits of all of its tokens: at most this many tokens and 2^30 logits (2 GiB of 16 bits), or one
# continuation. Its rows also stay far below the size from which shared prefixes are read row by row.
_PASS_TOKENS = 1 << 14
_PASS_LOGITS = 1 << 30


def _passes(lengths: list[int], most: int) -> list[range]:
    """Runs of the sequences of these lengths, in order, of at most `most` tokens (or of one sequence)."""
    runs, first, held = [], 0, 0
    for i, n in enumerate(lengths):
        if i > first and held + n > most:
            runs.append(range(first, i))
            first, held = i, 0
        held += n
    return [*runs, range(first, len(lengths))]


@t.no_grad()
def score_continuations(model: TransformerLM, prompt: t.Tensor, continuations: list[t.Tensor], top: int = 0,
                        cache_dtype=t.float8_e4m3fn, block_size: int = 16) -> list[TokenLogprobs]:
    """prompt [P] and continuations [n_i] int64, P and every n_i at least 1 -> one TokenLogprobs of n_i rows each."""
    cfg, device = model.cfg, model.embed.weight.device
    if prompt.ndim != 1 or prompt.shape[0] == 0 or not continuations or any(c.ndim != 1 or c.shape[0] == 0 for c in continuations):
        raise ValueError("score_continuations: a prompt and continuations of at least one token each")
    held, lengths = prompt.shape[0], [c.shape[0] for c in continuations]
    if held + max(lengths) > cfg.max_seq_len:
        raise ValueError("score_continuations: prompt and continuation together are at most the model's max_seq_len")
    runs = _passes(lengths, min(_PASS_TOKENS, _PASS_LOGITS // cfg.vocab_size))
    blocks, widest = [-(-n // block_size) for n in lengths], max(map(len, runs))
    pages = -(-held // block_size) + max(sum(blocks[i] for i in run) for run in runs)
    allocator = PageAllocator(pages, block_size, widest + 1, max(held, *lengths), device)
    caches = [PagedKVCache(pages, block_size, cfg.num_kv_heads, cfg.head_dim, device, cache_dtype) for _ in range(cfg.num_layers)]

    def packed(slots, sizes, first, **more):
        """What a pass over sequences of these sizes on these slots needs, positions counted from `first`."""
        own = t.cat([t.arange(n, device=device) for n in sizes])
        cu = t.tensor([0, *sizes], device=device).cumsum(0).to(t.int32)
        ctx = allocator.create_container(t.tensor(slots, dtype=t.int64, device=device), cu, own, validate=False)
        return StepMeta("prefill", own + first, ctx, cu_seqlens=cu, max_seqlen=max(sizes), **more)

    count = len(continuations)
    slot = allocator.allocate_request(count, held)
    before = model(prompt.to(device), packed([slot], [held], 0), caches)                  # [1, vocab]
    allocator.advance(count, held)
    start = token_logprobs(before.expand(count, -1), t.cat([c[:1].to(device) for c in continuations]), top)
    scores = []
    for run in runs:
        sizes = [lengths[i] for i in run]
        slots = [allocator.allocate_request(i, lengths[i]) for i in run]
        tokens = t.cat([continuations[i].to(device) for i in run])
        meta = packed(slots, sizes, held, prefix=SharedPrefix.one(slot, held, len(run), device), all_logits=True)
        # Row i of a continuation predicts its token i + 1; the prompt's last row predicts every first token.
        targets = tokens.roll(-1)
        targets[meta.cu_seqlens[1:].long() - 1] = -1
        rest = token_logprobs(model(tokens, meta, caches), targets, top)
        a = 0
        for i in run:
            scores.append(TokenLogprobs(*(t.cat([s[i:i + 1], r[a:a + lengths[i] - 1]]) for s, r in zip(start, rest))))
            a += lengths[i]
            allocator.free_request(i)
    return scores
