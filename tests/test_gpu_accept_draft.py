"""Kept nodes of drafts and their cache rows, against a walk on the host."""

import random

import pytest
import torch as t

from aiproj_amd.inference.paged_kv_cache import PagedKVCache
from aiproj_amd.kernals.draft_tree import DraftTree, accept_draft
from tests import draft_tree_cases as cases

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = t.bfloat16, t.float16, t.float32, t.float8_e4m3fn


def _walk(parents, tokens, best):
    path = [0] if parents else []
    while path:
        child = next((i for i, p in enumerate(parents) if p == path[-1] and tokens[i] == best[path[-1]]), None)
        if child is None:
            break
        path.append(child)
    return path


def _choices(c, rng, vocab, kept):
    """Tokens and choices: few tokens, so that siblings share some; a path of up to `kept` nodes agrees."""
    tokens, best = [], []
    for own in c.parents:
        mine, chosen = [rng.randrange(vocab) for _ in own], [rng.randrange(vocab) for _ in own]
        at = 0
        for _ in range(kept):
            below = [i for i, p in enumerate(own) if p == at and i > at]
            if not below:
                break
            nxt = rng.choice(below)
            chosen[at] = mine[nxt]
            at = nxt
        tokens.append(mine)
        best.append(chosen)
    return tokens, best


def _layers(c, layers):
    """Caches with rows of their own bytes."""
    out = []
    for i in range(layers):
        cache = PagedKVCache(*c.cache.k.shape, "cuda", c.cache.cache_dtype)
        gen = t.Generator(device="cuda").manual_seed(i)
        for x in (cache.k, cache.v, cache.k_scales, cache.v_scales):
            if x is not None:
                x.view(t.uint8).copy_(t.randint(0, 255, x.view(t.uint8).shape, generator=gen, device="cuda", dtype=t.uint8))
        out.append(cache)
    return out


def _bytes(cache):
    return [x.view(t.uint8).clone() for x in (cache.k, cache.v, cache.k_scales, cache.v_scales) if x is not None]


def _expected(c, before, paths):
    """The rows moved on the host."""
    after = [x.clone() for x in before]
    for b, path in enumerate(paths):
        slot, first = int(c.ctx.cache_slots[b]), int(c.ctx.context_lengths[b]) - c.nodes[b]
        if not 0 <= slot < c.table.shape[0] or first < 0:
            continue
        for j, i in enumerate(path):
            places = []
            for pos in (first + i, first + j):
                page = int(c.table[slot, pos // c.page]) if pos < c.table.shape[1] * c.page else -1
                places.append((page, pos % c.page) if 0 <= page < len(before[0]) else None)
            if None not in places:
                for x, y in zip(before, after):
                    y[places[1]] = x[places[0]]
    return after


def _check(c, tokens, best, layers=3, index=t.int64):
    caches = _layers(c, layers)
    before = [_bytes(x) for x in caches]
    lead, behind = [0] * c.starts[0], [0] * (len(c.q) - c.starts[-1])
    flat = [t.tensor(lead + [x for own in rows for x in own] + behind, dtype=index, device="cuda") for rows in (tokens, best)]
    got = accept_draft(*flat, c.tree, caches, c.ctx)
    cut = [(p[:c.max_nodes], x[:c.max_nodes], y) for p, x, y in zip(c.parents, tokens, best)]
    paths = [_walk(*x) for x in cut]
    assert got.counts.dtype == t.int32 and got.counts.tolist() == [len(p) for p in paths]
    assert got.path.dtype == t.int32 and got.path.tolist() == [p + [-1] * (c.max_nodes - len(p)) for p in paths]
    assert got.next_tokens.dtype == t.int64 and got.next_tokens.tolist() == [b[p[-1]] if p else -1 for p, b in zip(paths, best)]
    for cache, old in zip(caches, before):
        for x, y in zip(_bytes(cache), _expected(c, old, paths)):
            assert t.equal(x, y)
    return paths


@pytest.mark.parametrize("form", [(2, 64, FP8, 16), (4, 128, FP8, 16), (1, 40, FP8, 8), (3, 5, FP8, 1), (2, 64, BF16, 16), (3, 1, F16, 4),
                                  (2, 6, F32, 32), (8, 128, FP8, 64)], ids=str)
@pytest.mark.parametrize("shape", ["tree", "chain", "star", "roots"])
def test_against_a_walk(form, shape):
    hkv, d, dtype, page = form
    rng = random.Random(d)
    c = cases.case([0, 3, 17, 100, 31, 5], [1, 9, 70, 33, 256, 0], hkv, hkv, d, F32, dtype, page, shape)
    kept = 0
    for vocab, deep in ((3, 0), (50, 5), (9, 40)):
        kept += sum(map(len, _check(c, *_choices(c, rng, vocab, deep))))
    assert kept > 18 or shape == "roots"


def test_more_layers_than_a_launch_and_none():
    c = cases.case([40, 7], [12, 30], 2, 2, 64, BF16, FP8)
    _check(c, *_choices(c, random.Random(1), 9, 6), layers=131, index=t.int32)
    _check(c, *_choices(c, random.Random(2), 9, 6), layers=0)


def test_rows_of_no_sequence_and_past_max_nodes():
    c = cases.case([40, 7, 90], [12, 30, 5], 2, 2, 64, BF16, FP8, lead=2, behind=4, max_nodes=11, index=t.int32)
    _check(c, *_choices(c, random.Random(1), 3, 9))


def test_missing_pages_slots_and_lengths():
    c = cases.case([40, 7, 90, 33, 15, 64], [40, 30, 20, 20, 30, 30], 2, 2, 64, BF16, FP8, shape="chain")
    tokens = [[5] * n for n in c.nodes]                    # everything agrees: the whole chain stays where it is
    assert [len(p) for p in _check(c, tokens, tokens)] == c.nodes
    c.parents = [[-1, 0, 0] + list(range(2, n - 1)) for n in c.nodes]              # node 1 beside the chain
    c.tree.parents.copy_(t.tensor([p for own in c.parents for p in own]))
    tokens = [[5, 6] + [5] * (n - 2) for n in c.nodes]
    best = [[5] * n for n in c.nodes]
    slots = c.ctx.cache_slots
    c.table[slots[0], 3] = -1
    c.table[slots[1], 0] = len(c.cache.k)
    c.ctx.context_lengths[2] = 10 ** 5
    c.ctx.context_lengths[3] = 19
    slots[4] = 77
    _check(c, tokens, best)


def test_not_aligned_caches():
    """Rows at odd addresses move by bytes, at multiples of four by words."""
    c = cases.case([20], [16], 2, 2, 64, BF16, FP8)
    for shift in (1, 4):
        tokens, best = _choices(c, random.Random(shift), 4, 6)
        caches = _layers(c, 2)
        for cache in caches:
            raw = t.zeros(cache.k.numel() + 16, dtype=t.uint8, device="cuda")
            raw[shift:shift + cache.k.numel()] = cache.k.view(t.uint8).flatten()
            cache.k = raw[shift:shift + cache.k.numel()].view(cache.k.shape).view(FP8)
        before = [_bytes(x) for x in caches]
        accept_draft(t.tensor(tokens[0], device="cuda"), t.tensor(best[0], device="cuda"), c.tree, caches, c.ctx)
        for cache, old in zip(caches, before):
            assert all(t.equal(x, y) for x, y in zip(_bytes(cache), _expected(c, old, [_walk(c.parents[0], tokens[0], best[0])])))


def test_captured_and_replayed():
    c = cases.case([40, 7], [12, 30], 2, 2, 64, BF16, FP8)
    caches = _layers(c, 2)
    tokens, best = (t.zeros(42, dtype=t.int64, device="cuda") for _ in range(2))
    accept_draft(tokens, best, c.tree, caches, c.ctx)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        got = accept_draft(tokens, best, c.tree, caches, c.ctx)
    for i in range(3):
        x, y = _choices(c, random.Random(i), 4, 2 * i)
        tokens.copy_(t.tensor(sum(x, [])))
        best.copy_(t.tensor(sum(y, [])))
        before = [_bytes(z) for z in caches]
        graph.replay()
        t.cuda.synchronize()
        paths = [_walk(p, a, b) for p, a, b in zip(c.parents, x, y)]
        assert got.counts.tolist() == [len(p) for p in paths]
        for cache, old in zip(caches, before):
            assert all(t.equal(p, q) for p, q in zip(_bytes(cache), _expected(c, old, paths)))
