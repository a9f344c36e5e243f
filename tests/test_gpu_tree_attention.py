"""Attention of drafted trees against float64 over the cache as it is stored."""

import math
import random
from types import SimpleNamespace

import pytest
import torch as t

from aiproj_amd.inference.paged_kv_cache import PagedKVCache
from aiproj_amd.kernals import draft_tree
from aiproj_amd.kernals.decode_attention import decode_attention_wrapper
from aiproj_amd.kernals.draft_tree import DraftTree, append_tree_attention, tree_attention
from tests import draft_tree_cases as cases

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = t.bfloat16, t.float16, t.float32, t.float8_e4m3fn
HALF = {x: t.finfo(x).eps / 2 for x in (BF16, F16, F32)}
# (q heads, KV heads, head size, q type, cache type, page)
FORMS = [(8, 2, 64, BF16, FP8, 16), (32, 8, 128, BF16, FP8, 16), (16, 1, 128, F16, FP8, 32), (64, 8, 128, BF16, FP8, 64),
         (6, 2, 80, F16, FP8, 16), (4, 4, 96, BF16, FP8, 16), (8, 1, 112, F32, FP8, 16), (8, 2, 128, F32, FP8, 16),
         (24, 12, 64, BF16, FP8, 16), (8, 4, 64, BF16, BF16, 16), (32, 2, 128, BF16, BF16, 128), (8, 4, 128, F16, F16, 64),
         (4, 2, 64, F16, F16, 16), (34, 2, 64, F16, FP8, 16), (8, 2, 112, BF16, FP8, 32), (4, 2, 64, F16, BF16, 16),
         (8, 4, 64, BF16, F32, 16), (8, 8, 40, BF16, FP8, 8), (2, 1, 300, F32, F32, 4), (3, 3, 1, F32, BF16, 1), (4, 2, 512, F16, F16, 16)]
IDS = ["-".join(str(x).replace("torch.", "") for x in f) for f in FORMS]
# (tokens held, nodes, shape)
BATCHES = {
    "one": ([0], [1], "chain"),
    "first": ([0, 0, 5], [3, 40, 1], "tree"),
    "ragged": ([1, 0, 5, 33, 317, 64, 100], [1, 7, 16, 2, 33, 12, 0], "tree"),
    "chain": ([31, 250], [130, 9], "chain"),
    "roots": ([16, 47], [9, 65], "roots"),
    "star": ([100, 7], [64, 5], "star"),
    "large": ([300, 12], [256, 129], "tree"),
    "long": ([5003, 2], [21, 4], "tree"),
    "many": ([(7 * i) % 50 for i in range(75)], [1 + (5 * i) % 6 for i in range(75)], "tree"),
}


def _weights_half(q_dtype, cache_dtype):
    """bf16 q: weights of bf16. f16 q over an f16 cache: of f16. Others: parts that hold 16 bits and more."""
    if q_dtype == BF16 and cache_dtype in (FP8, BF16):
        return HALF[BF16]
    return HALF[F16] if (q_dtype, cache_dtype) == (F16, F16) else 2.0 ** -15


def _check(c, got):
    """float32 scores: D products and sums of |q k| scale, each with half a step of 2^-24, move a weight by as much relatively,
    and the sums over tokens add theirs: 2^-12 covers D 128 at |q k| scale of 10 and 5000 tokens (D 512: four times the
    products of a quarter of the size). Then the half step of the weights' type in the matrix products, and of the output's."""
    rows, want, size = cases.attention_64(c)
    assert got.dtype == c.q.dtype and got.shape == c.q.shape
    got = got[rows]
    bound = HALF[got.dtype] * want.abs() + (_weights_half(c.q.dtype, c.cache.k.dtype) + 2.0 ** -12) * size
    bound = bound + (2.0 ** -25 if got.dtype == F16 else 0.0)                  # half of the smallest step of float16
    fine = want.isfinite()
    assert t.equal(fine, got.isfinite())
    assert bool(((got.double() - want).abs() <= bound)[fine].all()), float(((got.double() - want).abs() - bound)[fine].max())


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_against_float64(form, batch):
    held, nodes, shape = BATCHES[batch]
    hq, hkv, d, q_dtype, cache_dtype, page = form
    if hq * d > 4000 and batch in ("large", "long"):
        held, nodes = held[1:], nodes[1:]
    c = cases.case(held, nodes, hq, hkv, d, q_dtype, cache_dtype, page, shape, index=t.int32 if batch == "many" else t.int64)
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))


@pytest.mark.parametrize("form", [FORMS[1], FORMS[4], FORMS[9], FORMS[17]])
def test_strided_q(form):
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([40, 3, 100], [9, 17, 1], hq, hkv, d, q_dtype, cache_dtype, page)
    for pad, at in ((8, 8), (3, 1)):
        wide = t.zeros(len(c.q), hq, d + pad, dtype=q_dtype, device="cuda")
        wide[:, :, at:at + d] = c.q
        c.q = wide[:, :, at:at + d]
        _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))
    c.q = c.q.transpose(1, 2).contiguous().transpose(1, 2)
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))
    c.ctx.cache_slots = c.ctx.cache_slots.repeat_interleave(2)[::2]
    c.ctx.block_table = t.cat([c.table, c.table], 1)[:, :c.table.shape[1]]
    c.tree = DraftTree(c.tree.starts.repeat_interleave(3)[::3], c.tree.parents.repeat_interleave(2)[::2], c.max_nodes)
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))


SOME = [FORMS[0], FORMS[1], FORMS[5], FORMS[9], FORMS[11], FORMS[17]]


@pytest.mark.parametrize("form", SOME)
def test_rows_of_no_sequence_and_past_max_nodes_stay(form):
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([20, 0, 70, 5], [6, 3, 40, 2], hq, hkv, d, q_dtype, cache_dtype, page, lead=3, behind=5, max_nodes=17)
    marked = t.full_like(c.q, 7.0)
    real = t.empty
    try:
        t.empty = lambda *a, **k: marked if a and a[0] == tuple(marked.shape) else real(*a, **k)
        got = tree_attention(c.q, c.cache, c.ctx, c.tree)
    finally:
        t.empty = real
    assert got is marked
    _check(c, got)
    rows = set(cases.attention_64(c)[0])
    others = [r for r in range(len(c.q)) if r not in rows]
    assert len(others) == 3 + 23 + 5 and bool((got[others] == 7.0).all())


@pytest.mark.parametrize("form", SOME)
def test_missing_pages_slots_and_lengths(form):
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([90, 90, 90, 9, 700, 33], [10, 10, 30, 3, 20, 4], hq, hkv, d, q_dtype, cache_dtype, page)
    slots = c.ctx.cache_slots
    c.table[slots[0], 1] = -1
    c.table[slots[1], 90 // page] = c.cache.k.shape[0]          # where the nodes begin
    c.table[slots[2], :] = 2 ** 30                              # every page
    c.table[slots[4], 300 // page] = -5
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))
    assert not bool(tree_attention(c.q, c.cache, c.ctx, c.tree)[c.starts[2]:c.starts[3]].any())
    c.ctx.context_lengths[0] = 9                                # fewer tokens than nodes
    c.ctx.context_lengths[3] = -5
    slots[1], slots[5] = 4096, -1
    c.ctx.context_lengths[4] = 10 ** 6                          # past the table: its nodes are not there
    got = tree_attention(c.q, c.cache, c.ctx, c.tree)
    _check(c, got)
    for b in (0, 1, 3, 5):
        assert not bool(got[c.starts[b]:c.starts[b + 1]].any())


@pytest.mark.parametrize("form", [FORMS[0], FORMS[17]])
def test_parents_that_are_none(form):
    """Numbers that are no smaller node of the sequence make roots, whatever their bits."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([40], [8], hq, hkv, d, q_dtype, cache_dtype, page)
    c.parents[0] = [5, 0, 2, 1, -9, 2 ** 40 + 1, -2 ** 40 + 3, 4]
    c.tree.parents.copy_(t.tensor(c.parents[0]))
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))


@pytest.mark.parametrize("form", SOME + [FORMS[6], FORMS[2], FORMS[12]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_other_branches_hold_does_not_matter(form, bad):
    """NaN and infinities in a node's key, value or scale reach the rows that attend it and no other."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([37, 0, 200], [20, 5, 70], hq, hkv, d, q_dtype, cache_dtype, page)
    hit = {}
    for b, node, where in ((0, 4, "v"), (0, 7, "k"), (1, 4, "v"), (2, 33, "v"), (2, 50, "k"), (2, 69, "v")):
        pos = c.held[b] + node
        p, o = int(c.table[c.ctx.cache_slots[b], pos // page]), pos % page
        x, scales = (c.cache.k, c.cache.k_scales) if where == "k" else (c.cache.v, c.cache.v_scales)
        if not c.cache.quantized:
            x[p, o, 0, d // 2] = bad
        elif bad != bad:
            x.view(t.uint8)[p, o, 0, d // 2] = 0xFF if node % 2 else 0x7F
        else:
            scales[p, o, 0] = bad
        hit.setdefault(b, []).append(node)
    got = tree_attention(c.q, c.cache, c.ctx, c.tree)
    _check(c, got)
    clean = [c.starts[b] + i for b, nodes in hit.items() for i in range(c.nodes[b]) if not cases.above(c.parents[b], i) & set(nodes)]
    assert len(clean) > 20 and bool(got[clean].isfinite().all()) and not bool(got.isfinite().all())


@pytest.mark.parametrize("form", [FORMS[9], FORMS[11]])
def test_values_of_another_branch_that_are_infinite(form):
    """The rows that attend an infinite value have it, as they would by the formula (codes hold none)."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([10], [6], hq, hkv, d, q_dtype, cache_dtype, page, shape="star")
    pos = 10 + 3
    p, o = int(c.table[c.ctx.cache_slots[0], pos // page]), pos % page
    c.cache.v[p, o, 1, 5] = -float("inf")
    got = tree_attention(c.q, c.cache, c.ctx, c.tree)
    g = hq // hkv
    assert bool((got[3, g:2 * g, 5] == -float("inf")).all()) and bool(got[[0, 1, 2, 4, 5]].isfinite().all())
    got[3, g:2 * g, 5] = 0
    assert bool(got[3].isfinite().all())


@pytest.mark.parametrize("form", [FORMS[1], FORMS[7], FORMS[9], FORMS[17]])
def test_one_node_is_a_decode_step(form):
    """A batch of single nodes: what the decode kernels give, each within its bound of float64."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([0, 5, 100, 777], [1, 1, 1, 1], hq, hkv, d, q_dtype, cache_dtype, page)
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))
    _check(c, decode_attention_wrapper(c.q, c.cache, c.ctx))


def test_append_then_attend():
    c = cases.case([30, 64], [7, 12], 8, 2, 64, BF16, FP8)
    k, v = (t.randn(19, 2, 64, device="cuda", dtype=BF16) for _ in range(2))
    pos = t.cat([c.held[b] + t.arange(c.nodes[b]) for b in range(2)]).cuda()
    seq = t.tensor([0] * 7 + [1] * 12, device="cuda")
    c.ctx.physical_blocks = c.table[c.ctx.cache_slots[seq], pos // 16]
    c.ctx.block_offsets = pos % 16
    got = append_tree_attention(c.q, k, v, c.cache, c.ctx, c.tree)
    _check(c, got)
    other = PagedKVCache(*c.cache.k.shape, "cuda", FP8)
    other.append_kv(c.ctx.physical_blocks, c.ctx.block_offsets, k, v)
    at = (c.ctx.physical_blocks, c.ctx.block_offsets)
    assert t.equal(other.k.view(t.uint8)[at], c.cache.k.view(t.uint8)[at]) and t.equal(other.v_scales[at], c.cache.v_scales[at])


@pytest.mark.parametrize("form", [FORMS[1], FORMS[9]])
def test_scores_of_any_size(form):
    """Equal keys share the weight, and the largest wins, at scores of thousands."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([500, 64], [10, 30], hq, hkv, d, q_dtype, cache_dtype, page, spread=30.0)
    c.q *= 20.0
    got = tree_attention(c.q, c.cache, c.ctx, c.tree)
    rows, want, size = cases.attention_64(c)
    # Scores of up to 1e4 are off by D half steps of float32: 2^-24 x 128 x 1e4 = 8e-2 of a weight.
    assert bool(((got.double() - want).abs() <= (HALF[q_dtype] * 2 + 0.16) * size).all()) and bool(got.isfinite().all())


@pytest.mark.parametrize("form", [FORMS[1], FORMS[9], FORMS[17]])
def test_captured_and_replayed(form):
    """Trees, lengths, pages and queries change between replays, beside eager calls of other sizes."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    sets = [cases.case([300, 20, 0], [12, 5, 30], hq, hkv, d, q_dtype, cache_dtype, page, "tree"),
            cases.case([40, 200, 80], [20, 17, 10], hq, hkv, d, q_dtype, cache_dtype, page, "chain", seed=3),
            cases.case([0, 0, 320], [1, 1, 45], hq, hkv, d, q_dtype, cache_dtype, page, "star", seed=5)]
    assert all(len(s.q) == 47 for s in sets)
    pool, width = max(len(s.cache.k) for s in sets), max(s.table.shape[1] for s in sets)
    live = cases.case([300, 20, 0], [12, 5, 30], hq, hkv, d, q_dtype, cache_dtype, page)
    live.cache = PagedKVCache(pool, page, hkv, d, "cuda", cache_dtype)
    live.ctx.block_table = t.full((3, width), -1, dtype=t.int32, device="cuda")
    live.tree = DraftTree(live.tree.starts, live.tree.parents, 45)

    def load(s):
        for name in ("k", "v", "k_scales", "v_scales"):
            x, y = getattr(live.cache, name), getattr(s.cache, name)
            if x is not None:
                x.view(t.uint8 if x.dtype == FP8 else x.dtype)[:len(y)] = y.view(t.uint8 if x.dtype == FP8 else x.dtype)
        live.ctx.block_table.fill_(-1)
        live.ctx.block_table[:, :s.table.shape[1]] = s.table
        for x, y in ((live.q, s.q), (live.tree.starts, s.tree.starts), (live.tree.parents, s.tree.parents),
                     (live.ctx.cache_slots, s.ctx.cache_slots), (live.ctx.context_lengths, s.ctx.context_lengths)):
            x.copy_(y)

    load(sets[0])
    tree_attention(live.q, live.cache, live.ctx, live.tree)
    graphs = []
    for _ in range(2):                                          # two graphs share no workspace
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            out = tree_attention(live.q, live.cache, live.ctx, live.tree)
        graphs.append((graph, out))
    for s in sets + sets[:1]:
        load(s)
        for graph, out in graphs:
            out.fill_(9.0)
            graph.replay()
            tree_attention(s.q[:1], s.cache, s.ctx, DraftTree(s.tree.starts.clamp(max=1), s.tree.parents[:1], 1))
        t.cuda.synchronize()
        for _, out in graphs:
            _check(s, out)


def test_two_streams_at_once():
    a = cases.case([900, 30], [20, 40], 32, 8, 128, BF16, FP8)
    b = cases.case([10, 1200], [30, 9], 32, 8, 128, BF16, FP8, seed=2)
    one, two = t.cuda.Stream(), t.cuda.Stream()
    for s in (one, two):
        s.wait_stream(t.cuda.current_stream())
    outs = []
    for _ in range(20):
        for s, c in ((one, a), (two, b)):
            with t.cuda.stream(s):
                outs.append((c, tree_attention(c.q, c.cache, c.ctx, c.tree)))
    t.cuda.synchronize()
    for c, got in outs[:2]:
        _check(c, got)
    assert all(t.equal(got, outs[i % 2][1]) for i, (_, got) in enumerate(outs))


def test_no_rows_and_no_sequences():
    c = cases.case([5], [2], 4, 2, 64, BF16, FP8)
    assert tree_attention(c.q[:0], c.cache, c.ctx, DraftTree(c.tree.starts, c.tree.parents[:0], 4)).shape == (0, 4, 64)
    c.ctx.cache_slots, c.ctx.context_lengths = c.ctx.cache_slots[:0], c.ctx.context_lengths[:0]
    assert tree_attention(c.q, c.cache, c.ctx, DraftTree(c.tree.starts[:1], c.tree.parents, 4)).shape == (2, 4, 64)


@pytest.mark.parametrize("q_dtype,cache_dtype", [(F16, FP8), (BF16, BF16), (F32, FP8), (F16, F32)])
@pytest.mark.parametrize("batch", [64, 150])
def test_more_columns_than_run_at_once(q_dtype, cache_dtype, batch):
    """Sequences of all lengths, which are then taken in the order of their lengths, 64 by 64."""
    rng = random.Random(batch)
    held = [rng.choice((0, 1, 15, 40, 64, 90, 150)) for _ in range(batch)]
    held[batch // 2], held[-1] = 1700, 900
    c = cases.case(held, [rng.randint(0, 20) for _ in range(batch)], 32, 8, 64, q_dtype, cache_dtype)
    c.ctx.context_lengths[3], c.ctx.cache_slots[9] = -1, -1
    _check(c, tree_attention(c.q, c.cache, c.ctx, c.tree))


@pytest.mark.parametrize("form", [FORMS[0], FORMS[1], FORMS[9], FORMS[17]])
def test_scales_of_either_sign(form, monkeypatch):
    """A negative scale is that of the negated queries, and 0 weighs all tokens alike."""
    hq, hkv, d, q_dtype, cache_dtype, page = form
    c = cases.case([70, 5], [20, 9], hq, hkv, d, q_dtype, cache_dtype, page)
    for root, factor in ((lambda d: -math.sqrt(d), -1.0), (lambda d: float("inf"), 0.0)):
        monkeypatch.setattr(draft_tree, "math", SimpleNamespace(sqrt=root))
        got, q = tree_attention(c.q, c.cache, c.ctx, c.tree), c.q
        c.q = q * factor
        _check(c, got)
        c.q = q
